// kv4_rows.cu -- attention over the 4-bit paged cache (kv4_attention.cu has the
// definition) for many query rows a KV head: the suffix of a request computed
// over its retrieved prefix, or several tokens checked at once.
//
// A unit is 128 query rows (query tokens times the heads that share a KV head)
// of one request and KV head; its rows are the lanes of the tensor memory. With
// a tile of 64 cache tokens:
//   S = Q Ck^T     tcgen05.mma 128 x 64 x D, Ck the K codes,
//   t = S sk + zk (sum of q), p = exp2(t a - m),
//   O += P V'      tcgen05.mma 128 x D x 64, P from tensor memory.
// The K codes are exact as in the decode kernel (the fp16 bit patterns c and
// 16 c, c 2^-24; Q's odd elements carry the 1/16), so a logit is an fp32 sum of
// exact products. V is made fp16 on the way, v 2^-e with 2^e above the largest
// of its 16 tokens; P takes the 2^e, relative to the row's own E, so neither
// loses small caches nor overflows. The rounding of v and of p are 2^-12 each
// of their own size: dequantising V costs 128 rows nothing, where taking sv
// into P, as the decode kernel does, would cost every element of S.
//
// Per tile and SM the tensor core needs 512 cycles, the exponentials 512 (16 a
// cycle), and the rest of softmax and dequantisation about as many issue
// slots. So two CTAs share an SM, each with its half of the tensor memory (two
// S of 64 columns and O), and one computes softmax while the other's products
// run: four warps of a CTA have a query row a thread, four bring the codes from
// the pages and expand them to 16 bits into two stages of shared memory (128-
// byte swizzled; a lane's 16-byte pieces of 4 tokens x 2 halves of a panel hit
// all banks). S of the next tile is under way before softmax starts. O stays
// in tensor memory; it is rescaled only when a row's reference grows by more
// than 2^12, which P's range leaves room for.
#include <climits>

#include "kv4_attention.cuh"
#include "kv4_plan.h"

namespace lmcb {
namespace kv4 {
namespace {

constexpr int kRows = 128;   // query rows of a unit
constexpr int kTok = 64;     // cache tokens of a tile
constexpr int kThreads = 256;
constexpr float kSlack = 12.0f;  // log2 of how far P may exceed 1

struct RowsParams {
  AttnParams a;
  int32_t splits;  // CTAs that share a unit's tiles
  float* part;     // [unit][splits][kRows][D + 4]
  int32_t row_tiles;
};

// Packed pairs of fp32.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// ---------------------------------------------------------------------------
// Tensor memory and tcgen05
// ---------------------------------------------------------------------------

__device__ __forceinline__ void tmem_load32(uint32_t (&r)[32], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}

__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_load() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_wait_store() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// Shared-memory operand descriptor: 128-byte swizzle (8 rows of 128 bytes),
// `stride` bytes from one group of 8 rows to the next and `lead` bytes from one
// 64-element panel to the next (operands whose rows run along K).
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead, uint32_t stride) {
  return static_cast<uint64_t>((addr >> 4) & 0x3fff) |
         (static_cast<uint64_t>((lead >> 4) & 0x3fff) << 16) |
         (static_cast<uint64_t>((stride >> 4) & 0x3fff) << 32) | (uint64_t{1} << 46) |
         (uint64_t{2} << 61);
}

// fp16 x fp16 into fp32, M = 128; `across`: B's rows run along K (V as it is
// stored: a token's values side by side).
__host__ __device__ constexpr uint32_t instruction(int n, bool across) {
  return (1u << 4) | (across ? 1u << 16 : 0u) | (static_cast<uint32_t>(n / 8) << 17) |
         (static_cast<uint32_t>(kRows / 16) << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t instr,
                                       bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(instr), "r"(add ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t instr,
                                       bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(instr), "r"(add ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smem_u32(bar))
               : "memory");
}

// ---------------------------------------------------------------------------
// Shared memory
// ---------------------------------------------------------------------------

template <int D>
struct Layout {
  static constexpr int kPanels = D / 64;                     // of 64 values, 128 bytes a row
  static constexpr int kQPanel = kRows * 128;
  static constexpr int kPanel = kTok * 128;
  static constexpr int kStage = kPanels * kPanel;
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + kPanels * kQPanel;
  static constexpr int kV = kK + 2 * kStage;
  static constexpr int kBytes = kV + 2 * kStage;
  static constexpr uint32_t kColumns = D <= 128 ? 256 : 512;  // tensor memory
  static constexpr uint32_t kO = 2 * kTok;                    // its columns behind two S
};

struct Control {
  uint64_t kfull[2], vfull[2], qkdone[2], pvdone[2], drained;
  float4 kpar[2][kTok / 2];  // tokens 2 i, 2 i + 1: (sk, sk, zk, zk)
  uint32_t valid[2][4];      // a bit a token, 16 tokens each
  int32_t vexp[2][4];        // e of 16 tokens
  float2 row[kRows];         // a, sum of q 2^-24
  uint32_t tmem;
};

// Byte offset of 16-byte piece `piece` of row `r` in a 128-byte swizzled panel.
__device__ __forceinline__ uint32_t swizzled(uint32_t r, uint32_t piece) {
  return r * 128 + ((piece ^ (r & 7)) << 4);
}

// The unit's query rows, scaled to fp16, into shared memory: two threads a row.
template <typename T, int D>
__device__ __forceinline__ void load_rows(const AttnParams& p, const Request& rq, int first_row,
                                          int kv_head, uint8_t* smem, Control& ctl) {
  const int r = threadIdx.x / 2, side = threadIdx.x % 2;
  constexpr int N = D / 2;
  const int flat = first_row + r;
  const int tok = static_cast<int>(p.div_group.div(static_cast<uint32_t>(flat)));
  const int head = kv_head * p.group + (flat - tok * p.group);
  const bool there = tok < rq.n;
  const T* src = static_cast<const T*>(p.q) + (rq.row0 + static_cast<int64_t>(tok)) * p.q_stride +
                 static_cast<int64_t>(head) * D + side * N;
  float big = 0.0f;
  if (there) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      float x[8];
      load_query<T, 8>(src + 8 * i, p.q_vec != 0, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf(x[j]));
    }
  }
  big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
  const int e = min(max(((__float_as_int(big) >> 23) & 255) - 127, -100), 100);
  // the sign of the scale goes into the rows, so that the largest t is the
  // largest logit
  const float up = p.scale_log2 < 0.0f ? -pow2i(13 - e) : pow2i(13 - e);
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < N / 8; ++i) {
    uint4 out = make_uint4(0, 0, 0, 0);
    if (there) {
      float x[8];
      load_query<T, 8>(src + 8 * i, p.q_vec != 0, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = __half2float(__float2half_rn(x[j] * up));
        sum += x[j];
      }
      out = make_uint4(pack_half2(x[0], x[4]), pack_half2(x[1] * 0.0625f, x[5] * 0.0625f),
                       pack_half2(x[2], x[6]), pack_half2(x[3] * 0.0625f, x[7] * 0.0625f));
    }
    const int at = side * (N / 8) + i;  // 8 values of the row
    *reinterpret_cast<uint4*>(smem + Layout<D>::kQ + (at / 8) * Layout<D>::kQPanel +
                              swizzled(r, at % 8)) = out;
  }
  sum += __shfl_xor_sync(0xffffffffu, sum, 1);
  if (side == 0) {
    // never zero, so that a key that is not seen stays at -inf
    const float a = fmaxf(fabsf(p.scale_log2) * pow2i(e - 13) * 16777216.0f, 1.2e-38f);
    ctl.row[r] = make_float2(a, sum * 5.9604645e-8f);
  }
}

// ---------------------------------------------------------------------------
// The warps that bring K and V
// ---------------------------------------------------------------------------

// What a lane holds of a tile on its way: 32 values in 16 bytes, for each panel
// of K and of V, of one token.
template <int D>
struct Codes {
  uint4 k[D / 64], v[D / 64];
  uint32_t kpar, vpar;
  bool there;
};

template <int D>
__device__ __forceinline__ void fetch(const AttnParams& p, const int32_t* k_head,
                                      const int32_t* par, int32_t row, int lane, Codes<D>& c) {
  c.there = row >= 0;
  if (c.there) {
    const int64_t at = row * p.row_words;
    const int32_t* k = k_head + at + (lane % 2) * 4;
    const int32_t* v = k + p.half_words;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      c.k[i] = __ldg(reinterpret_cast<const uint4*>(k + 8 * i));
      c.v[i] = __ldg(reinterpret_cast<const uint4*>(v + 8 * i));
    }
    c.kpar = static_cast<uint32_t>(__ldg(par + at));
    c.vpar = static_cast<uint32_t>(__ldg(par + p.half_words + at));
  } else {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) c.k[i] = c.v[i] = make_uint4(0, 0, 0, 0);
    c.kpar = c.vpar = 0;
  }
}

__device__ __forceinline__ uint32_t half2_bits(__half2 h) {
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ __half2 as_half2(uint32_t v) {
  return *reinterpret_cast<const __half2*>(&v);
}

// Eight values of V in the order 0, 4, 1, 5, 2, 6, 3, 7: codes on top of 1024,
// which comes off exactly, times s, plus z, rounded once.
__device__ __forceinline__ uint4 expand_v(uint32_t w, __half2 s, __half2 z) {
  const __half2 base = __half2half2(__ushort_as_half(0x6400));
  uint32_t r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __half2 c = __hsub2(as_half2(((w >> (4 * j)) & 0x000f000fu) | 0x64006400u), base);
    r[j] = half2_bits(__hfma2(c, s, z));
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

__device__ __forceinline__ uint4 expand_k(uint32_t w) {
  const uint32_t x = w >> 8;
  return make_uint4(w & 0x000f000fu, w & 0x00f000f0u, x & 0x000f000fu, x & 0x00f000f0u);
}

template <int D>
__device__ __forceinline__ bool bring(const AttnParams& p, const KeyRange& range, int b,
                                      int kv_head, int32_t t0, int32_t tiles, uint8_t* smem,
                                      Control& ctl) {
  using L = Layout<D>;
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32 - 4;
  const int tok = w * 16 + lane / 2;
  const int32_t* table = p.table + static_cast<int64_t>(b) * p.table_stride;
  const int32_t* k_head = p.cache + static_cast<int64_t>(kv_head) * (D / 8);
  const int32_t* par = p.cache + static_cast<int64_t>(p.kv_heads) * (D / 8) + kv_head;
  const auto row = [&](int32_t i) {
    return i < tiles ? row_of(p, table, range, (t0 + i) * kTok + tok) : -1;
  };
  // codes of the next tile and the row of the one after it are on their way
  // while a tile is expanded
  Codes<D> next;
  int32_t after = row(0);
  fetch<D>(p, k_head, par, after, lane, next);
  after = row(1);
  for (int32_t i = 0; i < tiles; ++i) {
    const int buf = i & 1;
    const uint32_t last = ((i >> 1) - 1) & 1;  // parity of the stage's last use
    const Codes<D> c = next;
    fetch<D>(p, k_head, par, after, lane, next);
    after = row(i + 2);
    if (i >= 2 && !mbar_wait(&ctl.qkdone[buf], last)) return false;
    uint8_t* k = smem + L::kK + buf * L::kStage;
    const uint32_t piece = (lane % 2) * 4;
#pragma unroll
    for (int n = 0; n < L::kPanels; ++n) {
      const uint32_t words[4] = {c.k[n].x, c.k[n].y, c.k[n].z, c.k[n].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        *reinterpret_cast<uint4*>(k + n * L::kPanel + swizzled(tok, piece + j)) =
            expand_k(words[j]);
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl.kfull[buf]);
    // the exponent above the largest value of these 16 tokens
    const float s = half_lo(c.vpar), z = half_hi(c.vpar);
    const float most = fmaxf(fabsf(z), fabsf(fmaf(15.0f, s, z)));
    const int e = static_cast<int>(__reduce_max_sync(
                      0xffffffffu, max((__float_as_uint(most) >> 23) & 255u, 80u))) - 126;
    const float down = pow2i(-e);
    const __half2 s2 = __half2half2(__float2half_rn(s * down));
    const __half2 z2 = __half2half2(__float2half_rn(z * down));
    const uint32_t there = __ballot_sync(0xffffffffu, c.there);
    if (i >= 2 && !mbar_wait(&ctl.pvdone[buf], last)) return false;
    uint8_t* v = smem + L::kV + buf * L::kStage;
#pragma unroll
    for (int n = 0; n < L::kPanels; ++n) {
      const uint32_t words[4] = {c.v[n].x, c.v[n].y, c.v[n].z, c.v[n].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        *reinterpret_cast<uint4*>(v + n * L::kPanel + swizzled(tok, piece + j)) =
            expand_v(words[j], s2, z2);
      }
    }
    if (lane % 2 == 0) {
      float* to = reinterpret_cast<float*>(&ctl.kpar[buf][tok / 2]) + tok % 2;
      to[0] = half_lo(c.kpar);
      to[2] = half_hi(c.kpar);
    }
    if (lane == 0) {
      ctl.valid[buf][w] = there;  // two bits a token
      ctl.vexp[buf][w] = e;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl.vfull[buf]);
  }
  return true;
}

// ---------------------------------------------------------------------------
// The warps that have the query rows
// ---------------------------------------------------------------------------

template <int D>
__device__ __forceinline__ void issue_qk(uint32_t tmem, uint32_t smem, int buf) {
  using L = Layout<D>;
  const uint64_t q = operand(smem + L::kQ, 0, 1024);
  const uint64_t k = operand(smem + L::kK + buf * L::kStage, 0, 1024);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const uint32_t in_panel = (i % 4) * 32;
    mma_ss(tmem + buf * kTok, q + (((i / 4) * L::kQPanel + in_panel) >> 4),
           k + (((i / 4) * L::kPanel + in_panel) >> 4), instruction(kTok, false), i > 0);
  }
}

template <int D>
__device__ __forceinline__ void issue_pv(uint32_t tmem, uint32_t smem, int buf, bool add) {
  using L = Layout<D>;
  const uint64_t v = operand(smem + L::kV + buf * L::kStage, L::kPanel, 1024);
#pragma unroll
  for (int i = 0; i < kTok / 16; ++i) {
    mma_ts(tmem + L::kO, tmem + buf * kTok + i * 8, v + ((i * 16 * 128) >> 4),
           instruction(D, true), add || i > 0);
  }
}

// A thread's row: its reference m (log2) and E, the sum l in units of 2^m; O in
// units of 2^(m + E).
struct Row {
  float a, qsum;
  float m, l;
  int e;
  int32_t pos;
};

template <int D>
__device__ __forceinline__ bool attend(const AttnParams& p, const KeyRange& range, int32_t t0,
                                       int32_t tiles, int32_t pos_first, int32_t pos_last,
                                       uint32_t smem, Control& ctl, Row& row) {
  using L = Layout<D>;
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
  const uint32_t tmem = ctl.tmem;
  const uint32_t mine = tmem + (static_cast<uint32_t>(w) << 21);  // lanes 32 w ...
  bool ok = true;
  if (w == 0 && tiles > 0) {
    ok = mbar_wait(&ctl.kfull[0], 0);
    if (ok && lane == 0) {
      fence_after();
      issue_qk<D>(tmem, smem, 0);
      commit(&ctl.qkdone[0]);
    }
    __syncwarp();
  }
  for (int32_t i = 0; i < tiles; ++i) {
    const int buf = i & 1;
    const uint32_t parity = (i >> 1) & 1;
    if (w == 0 && i + 1 < tiles && ok) {
      ok = mbar_wait(&ctl.kfull[buf ^ 1], ((i + 1) >> 1) & 1);
      if (ok && lane == 0) {
        fence_after();
        // into the S whose P the product before has read: products run in order
        issue_qk<D>(tmem, smem, buf ^ 1);
        commit(&ctl.qkdone[buf ^ 1]);
      }
      __syncwarp();
    }
    ok = ok && mbar_wait(&ctl.vfull[buf], parity) && mbar_wait(&ctl.qkdone[buf], parity);
    if (ok) {
      fence_after();
      uint32_t s[2][32];
      tmem_load32(s[0], mine + buf * kTok);
      tmem_load32(s[1], mine + buf * kTok + 32);
      // is every key of the tile there and seen by every row?
      const int32_t v0 = (t0 + i) * kTok;
      const uint32_t there = ctl.valid[buf][0] & ctl.valid[buf][1] & ctl.valid[buf][2] &
                             ctl.valid[buf][3];
      const int32_t key0 = key_of(range, v0), key1 = key_of(range, v0 + kTok - 1);
      const bool all = there == 0xffffffffu && key1 <= pos_first &&
                       (p.window == 0 || key0 > pos_last - p.window || key1 < p.sinks);
      tmem_wait_load();
      uint64_t t[kTok / 2];
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      const uint64_t qsum = pair(row.qsum, row.qsum);
#pragma unroll
      for (int c = 0; c < kTok / 2; ++c) {
        const float4 kp = ctl.kpar[buf][c];
        const uint64_t acc = pair(__uint_as_float(s[c / 16][(2 * c) % 32]),
                                  __uint_as_float(s[c / 16][(2 * c) % 32 + 1]));
        t[c] = fma2(acc, pair(kp.x, kp.y), mul2(pair(kp.z, kp.w), qsum));
      }
      if (!all) {
#pragma unroll
        for (int c = 0; c < kTok / 2; ++c) {
          float x[2];
          unpair(t[c], x[0], x[1]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int col = 2 * c + h;
            const int32_t key = key_of(range, v0 + col);
            const bool seen = ((ctl.valid[buf][col / 16] >> (2 * (col % 16))) & 1) &&
                              key <= row.pos &&
                              (p.window == 0 || key > row.pos - p.window || key < p.sinks);
            x[h] = seen ? x[h] : -INFINITY;
          }
          t[c] = pair(x[0], x[1]);
        }
      }
#pragma unroll
      for (int c = 0; c < kTok / 2; ++c) {
        float x[2];
        unpair(t[c], x[0], x[1]);
        top[c % 4] = fmaxf(top[c % 4], fmaxf(x[0], x[1]));
      }
      const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * row.a;
      int ve[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) ve[n] = ctl.vexp[buf][n];
      const int vmax = max(max(ve[0], ve[1]), max(ve[2], ve[3]));
      const bool grow = high + static_cast<float>(vmax - row.e) - row.m > kSlack;
      if (__any_sync(0xffffffffu, grow)) {
        float alpha = 1.0f;
        if (grow) {
          const float m = fmaxf(row.m, high);
          const int e = max(row.e, vmax);
          const float f = exp2_approx(row.m - m);
          row.l *= f;
          alpha = f * pow2i(max(row.e - e, -120));
          row.m = m;
          row.e = e;
        }
        __syncwarp();
        if (i > 0) {
          ok = mbar_wait(&ctl.pvdone[buf ^ 1], ((i - 1) >> 1) & 1);
          fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_load32(o, mine + L::kO + c);
            tmem_wait_load();
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
            tmem_store32(mine + L::kO + c, o);
          }
          tmem_wait_store();
        }
      }
      const uint64_t a2 = pair(row.a, row.a);
      uint32_t pr[32];
#pragma unroll
      for (int n = 0; n < 4; ++n) {  // 16 tokens: one exponent of V
        const int shift = ve[n] - row.e;
        const float ref = static_cast<float>(shift) - row.m;
        const uint64_t ref2 = pair(ref, ref);
        uint64_t sum = pair(0.0f, 0.0f);
#pragma unroll
        for (int c = 8 * n; c < 8 * n + 8; ++c) {
          float x[2];
          unpair(fma2(t[c], a2, ref2), x[0], x[1]);
          x[0] = exp2_approx(x[0]);
          x[1] = exp2_approx(x[1]);
          sum = add2(sum, pair(x[0], x[1]));
          pr[c] = pack_half2(x[0], x[1]);
        }
        float lo, hi;
        unpair(sum, lo, hi);
        row.l = fmaf(lo + hi, pow2i(min(-shift, 126)), row.l);
      }
      tmem_store32(mine + buf * kTok, pr);
      tmem_wait_store();
      fence_before();
    }
    // the rows of all four warps are written
    __syncwarp();
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (w == 0) {
      if (ok && lane == 0) {
        fence_after();
        issue_pv<D>(tmem, smem, buf, i > 0);
        commit(&ctl.pvdone[buf]);
      }
      __syncwarp();
    }
  }
  if (tiles > 0 && ok) {
    ok = mbar_wait(&ctl.pvdone[(tiles - 1) & 1], ((tiles - 1) >> 1) & 1);
    fence_after();
  }
  return ok;
}

template <typename T, int D>
__device__ __forceinline__ void write_row(const RowsParams& p, const Request& rq, int flat,
                                          int kv_head, float* part, const Row& row, bool any,
                                          uint32_t tmem) {
  using L = Layout<D>;
  const AttnParams& a = p.a;
  const int w = threadIdx.x / 32;
  const uint32_t mine = tmem + (static_cast<uint32_t>(w) << 21) + L::kO;
  const int tok = static_cast<int>(a.div_group.div(static_cast<uint32_t>(flat)));
  const bool there = tok < rq.n;
  const int head = kv_head * a.group + (flat - tok * a.group);
  const float unit = pow2i(min(max(row.e, -120), 120));
  const float f = part == nullptr ? inverse_sum(row.l) * unit : unit;
  T* dst = static_cast<T*>(a.out) + (rq.row0 + static_cast<int64_t>(tok)) * a.out_stride +
           static_cast<int64_t>(head) * D;
#pragma unroll 1
  for (int c = 0; c < D; c += 32) {
    uint32_t o[32];
    __syncwarp();
    if (any) {  // uniform: the whole CTA had tiles
      tmem_load32(o, mine + c);
      tmem_wait_load();
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) o[j] = 0;
    }
    if (there) {
      float x[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        // columns 0 ... 7 of eight are values 0, 4, 1, 5, 2, 6, 3, 7
        const int from = (j / 8) * 8 + (j % 8 < 4 ? 2 * (j % 8) : 2 * (j % 8 - 4) + 1);
        x[j] = __uint_as_float(o[from]) * f;
      }
      if (part == nullptr) {
        store_out<T, 32>(dst + c, a.out_vec != 0, x);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          reinterpret_cast<float4*>(part + 4 + c)[j] =
              make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
        }
      }
    }
  }
  if (part != nullptr && there) *reinterpret_cast<float2*>(part) = make_float2(row.m, row.l);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, D <= 128 ? 2 : 1)
kv4_rows_kernel(const __grid_constant__ RowsParams p) {
  using L = Layout<D>;
  extern __shared__ uint8_t rows_smem[];
  __shared__ Control ctl;
  const AttnParams& a = p.a;
  const int warp = threadIdx.x / 32;
  // the swizzle counts address bits: the operands start on 1024 bytes
  uint8_t* smem = rows_smem + (((smem_u32(rows_smem) + 1023) & ~1023u) - smem_u32(rows_smem));
  const int tile = blockIdx.x / p.splits, split = blockIdx.x % p.splits;
  const int kv_head = blockIdx.y, b = blockIdx.z;
  pdl_launch_dependents();
  const Request rq =
      load_request(a, b, blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0);
  const int64_t rows = static_cast<int64_t>(rq.n) * a.group;
  if (static_cast<int64_t>(tile) * kRows >= rows) return;
  const int first_row = tile * kRows;
  const int first_tok = static_cast<int>(a.div_group.div(static_cast<uint32_t>(first_row)));
  const int last_tok =
      min(rq.n - 1, static_cast<int>(a.div_group.div(static_cast<uint32_t>(first_row + kRows - 1))));
  const int32_t pos_first = rq.len - rq.n + first_tok, pos_last = rq.len - rq.n + last_tok;
  const KeyRange range = key_range(a, pos_first, pos_last);
  const int32_t all = range.count <= 0 ? 0 : (range.count + kTok - 1) / kTok;
  const int32_t t0 = static_cast<int32_t>(static_cast<int64_t>(all) * split / p.splits);
  const int32_t t1 = static_cast<int32_t>(static_cast<int64_t>(all) * (split + 1) / p.splits);

  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&ctl.tmem)),
                 "r"(L::kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 32) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl.kfull[i], 4);
      mbar_init(&ctl.vfull[i], 4);
      mbar_init(&ctl.qkdone[i], 1);
      mbar_init(&ctl.pvdone[i], 1);
    }
    mbar_init(&ctl.drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  load_rows<T, D>(a, rq, first_row, kv_head, smem, ctl);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  fence_before();
  __syncthreads();
  fence_after();

  bool ok;
  if (warp >= 4) {
    ok = bring<D>(a, range, b, kv_head, t0, t1 - t0, smem, ctl);
  } else {
    Row row;
    row.a = ctl.row[threadIdx.x].x;
    row.qsum = ctl.row[threadIdx.x].y;
    row.m = -1e30f;
    row.l = 0.0f;
    row.e = -100;
    const int flat = first_row + threadIdx.x;
    const int tok = static_cast<int>(a.div_group.div(static_cast<uint32_t>(flat)));
    row.pos = tok < rq.n ? rq.len - rq.n + tok : -1;
    ok = attend<D>(a, range, t0, t1 - t0, pos_first, pos_last, smem_u32(smem), ctl, row);
    float* part = nullptr;
    if (p.splits > 1) {
      const int64_t unit = (static_cast<int64_t>(b) * a.kv_heads + kv_head) * p.row_tiles + tile;
      part = p.part + ((unit * p.splits + split) * kRows + threadIdx.x) * (D + 4);
    }
    write_row<T, D>(p, rq, flat, kv_head, part, row, t1 > t0, ctl.tmem);
    fence_before();
  }
  if (__syncthreads_or(!ok)) {
    if (threadIdx.x == 0) {
      raise_flag(a.status, LMCB_DEVICE_FLAG_WAIT_TIMEOUT);
      commit(&ctl.drained);  // products in flight end before their memory is given back
      mbar_wait(&ctl.drained, 0);
    }
    __syncthreads();
  }
  if (warp == 0) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(ctl.tmem),
                 "r"(L::kColumns));
  }
}

// Joins the parts of units that several CTAs shared: D / 4 lanes a row.
constexpr int kJoinThreads = 256;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
kv4_rows_join_kernel(const __grid_constant__ RowsParams p) {
  constexpr int kLanes = D / 4;
  const AttnParams& a = p.a;
  const int flat = blockIdx.x * (kJoinThreads / kLanes) + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int kv_head = blockIdx.y, b = blockIdx.z;
  pdl_wait();
  const Request rq = load_request(a, b, false);
  const int tok = static_cast<int>(a.div_group.div(static_cast<uint32_t>(flat)));
  if (tok >= rq.n) return;
  const int64_t unit = (static_cast<int64_t>(b) * a.kv_heads + kv_head) * p.row_tiles + flat / kRows;
  const float* src = p.part + (unit * p.splits * kRows + flat % kRows) * (D + 4);
  float m = -1e30f, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int i = 0; i < p.splits; ++i, src += kRows * (D + 4)) {
    const float2 ml = *reinterpret_cast<const float2*>(src);
    const float4 v = *reinterpret_cast<const float4*>(src + 4 + lane * 4);
    const float nm = fmaxf(m, ml.x);
    const float fa = exp2_approx(m - nm), fb = exp2_approx(ml.x - nm);
    m = nm;
    l = l * fa + ml.y * fb;
    o.x = o.x * fa + v.x * fb;
    o.y = o.y * fa + v.y * fb;
    o.z = o.z * fa + v.z * fb;
    o.w = o.w * fa + v.w * fb;
  }
  const float inv = inverse_sum(l);
  const float x[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  store_out<T, 4>(static_cast<T*>(a.out) + (rq.row0 + static_cast<int64_t>(tok)) * a.out_stride +
                      static_cast<int64_t>(kv_head * a.group + flat - tok * a.group) * D + lane * 4,
                  a.out_vec != 0, x);
}

// CTAs that share a unit: enough that few units fill the GPU, with at least
// four tiles each.
int split_count(int64_t units, int64_t seen, int64_t head_size) {
  const int64_t slots = static_cast<int64_t>(current_sm_count()) * (head_size <= 128 ? 2 : 1);
  int64_t n = slots / units;
  const int64_t most = seen / (4 * kTok);
  if (n > most) n = most;
  return static_cast<int>(n < 1 ? 1 : n);
}

struct RowsPlan {
  int64_t row_tiles;
  int splits;
  int64_t part_bytes;
};

RowsPlan plan_rows(int64_t batch, int64_t max_query, int64_t max_len, int64_t kv_heads,
                   int64_t group, int64_t head_size, int64_t window, int64_t sinks) {
  RowsPlan pl;
  pl.row_tiles = (max_query * group + kRows - 1) / kRows;
  const int64_t units = batch * kv_heads * pl.row_tiles;
  int64_t seen = max_len;
  if (window > 0 && window + sinks + kRows < seen) seen = window + sinks + kRows;
  pl.splits = split_count(units, seen, head_size);
  pl.part_bytes = pl.splits > 1 ? units * pl.splits * kRows * (head_size + 4) * 4 : 0;
  return pl;
}

template <typename T, int D>
cudaError_t launch(const RowsParams& p, cudaStream_t stream) {
  constexpr size_t kSmem = Layout<D>::kBytes + 1024;
  cudaError_t err = ensure_smem_limit<kv4_rows_kernel<T, D>>(kSmem, kSmem);
  if (err != cudaSuccess) return err;
  const dim3 grid(static_cast<unsigned>(p.row_tiles * p.splits),
                  static_cast<unsigned>(p.a.kv_heads), static_cast<unsigned>(p.a.batch));
  kv4_rows_kernel<T, D><<<grid, kThreads, kSmem, stream>>>(p);
  err = cudaGetLastError();
  if (err != cudaSuccess || p.splits == 1) return err;
  const int64_t rows = static_cast<int64_t>(p.a.max_query) * p.a.group;
  const int per_block = kJoinThreads / (D / 4);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((rows + per_block - 1) / per_block),
                     static_cast<unsigned>(p.a.kv_heads), static_cast<unsigned>(p.a.batch));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_rows_join_kernel<T, D>, p);
}

template <typename T>
cudaError_t launch_size(const RowsParams& p, int64_t head_size, cudaStream_t stream) {
  if (head_size == 64) return launch<T, 64>(p, stream);
  if (head_size == 128) return launch<T, 128>(p, stream);
  return launch<T, 256>(p, stream);
}

}  // namespace

size_t rows_workspace(int64_t batch, int64_t max_query, int64_t max_len, int64_t kv_heads,
                      int64_t group, int64_t head_size, int64_t window, int64_t sinks) {
  return static_cast<size_t>(
      plan_rows(batch, max_query, max_len, kv_heads, group, head_size, window, sinks).part_bytes);
}

cudaError_t launch_rows(const AttnParams& a, int type, int64_t head_size, int64_t max_len,
                        void* workspace, cudaStream_t stream) {
  const RowsPlan pl = plan_rows(a.batch, a.max_query, max_len, a.kv_heads, a.group, head_size,
                                a.window, a.sinks);
  RowsParams p;
  p.a = a;
  p.splits = pl.splits;
  p.part = static_cast<float*>(workspace);
  p.row_tiles = static_cast<int32_t>(pl.row_tiles);
  return type == LMCB_DTYPE_BF16 ? launch_size<__nv_bfloat16>(p, head_size, stream)
                                 : launch_size<__half>(p, head_size, stream);
}

}  // namespace kv4
}  // namespace lmcb
