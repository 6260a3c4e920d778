// kv4_attention.cu -- attention over the paged KV cache held in 4 bits
// (layout in kv4.cuh), with an optional sliding window and first tokens that
// stay visible: the entry point, and the kernel for few query rows a KV head
// (decode steps).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q . k_j),
// over the visible keys j of a query at position i: j <= i, and with a window
// w > 0 also j > i - w or j < sinks.
//
// With k_j = zk_j + sk_j ck_j and v_j alike (ck, cv codes 0 ... 15) both
// products are taken on the codes themselves, which are exact in fp16:
//   q . k_j        = sk_j (q . ck_j) + zk_j (sum of q)
//   sum_j p_j v_j  = sum_j (p_j sv_j) cv_j + sum_j p_j zv_j
// so K is never rounded and V only as far as r_j = fp16(p_j sv_j) is; p_j is
// then taken as r_j / sv_j in the other sums too, so that a rounding of r_j
// weighs v_j - o and not the code. The code c goes into the matrix instruction
// as the fp16 bit pattern c, the subnormal c 2^-24, or shifted by four bits:
// one AND makes two operands, with no conversion (see codes for fp16 results).
// The factors are kept in range by powers of two that cancel: a query row is scaled to a largest
// element of 2^13 ... 2^14 (bf16 queries become fp16 without loss, but for
// elements below 2^-34 of the row's largest), and p_j sv_j by the largest sv
// exponent seen so far.
//
// A decode step is bound by the cache bytes (D + 8 a token and head), so the
// shape is chosen to read them once and to spend few instructions on them:
// mma.sync m16n8k16 with 16 cache tokens as its rows and 8 query rows (heads
// that share the KV head, times query tokens) as its columns. The A operand of
// q . k then wants, from lane (g, t) = (lane / 4, lane % 4), any four values of
// token g and of token g + 8 per step, the same for all lanes with that t: a
// lane holds a contiguous quarter of its tokens' code rows. The transposed A
// operand of p v wants token pairs for one value: a byte permute of two words.
// tcgen05 would want the codes expanded to 16 bits in shared memory first, four
// times the bytes read, for query tiles of 8 rows out of its 128.
//
// A CTA works on all KV heads of a token range (up to 8), so it reads whole
// rows: one warp at a time, in turn, brings the rows of a page with one bulk
// copy for K and one for V into a ring of stages, and eight warps take a head
// each (with fewer heads, several warps share a head's tokens). The tiles of all
// requests are one line that is cut into equal pieces, so ragged lengths
// leave no CTA idle; a second kernel joins requests that were cut.
//
// Measured: 96 requests of up to 16384 tokens, 8 KV heads of 128, 4 query heads
// each, bf16: 204 us, 4.0 TB/s of cache rows (0.63 of a plain copy). Issue slots
// bound it (60% used, with two CTAs an SM that is what their dependences leave):
// 313 instructions a warp for 16 tokens of a head, a third of them masks and
// shifts of codes. A warp that only brings tiles cost 222 us, loads straight from
// the pages without the ring 390. One request of 16384 tokens and one KV head
// takes 14.4 us (two launches and the join), 61 windows of 1024 tokens 29 us.
#include <climits>
#include <string>
#include <type_traits>

#include "kv4_attention.cuh"
#include "kv4_plan.h"

namespace lmcb {
namespace kv4 {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxStages = 8;
constexpr int kMaxRounds = 4;  // stage tokens / 32 at most

struct DecodeParams {
  AttnParams a;
  int32_t heads;   // KV heads a CTA works on, at most kWarps
  int32_t turns;   // warps that share a head: kWarps / heads
  int32_t groups;  // ceil(kv_heads / heads)
  int32_t stages;
  int32_t stage_tokens;  // 16 * ST * turns
  int32_t tok_stride;    // bytes a token's K (or V) row takes in a stage
  int32_t stage_bytes;
  int32_t rows;    // query rows of a unit that may exist: max_query * group
  float* part;     // [2 * CTAs][heads][8 NT][D + 4]
  int4* units;     // [groups * batch] where a unit's pieces are, for the join
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* src) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(src)[i];
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(src);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(src);
  }
}

// The tiles of all requests and head groups as one line, (group, request,
// tile), of which this CTA has [begin, end).
struct Line {
  const int32_t* prefix;  // [batch + 1] in shared memory
  int32_t batch, per_group;
  int64_t begin, end;

  // The unit of the tile at `at`, and its tile in it.
  __device__ __forceinline__ void find(int64_t at, int& group, int& b, int32_t& t) const {
    group = static_cast<int>(at / per_group);
    const int32_t in_group = static_cast<int32_t>(at - static_cast<int64_t>(group) * per_group);
    int lo = 0, hi = batch;  // prefix[lo] <= in_group < prefix[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= in_group) lo = mid; else hi = mid;
    }
    b = lo;
    t = in_group - prefix[lo];
  }
};

__device__ __forceinline__ KeyRange request_range(const AttnParams& p, const Request& r) {
  return key_range(p, r.len - r.n, r.len - 1);
}

// Tiles of a request. One without visible keys has one (empty) tile: its rows
// are written.
__device__ __forceinline__ int32_t request_tiles(const AttnParams& p, const Request& r,
                                                 int32_t stage_tokens) {
  if (r.n == 0) return 0;
  const KeyRange k = request_range(p, r);
  return k.count <= 0 ? 1 : (k.count - 1) / stage_tokens + 1;
}

// Of a unit that several CTAs work on, [first, last] with x < y, and in z the
// first one's slot (its first piece, or its second where it had others before).
__device__ __forceinline__ int4 unit_pieces(int64_t u0, int64_t u1, int64_t total, int64_t ctas) {
  if (u1 <= u0) return make_int4(0, 0, 0, 0);
  const auto cta_of = [&](int64_t x) {  // its tiles are [total c / ctas, total (c + 1) / ctas)
    int64_t c = x * ctas / total;
    while (total * (c + 1) / ctas <= x) ++c;
    return static_cast<int>(c);
  };
  const int c0 = cta_of(u0), c1 = cta_of(u1 - 1);
  return make_int4(c0, c1, 2 * c0 + (total * c0 / ctas >= u0 ? 0 : 1), 0);
}

// The CTAs that a line of `total` tiles is cut for.
__device__ __forceinline__ int64_t active_ctas(int64_t total, int ctas) {
  return total < ctas ? total : ctas;
}

// Two codes of a cache word as operands: bits 0 ... 3 of both halves of x (kHigh
// 0), or bits 4 ... 7, times 16 (kHigh 1).
//
// As they lie, c is the subnormal c 2^-24. That costs one AND, but the matrix
// unit lines up what it adds by exponents, where a subnormal counts as 2^-14,
// and cuts off 24 bits below: 2^-14 of a code. Results in bf16 do not show it.
// fp16 results do (3.6e-4 of their size at 32000 tokens), so they take kNormal:
// c on top of 1024, less 1024 and `zero`, exactly. V's zero is 8, the middle of
// the codes, so that sums over a long cache stay near their result (2.1e-4).
template <bool kNormal, int kHigh>
__device__ __forceinline__ uint32_t codes(uint32_t x, int zero) {
  const uint32_t bits = x & (kHigh ? 0x00f000f0u : 0x000f000fu);
  if constexpr (!kNormal) return bits;
  const __half2 base = __half2half2(__int2half_rn(1024 + (kHigh ? 16 : 1) * zero));
  const uint32_t up = bits | 0x64006400u;
  const __half2 c = __hsub2(*reinterpret_cast<const __half2*>(&up), base);
  return *reinterpret_cast<const uint32_t*>(&c);
}

// Query operands of a unit: B fragments of q . k, and per column the factors
//   s = acc * a * sk + zk * b  (log2 units).
template <int D, int NT>
struct Query {
  uint32_t frag[NT][D / 16][2];
  float a[NT][2], b[NT][2];
  int32_t pos[NT][2];  // position of the column's query token, -1: no such row
};

// Codes of kNormal are counted in ones, else in 2^-24.
template <bool kNormal>
__host__ __device__ constexpr float code_unit() {
  return kNormal ? 1.0f : 16777216.0f;
}

template <typename T, int D, int NT, bool kNormal>
__device__ __forceinline__ void load_unit_query(const AttnParams& p, const Request& rq,
                                                int kv_head, Query<D, NT>& q) {
  const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  constexpr int N = D / 4;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int flat = n * 8 + g;
    const int tok = static_cast<int>(p.div_group.div(static_cast<uint32_t>(flat)));
    const int head = kv_head * p.group + (flat - tok * p.group);
    float x[N];
    if (tok < rq.n) {
      load_query<T, N>(static_cast<const T*>(p.q) +
                           (rq.row0 + static_cast<int64_t>(tok)) * p.q_stride +
                           static_cast<int64_t>(head) * D + t * N,
                       p.q_vec != 0, x);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = 0.0f;
    }
    float big = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) big = fmaxf(big, fabsf(x[i]));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    // 2^e <= big < 2^(e + 1); zero and the smallest rows as 2^-100
    const int e = min(max(((__float_as_int(big) >> 23) & 255) - 127, -100), 100);
    const float up = pow2i(13 - e), down = pow2i(e - 13);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = __half2float(__float2half_rn(x[i] * up));
      sum += x[i];
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    // Word w of a code row meets values 8 w + j and 8 w + j + 4 in its operand
    // j; operands of odd j are codes shifted by four bits, times 16.
#pragma unroll
    for (int w = 0; w < N / 8; ++w)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = j % 2 ? 0.0625f : 1.0f;
        q.frag[n][2 * w + j / 2][j % 2] = pack_half2(x[8 * w + j] * f, x[8 * w + j + 4] * f);
      }
    const float unit = down * p.scale_log2;
    // columns 2 t and 2 t + 1 of a score tile are the rows of lanes g = 2 t, 2 t + 1
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int src = (2 * t + c) * 4;
      q.a[n][c] = __shfl_sync(0xffffffffu, unit, src) * code_unit<kNormal>();
      q.b[n][c] = __shfl_sync(0xffffffffu, unit * sum, src);
      const int ps = tok < rq.n ? rq.len - rq.n + tok : -1;
      q.pos[n][c] = __shfl_sync(0xffffffffu, ps, src);
    }
  }
}

// One warp's running softmax over the tiles it has taken, for 8 * NT query
// rows of one KV head. Lane (g, t) holds, for query columns 2 t and 2 t + 1 of
// each group of eight: the running maximum m (log2), its own tokens' parts of
// the sum l and of z = sum p zv, and the output's values g * D / 8 ... of
// sum p sv cv: even values in acc[.][.][0, 1], odd ones, times 16, in [2, 3].
template <int D, int NT>
struct Running {
  float acc[D / 16][NT][4];
  float m[NT][2], l[NT][2], z[NT][2];
  int vexp;

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][n][c] = 0.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) m[n][c] = -INFINITY, l[n][c] = 0.0f, z[n][c] = 0.0f;
    vexp = 0;
  }
  // r = p sv 2^(29 - vexp), vexp the largest biased fp16 exponent of the sv so
  // far: below 2^15 for p <= 1.
  __device__ __forceinline__ float value_factor() const { return pow2i(29 - vexp); }
  template <bool kNormal>
  __device__ __forceinline__ float value_unit() const {
    return pow2i(vexp - 29) * code_unit<kNormal>();
  }
};

// Tokens are the rows of a score tile in the order sigma: its rows 2 i and
// 2 i + 1 are tokens 2 or 6 apart (mod 8), and so are what a lane's loads of K
// meet in one shared-memory pass; loads of V meet tokens 0 ... 3. Rows of the
// common size of 544 bytes (8 heads of 128) then never share a bank.
__device__ __forceinline__ int sigma(int i) { return i % 2 ? ((i / 2 + 2) & 3) + 4 : i / 2; }

// ST * 16 tokens of a stage, the warp's turn of them. kAll: every token is
// there and seen by every query row.
template <int D, int NT, int ST, bool kAll, bool kNormal>
__device__ __forceinline__ void take_tile(const DecodeParams& p, const uint8_t* stage,
                                          const uint32_t* valid, int first, int code_off,
                                          int par_off, const KeyRange& range, int32_t v0,
                                          bool mask, const Query<D, NT>& q, Running<D, NT>& st) {
  constexpr int KW = D / 32;  // code words of K a lane holds of a token
  constexpr int VW = D / 64;  // code words of V
  const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const uint8_t* vstage = stage + p.stage_tokens * p.tok_stride;

  float s[ST][NT][4];
  uint32_t vpar[ST][2];
  float top[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = -INFINITY;
  uint32_t vmax = 0;
#pragma unroll
  for (int u = 0; u < ST; ++u) {
    uint32_t kw[2][KW], kpar[2];
    bool there[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int tok = first + u * 16 + i * 8 + sigma(g);
      const uint8_t* row = stage + tok * p.tok_stride;
      load_words<KW>(kw[i], row + code_off + t * (D / 8));
      kpar[i] = *reinterpret_cast<const uint32_t*>(row + par_off);
      vpar[u][i] = *reinterpret_cast<const uint32_t*>(vstage + tok * p.tok_stride + par_off);
      there[i] = true;
      if constexpr (!kAll) {
        // What is not there may hold anything. A V row whose parameters are no finite
        // numbers (kv4_store writes none) gives NaN, by its K, to the queries that see
        // it, and nothing to the others.
        there[i] = (valid[tok / 32] >> (tok % 32)) & 1;
        if (!there[i]) kpar[i] = vpar[u][i] = 0;
        if ((vpar[u][i] & 0x7c00u) == 0x7c00u || (vpar[u][i] & 0x7c000000u) == 0x7c000000u) {
          kpar[i] = 0x7e00u;
          vpar[u][i] = 0;
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[u][n][c] = 0.0f;
#pragma unroll
    for (int w = 0; w < KW; ++w) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t x0 = kw[0][w] >> (8 * j), x1 = kw[1][w] >> (8 * j);
        const uint32_t a0 = codes<kNormal, 0>(x0, 0), a1 = codes<kNormal, 0>(x1, 0);
        const uint32_t a2 = codes<kNormal, 1>(x0, 0), a3 = codes<kNormal, 1>(x1, 0);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_f16(s[u][n], a0, a1, a2, a3, q.frag[n][2 * w + j][0], q.frag[n][2 * w + j][1]);
        }
      }
    }
    vmax = max(vmax, max((vpar[u][0] >> 10) & 31u, (vpar[u][1] >> 10) & 31u));
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int i = c >> 1, col = c & 1;
        float v = fmaf(s[u][n][c] * q.a[n][col], half_lo(kpar[i]), half_hi(kpar[i]) * q.b[n][col]);
        if constexpr (!kAll) {
          bool seen = there[i];
          if (mask) {
            const int32_t key = key_of(range, v0 + first + u * 16 + i * 8 + sigma(g));
            const int32_t ps = q.pos[n][col];
            seen = seen && key <= ps && (key > window_end(p.a, ps) || key < p.a.sinks);
          }
          v = seen ? v : -INFINITY;
        }
        s[u][n][c] = v;
        top[n][col] = fmaxf(top[n][col], v);
      }
  }

  // The largest value exponent rescales the sums when it grows.
  const int vexp = static_cast<int>(__reduce_max_sync(0xffffffffu, vmax));
  float rescale = 1.0f;
  if (vexp > st.vexp) {
    rescale = pow2i(st.vexp - vexp);
    st.vexp = vexp;
  }
  const float vfac = st.value_factor();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float grow[2];
#pragma unroll
    for (int col = 0; col < 2; ++col) {
      float m = top[n][col];
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
      m = fmaxf(st.m[n][col], m);
      const float ref = m == -INFINITY ? 0.0f : m;
      grow[col] = exp2_approx(st.m[n][col] - ref);  // 0 for the first keys
      st.m[n][col] = m;
      st.l[n][col] *= grow[col];
      st.z[n][col] *= grow[col];
      top[n][col] = ref;
      grow[col] *= rescale;
    }
    if (__any_sync(0xffffffffu, grow[0] != 1.0f || grow[1] != 1.0f)) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        st.acc[i][n][0] *= grow[0];
        st.acc[i][n][1] *= grow[1];
        st.acc[i][n][2] *= grow[0];
        st.acc[i][n][3] *= grow[1];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < ST; ++u) {
    float sf[2], back[2], zv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sf[i] = half_lo(vpar[u][i]) * vfac;
      zv[i] = half_hi(vpar[u][i]);
      if constexpr (kNormal) zv[i] = fmaf(8.0f, half_lo(vpar[u][i]), zv[i]);
      // r is a normal fp16 number for p down to 2^-14 only where sf >= 1;
      // below, its rounding says nothing about p
      back[i] = sf[i] >= 1.0f ? rcp_approx(sf[i]) : 0.0f;
    }
    uint32_t pf[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float e[2];
#pragma unroll
        for (int col = 0; col < 2; ++col) e[col] = exp2_approx(s[u][n][2 * i + col] - top[n][col]);
        const uint32_t r = pack_half2(e[0] * sf[i], e[1] * sf[i]);
        if (back[i] != 0.0f) {
          e[0] = half_lo(r) * back[i];
          e[1] = half_hi(r) * back[i];
        }
#pragma unroll
        for (int col = 0; col < 2; ++col) {
          st.l[n][col] += e[col];
          st.z[n][col] = fmaf(e[col], zv[i], st.z[n][col]);
        }
        pf[n][i] = transpose_8x8(r);
      }
    // Values: rows of the A operand are two of the lane's D / 8 values, columns
    // its four tokens.
    uint32_t vw[4][VW];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int tok = first + u * 16 + (i / 2) * 8 + sigma(2 * t + (i & 1));
      load_words<VW>(vw[i], vstage + tok * p.tok_stride + code_off + g * (D / 16));
    }
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      const uint32_t lo0 = __byte_perm(vw[0][w], vw[1][w], 0x5410);
      const uint32_t hi0 = __byte_perm(vw[0][w], vw[1][w], 0x7632);
      const uint32_t lo1 = __byte_perm(vw[2][w], vw[3][w], 0x5410);
      const uint32_t hi1 = __byte_perm(vw[2][w], vw[3][w], 0x7632);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t x0 = (i < 2 ? lo0 : hi0) >> (8 * (i & 1));
        const uint32_t x1 = (i < 2 ? lo1 : hi1) >> (8 * (i & 1));
        const uint32_t a0 = codes<kNormal, 0>(x0, 8), a1 = codes<kNormal, 1>(x0, 8);
        const uint32_t a2 = codes<kNormal, 0>(x1, 8), a3 = codes<kNormal, 1>(x1, 8);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_f16(st.acc[4 * w + i][n], a0, a1, a2, a3, pf[n][0], pf[n][1]);
        }
      }
    }
  }
}

// Warps that share a head have a place each in shared memory, and all threads
// add them up: bytes for 8 * nt rows (66 KB at most; one warp a head: nothing to
// merge). Adding to one place in turn took less room and more time: 34.8 us
// against 20.5 for one request of 512 tokens, one KV head of 256.
__host__ __device__ constexpr int64_t merge_bytes(int heads, int nt, int64_t head_size) {
  return kWarps / heads == 1 ? 0 : kWarps * 8 * nt * (head_size + 2) * 4;
}

// Where a query row's output, or this CTA's part of it, goes.
template <int D, int NT>
__device__ __forceinline__ float* part_row(const DecodeParams& p, int slot, int head, int col) {
  return p.part + ((static_cast<int64_t>(slot) * p.heads + head) * (8 * NT) + col) * (D + 4);
}

// The rows of a unit out of one warp's registers (one warp a head).
template <typename T, int D, int NT>
__device__ __forceinline__ void write_rows(const DecodeParams& p, const Request& rq, int kv_head,
                                           int head, int slot, const Running<D, NT>& st) {
  constexpr int N = D / 8;
  const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const float unit = st.template value_unit<std::is_same<T, __half>::value>();
  const float unit16 = unit * 0.0625f;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int col = n * 8 + 2 * t + c;
      const int tok = static_cast<int>(p.a.div_group.div(static_cast<uint32_t>(col)));
      if (tok >= rq.n) continue;
      const float f = slot < 0 ? inverse_sum(st.l[n][c]) : 1.0f;
      float x[N];
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        x[2 * i] = fmaf(st.acc[i][n][c], unit, st.z[n][c]) * f;
        x[2 * i + 1] = fmaf(st.acc[i][n][c + 2], unit16, st.z[n][c]) * f;
      }
      if (slot < 0) {
        store_out<T, N>(static_cast<T*>(p.a.out) +
                            (rq.row0 + static_cast<int64_t>(tok)) * p.a.out_stride +
                            static_cast<int64_t>(kv_head * p.a.group + col - tok * p.a.group) * D +
                            g * N,
                        p.a.out_vec != 0, x);
      } else {
        float* dst = part_row<D, NT>(p, slot, head, col);
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
          reinterpret_cast<float4*>(dst + 4 + g * N)[i] =
              make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        }
        if (g == 0) *reinterpret_cast<float2*>(dst) = make_float2(st.m[n][c], st.l[n][c]);
      }
    }
}

// The same where several warps share a head.
template <typename T, int D, int NT>
__device__ __forceinline__ void merge_rows(const DecodeParams& p, const Request& rq, int group,
                                           int slot, const Running<D, NT>& st, float* smem) {
  constexpr int R = 8 * NT;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const int heads = p.heads, turns = p.turns;
  const int head = warp % heads, turn = warp / heads;
  const bool working = turn < turns;
  const int places = turns * heads, place = turn * heads + head;
  float* s_o = smem;                   // [places][R][D]
  float* s_l = s_o + places * R * D;   // [places][R]
  float* s_m = s_l + places * R;       // [turns][heads][R]
  if (working && g == 0) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) s_m[(turn * heads + head) * R + n * 8 + 2 * t + c] = st.m[n][c];
  }
  __syncthreads();
  const float unit = st.template value_unit<std::is_same<T, __half>::value>();
  const float unit16 = unit * 0.0625f;
  float f[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float m = -INFINITY;
      for (int w = 0; w < turns; ++w) m = fmaxf(m, s_m[(w * heads + head) * R + n * 8 + 2 * t + c]);
      f[n][c] = m == -INFINITY ? 0.0f : exp2_approx(st.m[n][c] - m);
    }
  if (working) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = n * 8 + 2 * t + c;
        if (col >= p.rows) continue;
        float* o = s_o + (place * R + col) * D + g * (D / 8);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          *reinterpret_cast<float2*>(o + 2 * i) =
              make_float2(fmaf(st.acc[i][n][c], unit, st.z[n][c]) * f[n][c],
                          fmaf(st.acc[i][n][c + 2], unit16, st.z[n][c]) * f[n][c]);
        }
        if (g == 0) s_l[place * R + col] = st.l[n][c] * f[n][c];
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * p.rows * (D / 4); i += kThreads) {
    const int row = i / (D / 4), e = (i % (D / 4)) * 4;
    const int h = row / p.rows, col = row % p.rows;
    const int kv_head = group * heads + h;
    const int tok = static_cast<int>(p.a.div_group.div(static_cast<uint32_t>(col)));
    if (tok >= rq.n || kv_head >= p.a.kv_heads) continue;
    float4 v = *reinterpret_cast<const float4*>(s_o + (h * R + col) * D + e);
    float l = s_l[h * R + col];
    for (int w = 1; w < turns; ++w) {
      const int other = w * heads + h;
      const float4 u = *reinterpret_cast<const float4*>(s_o + (other * R + col) * D + e);
      v.x += u.x;
      v.y += u.y;
      v.z += u.z;
      v.w += u.w;
      l += s_l[other * R + col];
    }
    if (slot < 0) {
      const float inv = inverse_sum(l);
      const float x[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
      store_out<T, 4>(static_cast<T*>(p.a.out) +
                          (rq.row0 + static_cast<int64_t>(tok)) * p.a.out_stride +
                          static_cast<int64_t>(kv_head * p.a.group + col - tok * p.a.group) * D + e,
                      p.a.out_vec != 0, x);
    } else {
      float* dst = part_row<D, NT>(p, slot, h, col);
      *reinterpret_cast<float4*>(dst + 4 + e) = v;
      if (e == 0) {
        float m = -INFINITY;
        for (int w = 0; w < turns; ++w) m = fmaxf(m, s_m[(w * heads + h) * R + col]);
        *reinterpret_cast<float2*>(dst) = make_float2(m, l);
      }
    }
  }
  __syncthreads();  // the buffer is used again by the next unit
}

// Shared state of the ring. Tile j of this CTA goes into stage j % stages.
struct Ring {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint32_t valid[kMaxStages][kMaxRounds];  // tokens that are there, a bit each
  uint32_t issued;                         // tiles brought so far
};

// One warp brings tile `j`: it finds the rows of the tile's tokens, waits for
// the stage and starts the copies.
__device__ __forceinline__ bool produce(const DecodeParams& p, const Line& line, uint32_t j,
                                        uint8_t* data, Ring& ring, int half_size) {
  const AttnParams& a = p.a;
  const int lane = threadIdx.x % 32;
  const int rounds = (p.stage_tokens + 31) / 32;
  const uint32_t row_bytes = static_cast<uint32_t>(a.row_words) * 4;
  const uint32_t stage = j % p.stages, turn = j / p.stages;
  int group, b;
  int32_t t;
  line.find(line.begin + j, group, b, t);
  const Request rq = load_request(a, b, false);
  const KeyRange range = request_range(a, rq);
  const int32_t* table = a.table + static_cast<int64_t>(b) * a.table_stride;
  int32_t row[kMaxRounds];
  uint32_t there[kMaxRounds];
  uint32_t count = 0;
#pragma unroll
  for (int r = 0; r < kMaxRounds; ++r) {
    row[r] = -1;
    there[r] = 0;
    if (r < rounds) {
      const int tok = r * 32 + lane;
      if (tok < p.stage_tokens) row[r] = row_of(a, table, range, t * p.stage_tokens + tok);
      there[r] = __ballot_sync(0xffffffffu, row[r] >= 0);
      count += __popc(there[r]);
    }
  }
  // what is copied of a row: all of it, or this group's codes and the 16-byte
  // pieces that hold its parameters
  const int heads = min(p.heads, a.kv_heads - group * p.heads);
  const uint32_t code_at = static_cast<uint32_t>(group * p.heads * half_size);
  const uint32_t code_bytes = static_cast<uint32_t>(heads * half_size);
  const uint32_t par = static_cast<uint32_t>(a.kv_heads * half_size + group * p.heads * 4);
  const uint32_t par_at = par & ~15u;
  const uint32_t par_bytes = ((par + heads * 4 + 15) & ~15u) - par_at;
  const uint32_t tok_bytes = 2 * (p.groups == 1 ? row_bytes : code_bytes + par_bytes);
  if (turn > 0 && !warp_wait(&ring.empty[stage], (turn - 1) & 1)) return false;
  uint64_t* full = &ring.full[stage];
  if (lane == 0) {
#pragma unroll
    for (int r = 0; r < kMaxRounds; ++r) {
      if (r < rounds) ring.valid[stage][r] = there[r];
    }
    atomicMax(&ring.issued, j + 1);
    mbar_arrive_expect_tx(full, count * tok_bytes);
  }
  __syncwarp();
  const uint8_t* k_rows = reinterpret_cast<const uint8_t*>(a.cache);
  const uint8_t* v_rows = k_rows + a.half_words * 4;
  uint8_t* dst = data + stage * p.stage_bytes;
  const uint32_t v_off = static_cast<uint32_t>(p.stage_tokens * p.tok_stride);
#pragma unroll
  for (int r = 0; r < kMaxRounds; ++r) {
    if (r >= rounds) continue;
    uint8_t* to = dst + (r * 32 + lane) * p.tok_stride;
    const int64_t from = static_cast<int64_t>(row[r]) * row_bytes;
    if (p.groups == 1) {
      // runs of rows that follow one another in the cache: one copy each. Row 0
      // does not follow a token that is not there (-1).
      const int32_t prev = __shfl_up_sync(0xffffffffu, row[r], 1);
      const bool start = row[r] >= 0 && (lane == 0 || prev < 0 || row[r] != prev + 1);
      const uint32_t stops = __ballot_sync(0xffffffffu, start) | ~there[r];
      if (start) {
        const uint32_t above = lane == 31 ? 0 : stops >> (lane + 1);
        const uint32_t n = above ? __ffs(above) : 32 - lane;
        bulk_load(to, k_rows + from, n * row_bytes, full);
        bulk_load(to + v_off, v_rows + from, n * row_bytes, full);
      }
    } else if (row[r] >= 0) {
      bulk_load(to, k_rows + from + code_at, code_bytes, full);
      bulk_load(to + p.heads * half_size, k_rows + from + par_at, par_bytes, full);
      bulk_load(to + v_off, v_rows + from + code_at, code_bytes, full);
      bulk_load(to + v_off + p.heads * half_size, v_rows + from + par_at, par_bytes, full);
    }
  }
  return true;
}

// The tiles of this CTA. In step j every warp works on tile j, and one of them,
// in turn, first brings the tile that takes the place of tile j - 1: the warps
// may drift a tile apart, and no warp stays behind for being the producer.
template <typename T, int D, int NT, int ST>
__device__ __forceinline__ bool run_line(const DecodeParams& p, const Line& line, uint8_t* data,
                                         Ring& ring, float* merge) {
  const AttnParams& a = p.a;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int head = warp % p.heads, turn = warp / p.heads;
  const int first = turn * ST * 16;  // this warp's tokens of a stage
  const uint32_t count = static_cast<uint32_t>(line.end - line.begin);
  constexpr bool kNormal = std::is_same<T, __half>::value;
  bool ok = true;
  if (warp < p.stages && static_cast<uint32_t>(warp) < count) {
    produce(p, line, warp, data, ring, D / 2);
  }
  __syncthreads();
  uint32_t stage = 0, phase = 0;
  Query<D, NT> q;
  Running<D, NT> st;
  for (uint32_t j = 0; j < count;) {
    int group, b;
    int32_t t;
    line.find(line.begin + j, group, b, t);
    const int32_t tiles = line.prefix[b + 1] - line.prefix[b];
    const uint32_t steps = min(static_cast<uint32_t>(tiles - t), count - j);
    // a whole unit goes to the output; a piece is this CTA's first or its last
    const int slot = steps == static_cast<uint32_t>(tiles)
                         ? -1
                         : 2 * static_cast<int>(blockIdx.x) + (j == 0 ? 0 : 1);
    const Request rq = load_request(a, b, false);
    const KeyRange range = request_range(a, rq);
    const int kv_head = group * p.heads + head;
    const bool working = turn < p.turns && kv_head < a.kv_heads;
    const bool mask = rq.n > 1;
    const int code_off = head * (D / 2);
    const int par_off = p.groups == 1
                            ? a.kv_heads * (D / 2) + head * 4
                            : p.heads * (D / 2) +
                                  ((a.kv_heads * (D / 2) + group * p.heads * 4) & 15) + head * 4;
    if (working) load_unit_query<T, D, NT, kNormal>(a, rq, kv_head, q);
    st.reset();
    for (const uint32_t j_end = j + steps; j < j_end; ++j, ++t) {
      if (j > 0 && j % kWarps == static_cast<uint32_t>(warp) && j - 1 + p.stages < count && ok) {
        ok = produce(p, line, j - 1 + p.stages, data, ring, D / 2);
      }
      ok = ok && warp_wait(&ring.full[stage], phase);
      if (working && ok) {
        const uint8_t* at = data + stage * p.stage_bytes;
        bool all = !mask;
#pragma unroll
        for (int u = 0; u < ST; ++u) {
          const int tok = first + u * 16;
          all = all && ((ring.valid[stage][tok / 32] >> (tok % 32)) & 0xffffu) == 0xffffu;
        }
        if (all) {
          take_tile<D, NT, ST, true, kNormal>(p, at, ring.valid[stage], first, code_off, par_off, range,
                                     t * p.stage_tokens, false, q, st);
        } else {
          take_tile<D, NT, ST, false, kNormal>(p, at, ring.valid[stage], first, code_off, par_off, range,
                                      t * p.stage_tokens, mask, q, st);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ring.empty[stage]);
      if (++stage == static_cast<uint32_t>(p.stages)) stage = 0, phase ^= 1;
    }
    // the warp's own sums over its tokens
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          st.l[n][c] += __shfl_xor_sync(0xffffffffu, st.l[n][c], o);
          st.z[n][c] += __shfl_xor_sync(0xffffffffu, st.z[n][c], o);
        }
      }
    if (p.turns == 1) {
      if (working) write_rows<T, D, NT>(p, rq, kv_head, head, slot, st);
    } else {
      merge_rows<T, D, NT>(p, rq, group, slot, st, merge);
    }
  }
  return ok;
}

// CTAs of this kernel that fit an SM: two where their registers do.
template <int D, int NT>
constexpr int ctas_per_sm() {
  return D * NT <= 128 ? 2 : 1;
}

template <typename T, int D, int NT, int ST>
__global__ void __launch_bounds__(kThreads, ctas_per_sm<D, NT>())
kv4_decode_kernel(const __grid_constant__ DecodeParams p) {
  extern __shared__ __align__(16) uint8_t decode_smem[];
  __shared__ Ring ring;
  __shared__ int32_t s_warp[kWarps];
  float* merge = reinterpret_cast<float*>(decode_smem + p.stages * p.stage_bytes);
  int32_t* prefix = reinterpret_cast<int32_t*>(reinterpret_cast<uint8_t*>(merge) +
                                               merge_bytes(p.heads, NT, D));
  const AttnParams& a = p.a;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  pdl_launch_dependents();  // the joining kernel may take its place; it waits for this one
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&ring.full[s], 1);
      mbar_init(&ring.empty[s], kWarps);
    }
    ring.issued = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  int32_t base = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    int32_t own = 0;
    if (b < a.batch) own = request_tiles(a, load_request(a, b, blockIdx.x == 0), p.stage_tokens);
    int32_t sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 31) s_warp[warp] = sum;
    __syncthreads();
    int32_t before = base;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s_warp[w];
      base += s_warp[w];
    }
    if (b < a.batch) prefix[b] = before + sum - own;
    __syncthreads();
  }
  if (threadIdx.x == 0) prefix[a.batch] = base;
  __syncthreads();
  const int64_t total = static_cast<int64_t>(base) * p.groups;
  const int64_t n = active_ctas(total, gridDim.x);
  // the last CTA has no more tiles than the others: it tells the join
  if (blockIdx.x == gridDim.x - 1) {
    for (int i = threadIdx.x; i < a.batch * p.groups; i += kThreads) {
      const int group = i / a.batch, b = i % a.batch;
      const int64_t before = static_cast<int64_t>(group) * base;
      p.units[i] = unit_pieces(before + prefix[b], before + prefix[b + 1], total, n);
    }
  }
  if (blockIdx.x >= n) return;
  Line line;
  line.prefix = prefix;
  line.batch = a.batch;
  line.per_group = base;
  line.begin = total * blockIdx.x / n;
  line.end = total * (blockIdx.x + 1) / n;
  const bool ok = run_line<T, D, NT, ST>(p, line, decode_smem, ring, merge);
  if (__syncthreads_or(!ok)) {
    if (threadIdx.x == 0) {
      raise_flag(a.status, LMCB_DEVICE_FLAG_WAIT_TIMEOUT);
      // copies in flight write to this CTA's shared memory: they land first
      const uint32_t issued = ring.issued;
      for (uint32_t j = issued > static_cast<uint32_t>(p.stages) ? issued - p.stages : 0;
           j < issued; ++j) {
        mbar_wait(&ring.full[j % p.stages], (j / p.stages) & 1);
      }
    }
    __syncthreads();
  }
}

// Joins the pieces of every unit that more than one CTA worked on: one query
// row for `parts` groups of D / 4 lanes, which share its pieces, always in the
// same order. A lane has kPieces pieces on their way at once.
constexpr int kJoinThreads = 512;
constexpr int kPieces = 8;

struct Merged {
  float m, l;
  float4 o;

  __device__ __forceinline__ void add(float pm, float pl, const float4& v) {
    const float nm = fmaxf(m, pm);
    const float ref = nm == -INFINITY ? 0.0f : nm;
    const float fa = exp2_approx(m - ref), fb = exp2_approx(pm - ref);
    m = nm;
    l = l * fa + pl * fb;
    o.x = o.x * fa + v.x * fb;
    o.y = o.y * fa + v.y * fb;
    o.z = o.z * fa + v.z * fb;
    o.w = o.w * fa + v.w * fb;
  }
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kJoinThreads)
kv4_join_kernel(const __grid_constant__ DecodeParams p, const int parts) {
  constexpr int kLanes = D / 4;
  __shared__ float4 s_o[kJoinThreads];
  __shared__ float2 s_ml[kJoinThreads / kLanes];
  const AttnParams& a = p.a;
  const int who = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const int part = who % parts;
  const int row = blockIdx.x * (blockDim.x / kLanes / parts) + who / parts;
  const int b = blockIdx.y;
  const int kv_head = row / p.rows, col = row % p.rows;
  const int group = kv_head / p.heads, h = kv_head % p.heads;
  const int tok = static_cast<int>(a.div_group.div(static_cast<uint32_t>(col)));
  pdl_wait();
  Merged sum{-INFINITY, 0.0f, make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
  bool cut = false;
  Request rq{};
  if (kv_head < a.kv_heads) {
    const int4 unit = p.units[group * a.batch + b];
    rq = load_request(a, b, false);
    cut = unit.x < unit.y && tok < rq.n;  // else its CTA has written it
    if (cut) {
      for (int c = unit.x + part; c <= unit.y; c += parts * kPieces) {
        float2 ml[kPieces];
        float4 v[kPieces];
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
          const int at = c + k * parts;
          if (at <= unit.y) {
            const float* src = part_row<D, NT>(p, at == unit.x ? unit.z : 2 * at, h, col);
            ml[k] = *reinterpret_cast<const float2*>(src);
            v[k] = *reinterpret_cast<const float4*>(src + 4 + lane * 4);
          }
        }
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
          if (c + k * parts <= unit.y) sum.add(ml[k].x, ml[k].y, v[k]);
        }
      }
    }
  }
  if (parts > 1) {
    s_o[threadIdx.x] = sum.o;
    if (lane == 0) s_ml[who] = make_float2(sum.m, sum.l);
    __syncthreads();
    if (part == 0) {
      for (int i = 1; i < parts; ++i) {
        const float2 ml = s_ml[who + i];
        sum.add(ml.x, ml.y, s_o[threadIdx.x + i * kLanes]);
      }
    }
  }
  if (!cut || part != 0) return;
  const float inv = inverse_sum(sum.l);
  const float x[4] = {sum.o.x * inv, sum.o.y * inv, sum.o.z * inv, sum.o.w * inv};
  store_out<T, 4>(static_cast<T*>(a.out) + (rq.row0 + static_cast<int64_t>(tok)) * a.out_stride +
                      static_cast<int64_t>(kv_head * a.group + col - tok * a.group) * D + lane * 4,
                  a.out_vec != 0, x);
}

// ---------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------

// How a decode call is cut up; the same for the workspace size and the launch.
struct Plan {
  int nt, st;
  int heads, turns, groups;
  int stage_tokens, tok_stride, stage_bytes, stages;
  int ctas;
  int64_t part_bytes, unit_bytes;
};

Plan make_plan(int64_t batch, int64_t max_query, int64_t max_len, int64_t kv_heads, int64_t group,
               int64_t head_size, int64_t window, int64_t sinks) {
  Plan pl;
  pl.nt = max_query * group <= 8 ? 1 : 2;
  pl.groups = static_cast<int>((kv_heads + kWarps - 1) / kWarps);
  pl.heads = static_cast<int>((kv_heads + pl.groups - 1) / pl.groups);
  pl.turns = kWarps / pl.heads;
  pl.st = pl.turns == 1 && head_size * pl.nt <= 128 ? 2 : 1;
  pl.stage_tokens = 16 * pl.st * pl.turns;
  pl.tok_stride = static_cast<int>(
      pl.groups == 1 ? kv4_row_words(kv_heads, head_size) * 4
                     : pl.heads * (head_size / 2) + (pl.heads * 4 + 12 + 15) / 16 * 16);
  pl.stage_bytes = 2 * pl.stage_tokens * pl.tok_stride;
  const int per_sm = head_size * pl.nt <= 128 ? 2 : 1;
  const int64_t merge = merge_bytes(pl.heads, pl.nt, head_size);
  const int64_t room = 220 * 1024 / per_sm - merge - (batch + 1) * 4 - 1024;
  pl.stages = static_cast<int>(room / pl.stage_bytes);
  if (pl.stages > kMaxStages) pl.stages = kMaxStages;
  if (pl.stages < 2) pl.stages = 2;
  int64_t seen = max_len;
  if (window > 0 && window + sinks + max_query < seen) seen = window + sinks + max_query;
  int64_t tiles = batch * pl.groups * ((seen + pl.stage_tokens - 1) / pl.stage_tokens);
  const int64_t most = static_cast<int64_t>(current_sm_count()) * per_sm;
  if (tiles > most) tiles = most;
  pl.ctas = static_cast<int>(tiles < 1 ? 1 : tiles);
  pl.unit_bytes = batch * pl.groups * 16;
  pl.part_bytes = int64_t(2) * pl.ctas * pl.heads * pl.nt * 8 * (head_size + 4) * 4;
  return pl;
}

template <typename T, int D, int NT, int ST>
cudaError_t launch(const DecodeParams& p, const Plan& pl, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(p.stages) * p.stage_bytes + merge_bytes(p.heads, NT, D) +
                      (static_cast<size_t>(p.a.batch) + 1) * 4;
  cudaError_t err = ensure_smem_limit<kv4_decode_kernel<T, D, NT, ST>>(smem, 224 * 1024);
  if (err != cudaSuccess) return err;
  kv4_decode_kernel<T, D, NT, ST><<<pl.ctas, kThreads, smem, stream>>>(p);
  err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  // Few long requests: the pieces of a row are shared by several lane groups, so
  // that each has no more than it takes at once.
  int parts = 1;
  const int64_t pieces = pl.ctas / (static_cast<int64_t>(p.a.batch) * p.groups);
  while (parts < kJoinThreads / (D / 4) && pieces > parts * kPieces) parts *= 2;
  const int threads = parts * (D / 4) > 256 ? kJoinThreads : 256;
  const int per_block = threads / (D / 4) / parts;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((p.a.kv_heads * p.rows + per_block - 1) / per_block),
                     static_cast<unsigned>(p.a.batch));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_join_kernel<T, D, NT>, p, parts);
}

template <typename T>
cudaError_t launch_size(const DecodeParams& p, const Plan& pl, int64_t head_size,
                        cudaStream_t stream) {
  if (head_size == 64) {
    if (pl.nt == 1) {
      return pl.st == 2 ? launch<T, 64, 1, 2>(p, pl, stream) : launch<T, 64, 1, 1>(p, pl, stream);
    }
    return pl.st == 2 ? launch<T, 64, 2, 2>(p, pl, stream) : launch<T, 64, 2, 1>(p, pl, stream);
  }
  if (head_size == 128) {
    if (pl.nt == 1) {
      return pl.st == 2 ? launch<T, 128, 1, 2>(p, pl, stream) : launch<T, 128, 1, 1>(p, pl, stream);
    }
    return launch<T, 128, 2, 1>(p, pl, stream);
  }
  return launch<T, 256, 1, 1>(p, pl, stream);  // 8 rows at most, see is_decode
}

// The decode kernel takes up to 16 query rows a KV head, and with heads of 256,
// whose second eight rows leave it too few registers, up to 8. The time of the
// other kernel hardly depends on the rows up to 128. Measured, decode / rows: 64
// requests of 8192 tokens, 8 KV heads of 128: 8 rows 150 / 612 us, 16 rows 317
// ... 354 / 616; one request of 32768, one head: 16 rows 37 / 59. Heads of 256, 64
// requests of 8192, 2 KV heads: 8 rows 117 / 244, 16 rows 262 / 244; 4 requests of
// 4096: 25 / 35 and 41 / 35; 16 of 8192 with 8 KV heads: 100 / 246 and 242 / 246.
bool is_decode(int64_t max_query, int64_t group, int64_t head_size) {
  return max_query * group <= (head_size > 128 ? 8 : 16);
}

constexpr int64_t kMaxBatch = 4096;  // tiles before each request, in shared memory
constexpr int64_t kMaxKeys = INT_MAX - 1024;  // of a table row: a tile's end is an int32

int check_shape(const std::string& who, int64_t batch, int64_t max_query, int64_t max_len,
                int64_t kv_heads, int64_t query_heads, int64_t head_size, int64_t window,
                int64_t sinks) {
  if (head_size != 64 && head_size != 128 && head_size != 256) {
    return fail(LMCB_ERR_INVALID_ARGUMENT, who + ": head_size must be 64, 128 or 256.");
  }
  if (batch < 0 || max_query < 0 || max_len < 0 || kv_heads <= 0 || query_heads <= 0 ||
      query_heads % kv_heads != 0 || query_heads > 4096 || window < 0 || sinks < 0 ||
      window > INT_MAX || sinks > INT_MAX || max_len > INT_MAX ||
      max_query > (INT_MAX / 2) / query_heads) {
    return fail(LMCB_ERR_INVALID_ARGUMENT, who + ": invalid shape.");
  }
  if (batch > kMaxBatch) {
    return fail(LMCB_ERR_CAPACITY,
                who + ": at most " + std::to_string(kMaxBatch) + " requests a call.");
  }
  return LMCB_OK;
}

}  // namespace
}  // namespace kv4
}  // namespace lmcb

extern "C" {

int lmcb_kv4_attention_workspace(int64_t batch, int64_t maxQueryLen, int64_t maxSeqLen,
                                 int64_t numKvHeads, int64_t numQueryHeads, int64_t headSize,
                                 int64_t window, int64_t sinks, size_t* bytesOut) {
  using namespace lmcb;
  clear_error();
  const std::string who = "kv4_attention_workspace";
  if (bytesOut == nullptr) return fail(LMCB_ERR_INVALID_ARGUMENT, who + ": bytesOut is NULL.");
  const int st = kv4::check_shape(who, batch, maxQueryLen, maxSeqLen, numKvHeads, numQueryHeads,
                                  headSize, window, sinks);
  if (st != LMCB_OK) return st;
  const int64_t group = numQueryHeads / numKvHeads;
  *bytesOut = 0;
  if (batch == 0 || maxQueryLen == 0) return LMCB_OK;
  if (kv4::is_decode(maxQueryLen, group, headSize)) {
    const kv4::Plan pl = kv4::make_plan(batch, maxQueryLen, maxSeqLen, numKvHeads, group, headSize,
                                        window, sinks);
    *bytesOut = static_cast<size_t>(pl.part_bytes + pl.unit_bytes);
  } else {
    *bytesOut = kv4::rows_workspace(batch, maxQueryLen, maxSeqLen, numKvHeads, group, headSize,
                                    window, sinks);
  }
  return LMCB_OK;
}

int lmcb_kv4_attention(const void* query, int type, int64_t queryTokenStride, int64_t numQueryRows,
                       const int32_t* kvCache, int64_t numBlocks, int64_t blockSize,
                       const int32_t* blockTable, int64_t tableStride, int64_t tableCols,
                       const int32_t* seqLens, const int32_t* queryStart, int64_t batch,
                       int64_t maxQueryLen, int64_t maxSeqLen, int64_t numKvHeads,
                       int64_t numQueryHeads, int64_t headSize, double scale, int64_t window,
                       int64_t sinks, void* out, int64_t outTokenStride, void* workspace,
                       size_t workspaceBytes, void* stream) {
  using namespace lmcb;
  clear_error();
  const std::string who = "kv4_attention";
  if (type != LMCB_DTYPE_BF16 && type != LMCB_DTYPE_FP16) {
    return fail(LMCB_ERR_UNSUPPORTED_DTYPE, who + ": queries must be bf16 or fp16.");
  }
  int st = kv4::check_shape(who, batch, maxQueryLen, maxSeqLen, numKvHeads, numQueryHeads,
                            headSize, window, sinks);
  if (st != LMCB_OK) return st;
  if (numQueryRows < 0 || numQueryRows > INT_MAX / 2 || numBlocks < 0 || blockSize <= 0 ||
      (numBlocks > 0 && blockSize > INT_MAX / numBlocks) || tableCols < 0 ||
      tableStride < tableCols || (tableCols > 0 && blockSize > kv4::kMaxKeys / tableCols) ||
      queryTokenStride < numQueryHeads * headSize || outTokenStride < numQueryHeads * headSize ||
      (queryStart == nullptr && (maxQueryLen < 1 || numQueryRows < batch))) {
    return fail(LMCB_ERR_INVALID_ARGUMENT, who + ": invalid shape.");
  }
  // tiles of 16 keys of all requests are counted in an int32
  if (batch > 0 && (tableCols * blockSize + 15) / 16 > INT_MAX / batch) {
    return fail(LMCB_ERR_CAPACITY, who + ": too many keys in one call.");
  }
  if (batch == 0 || numQueryRows == 0 || maxQueryLen == 0) return LMCB_OK;
  if (query == nullptr || out == nullptr || seqLens == nullptr ||
      (tableCols > 0 && blockTable == nullptr) || (numBlocks > 0 && kvCache == nullptr)) {
    return fail(LMCB_ERR_INVALID_ARGUMENT, who + ": NULL pointer.");
  }
  if (reinterpret_cast<uintptr_t>(kvCache) % 16 != 0) {
    return fail(LMCB_ERR_INVALID_ARGUMENT, who + ": the cache must be 16-byte aligned.");
  }
  size_t need = 0;
  st = lmcb_kv4_attention_workspace(batch, maxQueryLen, maxSeqLen, numKvHeads, numQueryHeads,
                                    headSize, window, sinks, &need);
  if (st != LMCB_OK) return st;
  if (need > 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 ||
                   workspaceBytes < need)) {
    return fail(LMCB_ERR_CAPACITY, who + ": the workspace is too small or not aligned.");
  }
  kv4::AttnParams a;
  a.q = query;
  a.q_vec = reinterpret_cast<uintptr_t>(query) % 16 == 0 && queryTokenStride % 8 == 0;
  a.q_stride = queryTokenStride;
  a.out = out;
  a.out_vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && outTokenStride % 8 == 0;
  a.out_stride = outTokenStride;
  a.cache = kvCache;
  a.row_words = kv4_row_words(numKvHeads, headSize);
  a.half_words = numBlocks * blockSize * a.row_words;
  a.num_blocks = static_cast<int32_t>(numBlocks);
  a.div_block = FastDiv(static_cast<uint32_t>(blockSize));
  a.table = blockTable;
  a.table_stride = tableStride;
  a.table_cols = static_cast<int32_t>(tableCols);
  a.seq_lens = seqLens;
  a.query_start = queryStart;
  a.num_rows = static_cast<int32_t>(numQueryRows);
  a.batch = static_cast<int32_t>(batch);
  a.max_query = static_cast<int32_t>(maxQueryLen);
  a.kv_heads = static_cast<int32_t>(numKvHeads);
  a.group = static_cast<int32_t>(numQueryHeads / numKvHeads);
  a.div_group = FastDiv(static_cast<uint32_t>(a.group));
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  a.window = static_cast<int32_t>(window);
  a.sinks = static_cast<int32_t>(sinks);
  a.status = device_status_ptr();
  if (a.status == nullptr) return LMCB_ERR_CUDA;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t err;
  if (kv4::is_decode(maxQueryLen, a.group, headSize)) {
    const kv4::Plan pl = kv4::make_plan(batch, maxQueryLen, maxSeqLen, numKvHeads, a.group,
                                        headSize, window, sinks);
    kv4::DecodeParams p;
    p.a = a;
    p.heads = pl.heads;
    p.turns = pl.turns;
    p.groups = pl.groups;
    p.stages = pl.stages;
    p.stage_tokens = pl.stage_tokens;
    p.tok_stride = pl.tok_stride;
    p.stage_bytes = pl.stage_bytes;
    p.rows = static_cast<int32_t>(maxQueryLen * a.group);
    p.part = static_cast<float*>(workspace);
    p.units = reinterpret_cast<int4*>(static_cast<char*>(workspace) + pl.part_bytes);
    err = type == LMCB_DTYPE_BF16 ? kv4::launch_size<__nv_bfloat16>(p, pl, headSize, s)
                                  : kv4::launch_size<__half>(p, pl, headSize, s);
  } else {
    err = kv4::launch_rows(a, type, headSize, maxSeqLen, workspace, s);
  }
  if (err != cudaSuccess) return cuda_fail(err, who.c_str());
  return LMCB_OK;
}

}  // extern "C"
