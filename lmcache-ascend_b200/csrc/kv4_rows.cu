// kv4_rows.cu -- attention over the 4-bit paged cache (kv4_attention.cu has the
// definition) for many query rows a KV head: the suffix of a request computed
// over its retrieved prefix, or several tokens checked at once.
//
// A unit is 128 query rows (query tokens times the heads that share a KV head)
// of one request and KV head; its rows are the lanes of the tensor memory. With
// a tile of 64 cache tokens:
//   S = Q Ck^T     tcgen05.mma 128 x 64 x D, Ck the K codes,
//   t = S sk + zk (sum of q), p = exp2(t a + e - m),
//   O += P V'      tcgen05.mma 128 x D x 64, P from tensor memory.
// The K codes are exact as in the decode kernel (the fp16 bit patterns c and
// 16 c, c 2^-24; Q's odd elements carry the 1/16), so a logit is an fp32 sum of
// exact products. V is made fp16 on the way, v 2^-e with the largest of 16 tokens
// near the end of fp16's range, and P takes the 2^e. Both are rounded to fp16
// once; for bf16 results that is an eighth of their own rounding. fp16 results
// are rounded no more coarsely than V and P: they take P as two fp16 numbers, p
// and what its rounding left, in a second product, which leaves V's rounding
// alone (error against 64 bits 2.9e-4 of the result's size, 2.1e-4 is the result's
// own, and 3.4e-4 with one number).
//   What a row does not see, or gives no weight, costs it nothing as long as its
// values are within 2^21 of the others': m is the row's own, from the p 2^e of
// the keys that it sees, so the largest P lies between 2^7 and 2^15 and numbers
// down to 2^-21 of 2^7 are normal; V is normal down to 2^-28 of the largest of
// its 16 tokens. Further apart, values in the 16 of a larger one lose bits (2^24
// apart, those that bf16 does not have). Exact codes as V, with s in P and z in a
// sum of its own, would not: they took 1280 us where this takes 1100, for what
// every pair of tokens then has to load and add. More head for P costs time too:
// with 2^9 instead of 2^7 more tiles are taken again, 5% of the time.
//
// A CTA has two such units (one for D = 256), 256 query rows, which share the
// tiles. Per tile the tensor core needs 1024 cycles for them, the exponentials
// 1024 (16 a cycle), the rest of softmax and the expanding of codes about as
// many issue slots, and shared memory as many accesses of 128 bytes; so the
// work is laid out to keep all four going at once:
//  - four warps bring the codes from the pages and expand them into a ring of
//    stages (128-byte swizzle; a lane's 16-byte pieces of 4 tokens x 2 halves of
//    a panel hit all banks), ahead of the products;
//  - one thread issues products, Q K^T a tile ahead of P V, into one of two S (P,
//    from tensor memory, takes the place of its S);
//  - eight warps a unit compute softmax. A lane has 2 rows x 16 tokens, not one
//    row x 32 tokens, and so loads half as many of the tokens' scales.
// O stays in tensor memory; it is rescaled only when a row's P outgrows 2^15, and
// its m then leaves room for 2^8 more.
//
// Measured: 4 suffixes of up to 1024 tokens behind prefixes of up to 16384, 64
// query heads over 8 of 128, bf16: 1091 us, 736 TFLOP/s (0.44 of a plain bf16
// product). By its counters no one unit bounds it: 58% of the issue slots, 37% of
// the tensor pipe. Nor does one of its parts: with K and V not written at all it
// takes 970 us, without the exponentials 1092, without both 905. What is left is
// the chain of waits from S through softmax to P V, of which a CTA has two units'
// worth under way. Q K^T with 64 columns takes 46 cycles of the tensor core where
// 32 would do (128 columns: 64.5); two S of 128 columns a unit do not fit beside its
// O, one would, without Q K^T running ahead in its unit. On the way: one unit a CTA
// 1856 us, two 1513, eight softmax warps a unit instead of four 1455, one elected
// lane that issues products instead of a branch by lane 1191, pairs of fp32 1150, one
// thread for the whole loop of products and a reference a row 1091; eight warps that
// bring instead of four 1380 (fewer registers for softmax). The compiler's schedule
// of softmax alone moved it by 8% both ways between forms with the same instructions.
#include <climits>
#include <type_traits>

#include "kv4_attention.cuh"
#include "kv4_plan.h"

namespace lmcb {
namespace kv4 {
namespace {

constexpr int kRows = 128;  // query rows of a unit
constexpr int kTok = 64;    // cache tokens of a tile
// log2 of a row's largest P: what it may grow to before O is rescaled (fp16 ends
// at 2^16), and what it is then.
constexpr float kMost = 15.0f;
constexpr float kHead = 7.0f;

struct RowsParams {
  AttnParams a;
  int32_t splits;  // CTAs that share a unit's tiles
  float* part;        // [CTA's rows][splits][rows][D + 4]
  int32_t row_tiles;  // CTAs a request's rows may take
};

// Packed pairs of fp32: one instruction for two values.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
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

// 16 lanes x 64 columns: lane (g, t) of the warp has, of each 8 columns, columns
// 2 t and 2 t + 1 of lanes g (r[4 n], r[4 n + 1]) and g + 8 (r[4 n + 2, 3]).
__device__ __forceinline__ void tmem_load_rows(uint32_t (&r)[32], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}

// 16 lanes x 32 columns: lane (g, t) has, of each 4 columns, column t of lanes g
// (r[2 n]) and g + 8 (r[2 n + 1]).
__device__ __forceinline__ void tmem_store_rows(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// The layout of the first, 32 columns.
__device__ __forceinline__ void tmem_load_rows(uint32_t (&r)[16], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_store_rows_f32(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// The registers of a load are there after its wait: they pass through it.
__device__ __forceinline__ void tmem_wait_load(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait_load(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                 "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
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

// True in one lane of a converged warp. The compiler knows that what such a
// branch guards runs in one thread, and issues its products without asking
// again for each of them.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

// Shared-memory operand descriptor: 128-byte swizzle (8 rows of 128 bytes),
// 1024 bytes from one group of 8 rows to the next and `lead` bytes from one
// 64-element panel to the next (operands whose rows run along K). The low word
// holds the address and `lead`; adding bytes / 16 to it moves the operand.
__device__ __forceinline__ uint32_t operand_low(uint32_t addr, uint32_t lead) {
  return ((addr >> 4) & 0x3fff) | (((lead >> 4) & 0x3fff) << 16);
}
__device__ __forceinline__ uint64_t operand(uint32_t low) {
  constexpr uint32_t kHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
  return static_cast<uint64_t>(low) | (static_cast<uint64_t>(kHigh) << 32);
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
  static constexpr int kUnits = D <= 128 ? 2 : 1;  // of a CTA
  static constexpr int kPanels = D / 64;           // of 64 values, 128 bytes a token
  static constexpr int kPanel = kTok * 128;
  static constexpr int kV = kPanels * kPanel;      // V behind K in a stage
  static constexpr int kStage = 2 * kV;
  static constexpr int kStages = D == 64 ? 6 : D == 128 ? 4 : 2;
  static constexpr int kQPanel = kRows * 128;
  static constexpr int kQ = kPanels * kQPanel;     // a unit's rows, in front of the stages
  static constexpr int kBytes = kUnits * kQ + kStages * kStage;
  // Warps: eight of softmax a unit, four that bring, one that issues products;
  // three more fill its warpgroup. With two units the 80 registers a thread that
  // 768 threads start with are dealt out anew by warpgroup:
  // 16 * 96 + 4 * 64 + 4 * 32 = 24 * 80.
  static constexpr int kBring = kUnits * 8, kIssue = kBring + 4;
  static constexpr int kThreads = (kIssue + 4) * 32;
  // Tensor memory of a unit: two S (P takes an S's first half), then O.
  static constexpr uint32_t kUnit = 256;
  static constexpr uint32_t kO = 2 * kTok;
  static constexpr uint32_t kColumns = 512;
};

constexpr int kMaxStages = 6;

struct Control {
  uint64_t full[kMaxStages], free[kMaxStages];
  uint64_t sready[2][2], pready[2][2], pvdone[2];  // by unit and S
  uint64_t drained;
  float4 kpar[kMaxStages][kTok / 2];  // tokens 2 i, 2 i + 1: (sk, sk, zk, zk)
  uint32_t valid[kMaxStages][4];      // two bits a token, 16 tokens each
  float4 vexp[kMaxStages][4];         // of 16 tokens: e, twice, and 2^-e
  float2 row[2 * kRows];              // a, sum of q in its unit; at the end m, l
  uint32_t tmem;
};

// Byte offset of 16-byte piece `piece` of row `r` in a 128-byte swizzled panel.
__device__ __forceinline__ uint32_t swizzled(uint32_t r, uint32_t piece) {
  return r * 128 + ((piece ^ (r & 7)) << 4);
}

// A thread's query row, scaled to fp16, into shared memory.
template <typename T, int D>
__device__ __forceinline__ void load_row(const AttnParams& p, const Request& rq, int flat,
                                         int kv_head, int r, uint8_t* smem, float2& factors) {
  using L = Layout<D>;
  const int tok = static_cast<int>(p.div_group.div(static_cast<uint32_t>(flat)));
  const int head = kv_head * p.group + (flat - tok * p.group);
  const bool there = tok < rq.n;
  const T* src = static_cast<const T*>(p.q) + (rq.row0 + static_cast<int64_t>(tok)) * p.q_stride +
                 static_cast<int64_t>(head) * D;
  float big = 0.0f;
  if (there) {
#pragma unroll 4
    for (int i = 0; i < D / 8; ++i) {
      float x[8];
      load_query<T, 8>(src + 8 * i, p.q_vec != 0, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf(x[j]));
    }
  }
  const int e = min(max(((__float_as_int(big) >> 23) & 255) - 127, -100), 100);
  // the sign of the scale goes into the rows, so that the largest t is the
  // largest logit
  const float up = p.scale_log2 < 0.0f ? -pow2i(13 - e) : pow2i(13 - e);
  float sum = 0.0f;
#pragma unroll 4
  for (int i = 0; i < D / 8; ++i) {
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
    *reinterpret_cast<uint4*>(smem + (i / 8) * L::kQPanel + swizzled(r, i % 8)) = out;
  }
  // codes count 2^-24, or 1 (expand_k); a is never zero, so that a key that is
  // not seen stays at -inf
  constexpr float kUnit = std::is_same<T, __half>::value ? 1.0f : 16777216.0f;
  factors = make_float2(fmaxf(fabsf(p.scale_log2) * pow2i(e - 13) * kUnit, 1.2e-38f),
                        sum / kUnit);
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

// Loads that stay where they are written: a tile ahead of their use.
__device__ __forceinline__ uint4 load_ahead4(const int32_t* src) {
  uint4 v;
  asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(src));
  return v;
}
__device__ __forceinline__ uint32_t load_ahead(const int32_t* src) {
  uint32_t v;
  asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(src));
  return v;
}

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
      c.k[i] = load_ahead4(k + 8 * i);
      c.v[i] = load_ahead4(v + 8 * i);
    }
    c.kpar = load_ahead(par + at);
    c.vpar = load_ahead(par + p.half_words + at);
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

// Codes as normal numbers, exactly: on top of 1024, less 1024.
__device__ __forceinline__ __half2 normal(uint32_t bits) {
  return __hsub2(as_half2(bits | 0x64006400u), __half2half2(__ushort_as_half(0x6400)));
}

// Eight values of V in the order 0, 4, 1, 5, 2, 6, 3, 7: s c + z, or s16 16 c + z,
// rounded once.
__device__ __forceinline__ uint4 expand_v(uint32_t w, __half2 s, __half2 s16, __half2 z) {
  const uint32_t x = w >> 8;
  return make_uint4(half2_bits(__hfma2(normal(w & 0x000f000fu), s, z)),
                    half2_bits(__hfma2(normal(w & 0x00f000f0u), s16, z)),
                    half2_bits(__hfma2(normal(x & 0x000f000fu), s, z)),
                    half2_bits(__hfma2(normal(x & 0x00f000f0u), s16, z)));
}

// Eight codes of K in the same order, the odd ones times 16, as their bits lie:
// c 2^-24. fp16 results take normal numbers: the matrix unit cuts off bits of sums
// of subnormals (codes in the decode kernel).
template <bool kNormal>
__device__ __forceinline__ uint4 expand_k(uint32_t w) {
  const uint32_t x = w >> 8;
  uint32_t r[4] = {w & 0x000f000fu, w & 0x00f000f0u, x & 0x000f000fu, x & 0x00f000f0u};
  if constexpr (kNormal) {
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = half2_bits(normal(r[j]));
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

template <int D, bool kNormal>
__device__ __forceinline__ bool bring(const AttnParams& p, const KeyRange& range, int b,
                                      int kv_head, int32_t t0, int32_t tiles, uint8_t* smem,
                                      Control& ctl) {
  using L = Layout<D>;
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32 - L::kBring;
  const int tok = w * 16 + lane / 2;
  const int32_t* table = p.table + static_cast<int64_t>(b) * p.table_stride;
  const int32_t* k_head = p.cache + static_cast<int64_t>(kv_head) * (D / 8);
  const int32_t* par = p.cache + static_cast<int64_t>(p.kv_heads) * (D / 8) + kv_head;
  const int32_t size = static_cast<int32_t>(p.div_block.d);
  // The page of this lane's token of tile i, unchecked: nothing waits for it
  // before the tile's turn.
  const auto page_of = [&](int32_t i) {
    const int32_t v = (t0 + i) * kTok + tok;
    if (i >= tiles || v >= range.count) return -1;
    return static_cast<int32_t>(
        load_ahead(table + p.div_block.div(static_cast<uint32_t>(key_of(range, v)))));
  };
  const auto row_in = [&](int32_t i, int32_t page) {
    const int32_t v = (t0 + i) * kTok + tok;
    if (i >= tiles || v >= range.count) return -1;
    if (page < 0 || page >= p.num_blocks) {
      raise_flag(p.status, LMCB_DEVICE_FLAG_SLOT_OUT_OF_RANGE);
      return -1;
    }
    const int32_t key = key_of(range, v);
    return page * size +
           (key - static_cast<int32_t>(p.div_block.div(static_cast<uint32_t>(key))) * size);
  };
  // codes of the next tile and the page of the one after it are on their way
  // while a tile is expanded
  Codes<D> next;
  int32_t page = page_of(0);
  fetch<D>(p, k_head, par, row_in(0, page), lane, next);
  page = page_of(1);
  int stage = 0;
  uint32_t phase = 1;  // parity of the stage's last use
  for (int32_t i = 0; i < tiles; ++i) {
    const Codes<D> c = next;
    fetch<D>(p, k_head, par, row_in(i + 1, page), lane, next);
    page = page_of(i + 2);
    // e places the largest value of these 16 tokens between 2^14 and 2^15. A row
    // whose parameters are no finite numbers (kv4_store writes none) gives NaN, by
    // its K, to the queries that see it, and nothing to its neighbours.
    float s = half_lo(c.vpar), z = half_hi(c.vpar);
    const bool finite = fabsf(s) <= 65504.0f && fabsf(z) <= 65504.0f;
    if (!finite) s = z = 0.0f;
    const float most = fmaxf(fabsf(z), fabsf(fmaf(15.0f, s, z)));
    const int e = static_cast<int>(__reduce_max_sync(
                      0xffffffffu, max((__float_as_uint(most) >> 23) & 255u, 80u))) - 141;
    const float down = pow2i(-e);
    const __half2 vs = __half2half2(__float2half_rn(s * down));
    const __half2 vs16 = __half2half2(__float2half_rn(s * down * 0.0625f));
    const __half2 vz = __half2half2(__float2half_rn(z * down));
    const uint32_t there = __ballot_sync(0xffffffffu, c.there);
    if (i >= L::kStages && !warp_wait(&ctl.free[stage], phase)) return false;
    uint8_t* k = smem + stage * L::kStage;
    const uint32_t piece = (lane % 2) * 4;
#pragma unroll
    for (int n = 0; n < L::kPanels; ++n) {
      const uint32_t kw[4] = {c.k[n].x, c.k[n].y, c.k[n].z, c.k[n].w};
      const uint32_t vw[4] = {c.v[n].x, c.v[n].y, c.v[n].z, c.v[n].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint8_t* to = k + n * L::kPanel + swizzled(tok, piece + j);
        *reinterpret_cast<uint4*>(to) = expand_k<kNormal>(kw[j]);
        *reinterpret_cast<uint4*>(to + L::kV) = expand_v(vw[j], vs, vs16, vz);
      }
    }
    if (lane % 2 == 0) {
      float* to = reinterpret_cast<float*>(&ctl.kpar[stage][tok / 2]) + tok % 2;
      to[0] = finite ? half_lo(c.kpar) : __int_as_float(0x7fffffff);
      to[2] = half_hi(c.kpar);
    }
    if (lane == 0) {
      ctl.valid[stage][w] = there;
      ctl.vexp[stage][w] =
          make_float4(static_cast<float>(e), static_cast<float>(e), down, down);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl.full[stage]);
    if (++stage == L::kStages) stage = 0, phase ^= 1;
  }
  return true;
}

// ---------------------------------------------------------------------------
// The thread that issues the products
// ---------------------------------------------------------------------------

template <int D>
__device__ __forceinline__ void issue_qk(uint32_t s, uint32_t rows, uint32_t stage) {
  using L = Layout<D>;
  const uint32_t q = operand_low(rows, 0), k = operand_low(stage, 0);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    mma_ss(s, operand(q + ((i / 4) * L::kQPanel + (i % 4) * 32) / 16),
           operand(k + ((i / 4) * L::kPanel + (i % 4) * 32) / 16), instruction(kTok, false), i > 0);
  }
}

template <int D>
__device__ __forceinline__ void issue_pv(uint32_t o, uint32_t p, uint32_t stage, bool add) {
  using L = Layout<D>;
  const uint32_t v = operand_low(stage + L::kV, L::kPanel);
#pragma unroll
  for (int i = 0; i < kTok / 16; ++i) {
    mma_ts(o, p + i * 8, operand(v + i * 16 * 128 / 16), instruction(D, true), add || i > 0);
  }
}

// Q K^T runs ahead of P V: softmax finds the next S when it is done with one.
// Only products into the same accumulator keep their order by themselves. So
// Q K^T of tile j waits until the P V of tile j - 2, whose P lay in the same S,
// has ended; with two units, each one's P V is waited for while the other's
// runs.
template <int D, bool kTwo>
struct Issuer {
  using L = Layout<D>;
  uint32_t tmem, rows, stages;
  int units;
  Control& ctl;

  __device__ __forceinline__ bool qk(int u, int32_t j) const {
    const int stage = j % L::kStages, buf = j & 1;
    if (!mbar_wait(&ctl.full[stage], (j / L::kStages) & 1)) return false;
    if (j >= 2 && !mbar_wait(&ctl.pvdone[u], j & 1)) return false;
    fence_after();
    issue_qk<D>(tmem + u * L::kUnit + buf * kTok, rows + u * L::kQ, stages + stage * L::kStage);
    commit(&ctl.sready[u][buf]);
    return true;
  }

  __device__ __forceinline__ bool pv(int u, int32_t j) const {
    const int stage = j % L::kStages, buf = j & 1;
    if (!mbar_wait(&ctl.pready[u][buf], (j >> 1) & 1)) return false;
    fence_after();
    const uint32_t unit = tmem + u * L::kUnit, p = unit + buf * kTok;
    issue_pv<D>(unit + L::kO, p, stages + stage * L::kStage, j > 0);
    if constexpr (kTwo) {
      issue_pv<D>(unit + L::kO, p + kTok / 2, stages + stage * L::kStage, true);
    }
    commit(&ctl.pvdone[u]);
    if (u == units - 1) commit(&ctl.free[stage]);
    return true;
  }

  __device__ __forceinline__ bool run(int32_t tiles) const {
    if (tiles == 0) return true;
    if (!qk(0, 0)) return false;
    if (units == 1) {
      for (int32_t j = 0; j < tiles; ++j) {
        if (j + 1 < tiles && !qk(0, j + 1)) return false;
        if (!pv(0, j)) return false;
      }
      return true;
    }
    if (!qk(1, 0) || (tiles > 1 && !qk(0, 1))) return false;
    for (int32_t j = 0; j < tiles; ++j) {
      if (!pv(0, j)) return false;
      if (j + 1 < tiles && !qk(1, j + 1)) return false;
      if (!pv(1, j)) return false;
      if (j + 2 < tiles && !qk(0, j + 2)) return false;
    }
    return true;
  }
};

// ---------------------------------------------------------------------------
// The warps that have the query rows
// ---------------------------------------------------------------------------

// A thread's part of a tile: lane (g, t) has rows g and g + 8 of its warp's 16,
// and of each the tokens 8 n + 2 t and 8 n + 2 t + 1.
struct Part {
  float a[2];
  uint64_t qsum[2];     // rows' factors, the second twice
  float m[2];           // references (log2)
  float top[2];         // largest t a + e of this tile
  float l[2];           // sums of this tile, in units of 2^m
  int32_t hi[2];        // last key seen, as a virtual token
};

// S into P and the rows' largest t a + e and sums.
template <bool kAll, bool kTwo>
__device__ __forceinline__ void softmax_tile(const AttnParams& p, uint32_t s_cols,
                                             const ulonglong2* kpar, const uint32_t* valid,
                                             const ulonglong2* vexp, int32_t v0, Part& part,
                                             uint32_t (&pr)[16], uint32_t (&rest)[16]) {
  const int t4 = threadIdx.x % 4;
  uint32_t s[32];
  tmem_load_rows(s, s_cols);
  uint64_t back_ref[2], a2[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    back_ref[k] = pair(-part.m[k], -part.m[k]);
    a2[k] = pair(part.a[k], part.a[k]);
    part.top[k] = -INFINITY;
    part.l[k] = 0.0f;
  }
  tmem_wait_load(s);
#pragma unroll
  for (int n = 0; n < 4; ++n) {  // 16 tokens: one exponent of V
    const ulonglong2 ve = vexp[n];
    const float back = unpair(ve.y).x;  // to the units of l
    const ulonglong2 kp[2] = {kpar[8 * n + t4], kpar[8 * n + 4 + t4]};  // (sk, sk), (zk, zk)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint64_t ref = add2(ve.x, back_ref[k]);
      float2 x[2];
      float top = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = 8 * n + 4 * h + 2 * k;
        uint64_t t2 = fma2(pair(__uint_as_float(s[at]), __uint_as_float(s[at + 1])), kp[h].x,
                           mul2(kp[h].y, part.qsum[k]));
        float2 t = unpair(t2);
        if constexpr (!kAll) {
          const int col = 16 * n + 8 * h + 2 * t4, v = v0 + col;
          const uint32_t there = valid[n] >> (2 * (col % 16));
          const auto seen = [&](int32_t at_v, uint32_t bit) {
            return at_v <= part.hi[k] &&
                   (at_v > window_end(p, part.hi[k]) || at_v < p.sinks) && (bit & 1);
          };
          t.x = seen(v, there) ? t.x : -INFINITY;
          t.y = seen(v + 1, there >> 2) ? t.y : -INFINITY;
          t2 = pair(t.x, t.y);
        }
        top = fmaxf(top, fmaxf(t.x, t.y));
        x[h] = unpair(fma2(t2, a2[k], ref));
        x[h].x = exp2_approx(x[h].x);
        x[h].y = exp2_approx(x[h].y);
        const uint32_t r = pack_half2(x[h].x, x[h].y);
        pr[4 * n + 2 * h + k] = r;
        if constexpr (kTwo) {
          rest[4 * n + 2 * h + k] = pack_half2(x[h].x - half_lo(r), x[h].y - half_hi(r));
        }
      }
      const float2 sum = unpair(add2(pair(x[0].x, x[0].y), pair(x[1].x, x[1].y)));
      part.l[k] = fmaf(sum.x + sum.y, back, part.l[k]);
      part.top[k] = fmaxf(part.top[k], fmaf(top, part.a[k], unpair(ve.x).x));
    }
  }
}

// A warp has 16 of a unit's rows: warps w and w + 4 have those of tensor memory
// lanes 32 w ..., 16 each. l and O are in units of 2^m, a row's own. P is taken
// with the references that are there; only a tile that outgrows them (the first
// one, and few after it) is taken again, with new ones. So nothing waits for a
// tile's maximum, and a thread never holds more than the tile's S.
template <int D, bool kTwo>
__device__ __forceinline__ bool attend(const AttnParams& p, const KeyRange& range, int32_t t0,
                                       int32_t tiles, int32_t pos_first, int32_t pos_last,
                                       const Request& rq, int first_row, Control& ctl) {
  using L = Layout<D>;
  const int warp = threadIdx.x / 32, unit = warp / 8;
  const int lane = threadIdx.x % 32, g = lane / 4, t4 = lane % 4;
  const int lanes = (warp % 4) * 32 + (warp / 4 % 2) * 16;  // of tensor memory
  const int warp_row = unit * kRows + lanes;                // of the CTA's rows
  const uint32_t mine = ctl.tmem + unit * L::kUnit + (static_cast<uint32_t>(lanes) << 16);
  // Visible keys of a row at position i, as virtual tokens (KeyRange): v <= hi,
  // and v > window_end(hi) or v < sinks.
  const int32_t to_v = range.head - range.first;
  const int32_t hi_first = pos_first + to_v, hi_last = pos_last + to_v;
  Part part;
  float l[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int row = warp_row + g + 8 * k;
    const float2 f = ctl.row[row];
    part.a[k] = f.x;
    part.qsum[k] = pair(f.y, f.y);
    part.m[k] = -1e30f;
    l[k] = 0.0f;
    const int tok = static_cast<int>(p.div_group.div(static_cast<uint32_t>(first_row + row)));
    part.hi[k] = tok < rq.n ? rq.len - rq.n + tok + to_v : -1;
  }
  bool ok = true;
  int stage = 0;
  uint32_t phase = 0;
  for (int32_t i = 0; i < tiles; ++i) {
    if (!warp_wait(&ctl.full[stage], phase) ||
        !warp_wait(&ctl.sready[unit][i & 1], (i >> 1) & 1)) {
      ok = false;
      break;
    }
    fence_after();
    const uint32_t s_cols = mine + (i & 1) * kTok;
    // is every key of the tile there and seen by every row?
    const int32_t v0 = (t0 + i) * kTok;
    const uint4 valid = *reinterpret_cast<const uint4*>(ctl.valid[stage]);
    const bool all = (valid.x & valid.y & valid.z & valid.w) == 0xffffffffu &&
                     v0 + kTok - 1 <= hi_first &&
                     (v0 > window_end(p, hi_last) || v0 + kTok - 1 < p.sinks);
    const ulonglong2* kpar = reinterpret_cast<const ulonglong2*>(ctl.kpar[stage]);
    const ulonglong2* vexp = reinterpret_cast<const ulonglong2*>(ctl.vexp[stage]);
    uint32_t pr[16], rest[16];
    for (;;) {
      if (all) {
        softmax_tile<true, kTwo>(p, s_cols, kpar, ctl.valid[stage], vexp, v0, part, pr, rest);
      } else {
        softmax_tile<false, kTwo>(p, s_cols, kpar, ctl.valid[stage], vexp, v0, part, pr, rest);
      }
      if (!__any_sync(0xffffffffu, part.top[0] - part.m[0] > kMost ||
                                       part.top[1] - part.m[1] > kMost)) {
        break;
      }
      float alpha[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float top = part.top[k];
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float m_new = top - part.m[k] > kMost ? top - kHead : part.m[k];
        alpha[k] = exp2_approx(part.m[k] - m_new);
        part.m[k] = m_new;
        l[k] *= alpha[k];
      }
      if (i > 0) {
        ok = warp_wait(&ctl.pvdone[unit], (i - 1) & 1) && ok;
        fence_after();
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[16];
          tmem_load_rows(o, mine + L::kO + c);
          tmem_wait_load(o);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha[j / 2 % 2]);
          }
          tmem_store_rows_f32(mine + L::kO + c, o);
        }
      }
    }
    tmem_store_rows(s_cols, pr);
    if constexpr (kTwo) tmem_store_rows(s_cols + kTok / 2, rest);
#pragma unroll
    for (int k = 0; k < 2; ++k) l[k] += part.l[k];
    tmem_wait_store();
    fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl.pready[unit][i & 1]);
    if (++stage == L::kStages) stage = 0, phase ^= 1;
  }
  if (tiles > 0 && ok) {
    ok = warp_wait(&ctl.pvdone[unit], (tiles - 1) & 1);  // the last product
    fence_after();
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    l[k] += __shfl_xor_sync(0xffffffffu, l[k], 1);
    l[k] += __shfl_xor_sync(0xffffffffu, l[k], 2);
    if (t4 == 0) {
      ctl.row[warp_row + g + 8 * k] = make_float2(part.m[k], l[k]);
    }
  }
  return ok;
}

template <typename T, int D>
__device__ __forceinline__ void write_row(const RowsParams& p, const Request& rq, int flat,
                                          int kv_head, float* part, float2 ml, bool any,
                                          uint32_t mine, int c0, int c1) {
  using L = Layout<D>;
  const AttnParams& a = p.a;
  const int tok = static_cast<int>(a.div_group.div(static_cast<uint32_t>(flat)));
  const bool there = tok < rq.n;
  const int head = kv_head * a.group + (flat - tok * a.group);
  const float f = part == nullptr ? inverse_sum(ml.y) : 1.0f;
  T* dst = static_cast<T*>(a.out) + (rq.row0 + static_cast<int64_t>(tok)) * a.out_stride +
           static_cast<int64_t>(head) * D;
#pragma unroll 1
  for (int c = c0; c < c1; c += 32) {
    uint32_t o[32];
    __syncwarp();
    if (any) {  // uniform: the whole CTA had tiles
      tmem_load32(o, mine + L::kO + c);
      tmem_wait_load(o);
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
  if (part != nullptr && there && c0 == 0) *reinterpret_cast<float2*>(part) = ml;
}

template <typename T, int D>
__global__ void __launch_bounds__(Layout<D>::kThreads, 1)
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
  // fp16 results show the rounding of P: they take P in two parts
  constexpr bool kTwo = std::is_same<T, __half>::value;
  constexpr int kCtaRows = kRows * L::kUnits;
  const int64_t rows = static_cast<int64_t>(rq.n) * a.group;
  if (static_cast<int64_t>(tile) * kCtaRows >= rows) return;
  const int first_row = tile * kCtaRows;
  const int units = rows - first_row > kRows ? L::kUnits : 1;
  const int first_tok = static_cast<int>(a.div_group.div(static_cast<uint32_t>(first_row)));
  const int last_tok = min(
      rq.n - 1, static_cast<int>(a.div_group.div(static_cast<uint32_t>(first_row + kCtaRows - 1))));
  const int32_t pos_first = rq.len - rq.n + first_tok, pos_last = rq.len - rq.n + last_tok;
  const KeyRange range = key_range(a, pos_first, pos_last);
  const int32_t all = range.count <= 0 ? 0 : (range.count + kTok - 1) / kTok;
  const int32_t t0 = static_cast<int32_t>(static_cast<int64_t>(all) * split / p.splits);
  const int32_t t1 = static_cast<int32_t>(static_cast<int64_t>(all) * (split + 1) / p.splits);

  if (warp == L::kIssue) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&ctl.tmem)),
                 "r"(L::kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&ctl.full[i], 4);
      mbar_init(&ctl.free[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      for (int j = 0; j < 2; ++j) {
        mbar_init(&ctl.sready[i][j], 1);
        mbar_init(&ctl.pready[i][j], 8);
      }
      mbar_init(&ctl.pvdone[i], 1);
    }
    mbar_init(&ctl.drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  // softmax warps: this thread's row and half of the columns for what is done
  // by rows
  const int unit = warp / 8, side = warp / 4 % 2;
  const int cta_row = unit * kRows + threadIdx.x % kRows, flat = first_row + cta_row;
  const uint32_t mine = ctl.tmem + unit * L::kUnit + (static_cast<uint32_t>(warp % 4) << 21);
  if (warp < 8 * units && side == 0) {
    load_row<T, D>(a, rq, flat, kv_head, threadIdx.x % kRows, smem + unit * L::kQ,
                   ctl.row[cta_row]);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();

  bool ok = true;
  if (warp >= L::kIssue) {
    if (L::kUnits == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
    if (warp == L::kIssue) {
      const uint32_t q = smem_u32(smem);
      if (elect_one()) {  // always the same lane: commits track what their thread issued
        ok = Issuer<D, kTwo>{ctl.tmem, q, q + L::kUnits * L::kQ, units, ctl}.run(t1 - t0);
      }
      __syncwarp();
    }
  } else if (warp >= L::kBring) {
    if (L::kUnits == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    ok = bring<D, kTwo>(a, range, b, kv_head, t0, t1 - t0, smem + L::kUnits * L::kQ, ctl);
  } else if (warp < 8 * units) {
    if (L::kUnits == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 96;");
    ok = attend<D, kTwo>(a, range, t0, t1 - t0, pos_first, pos_last, rq, first_row, ctl);
    asm volatile("bar.sync %0, 256;" ::"r"(1 + unit) : "memory");  // the unit's rows are done
    float* part = nullptr;
    if (p.splits > 1) {
      const int64_t at = (static_cast<int64_t>(b) * a.kv_heads + kv_head) * p.row_tiles + tile;
      part = p.part + ((at * p.splits + split) * kCtaRows + cta_row) * (D + 4);
    }
    write_row<T, D>(p, rq, flat, kv_head, part, ctl.row[cta_row], t1 > t0, mine,
                    side * (D / 2), (side + 1) * (D / 2));
  }
  fence_before();
  if (__syncthreads_or(!ok)) {
    if (warp == L::kIssue && elect_one()) {
      raise_flag(a.status, LMCB_DEVICE_FLAG_WAIT_TIMEOUT);
      commit(&ctl.drained);  // products in flight end before their memory is given back
      mbar_wait(&ctl.drained, 0);
    }
    __syncthreads();
  }
  if (warp == L::kIssue) {
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
  constexpr int kCtaRows = kRows * Layout<D>::kUnits;
  const int64_t at =
      (static_cast<int64_t>(b) * a.kv_heads + kv_head) * p.row_tiles + flat / kCtaRows;
  const float* src = p.part + (at * p.splits * kCtaRows + flat % kCtaRows) * (D + 4);
  float m = -1e30f, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int i = 0; i < p.splits; ++i, src += kCtaRows * (D + 4)) {
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
int split_count(int64_t units, int64_t seen) {
  int64_t n = current_sm_count() / units;
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
  const int64_t cta_rows = kRows * (head_size <= 128 ? 2 : 1);
  pl.row_tiles = (max_query * group + cta_rows - 1) / cta_rows;
  const int64_t units = batch * kv_heads * pl.row_tiles;
  int64_t seen = max_len;
  if (window > 0 && window + sinks + cta_rows < seen) seen = window + sinks + cta_rows;
  pl.splits = split_count(units, seen);
  pl.part_bytes = pl.splits > 1 ? units * pl.splits * cta_rows * (head_size + 4) * 4 : 0;
  return pl;
}

template <typename T, int D>
cudaError_t launch(const RowsParams& p, cudaStream_t stream) {
  constexpr size_t kSmem = Layout<D>::kBytes + 1024;
  cudaError_t err = ensure_smem_limit<kv4_rows_kernel<T, D>>(kSmem, kSmem);
  if (err != cudaSuccess) return err;
  const dim3 grid(static_cast<unsigned>(p.row_tiles * p.splits),
                  static_cast<unsigned>(p.a.kv_heads), static_cast<unsigned>(p.a.batch));
  kv4_rows_kernel<T, D><<<grid, Layout<D>::kThreads, kSmem, stream>>>(p);
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
