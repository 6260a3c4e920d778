// kv4_attention.cu -- attention over the paged KV cache held in 4 bits
// (layout in kv4.cuh), for one query token a request or several, with an
// optional sliding window and first tokens that stay visible.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q . k_j),
// over the visible keys j of a query at position i: j <= i, and with a window
// w > 0 also j > i - w or j < sinks.
//
// With k_j = zk_j + sk_j ck_j and v_j alike (ck, cv codes 0 ... 15) both
// products are taken on the codes themselves, which are exact in fp16:
//   q . k_j        = sk_j (q . ck_j) + zk_j (sum of q)
//   sum_j p_j v_j  = sum_j (p_j sv_j) cv_j + sum_j p_j zv_j
// so K is never rounded, and V only as far as p_j sv_j is (fp16, 2^-12). The
// code c goes into the matrix instruction as the fp16 bit pattern c, the
// subnormal c 2^-24: two masked bits of a cache word are two operands, with no
// conversion. The factors are kept in range by powers of two that cancel: a
// query row is scaled to a largest element of 2^13 ... 2^14 (bf16 queries
// become fp16 without loss, but for elements below 2^-38 of the row's
// largest), and p_j sv_j by the largest sv exponent seen so far.
//
// A decode step is bound by the cache bytes (D + 8 a token and head), so the
// shape is chosen to read them once and straight into operand registers:
// mma.sync m16n8k16 with 16 cache tokens as its rows and 8 query rows (heads
// that share the KV head, times query tokens) as its columns. The A operand of
// q . k then wants, from lane (g, t) = (lane / 4, lane % 4), any four values of
// token g and of token g + 8 per step, the same for all lanes with that t: a
// lane holds a contiguous quarter of its tokens' code rows. The transposed A
// operand of p v wants token pairs for one value: a byte permute of two words.
// tcgen05 would want the codes expanded to 16 bits in shared memory first, four
// times the bytes read, for query tiles of 8 rows out of its 128.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <climits>
#include <string>

#include "common.cuh"
#include "kv4.cuh"
#include "lmcache_b200.h"

namespace lmcb {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 16;  // cache tokens a warp takes at once
constexpr int kMaxSplitUnits = 4096;
constexpr float kLog2e = 1.4426950408889634f;

struct AttnParams {
  const void* q;
  int q_type;
  int q_vec;  // query rows are 16-byte aligned
  int64_t q_stride;  // elements between query tokens
  void* out;
  int64_t out_stride;
  const int32_t* cache;
  int64_t half_words;
  int64_t row_words;
  int32_t num_blocks;
  FastDiv div_block;
  const int32_t* table;
  int64_t table_stride;
  int32_t table_cols;
  const int32_t* seq_lens;
  const int32_t* query_start;  // NULL: request b is row b
  int32_t num_rows;            // query tokens in q
  int32_t batch;
  int32_t max_query;
  int32_t kv_heads;
  int32_t group;
  FastDiv div_group;
  int32_t heads_per_cta;  // KV heads a CTA works on, a power of two <= kWarps
  int32_t head_groups;    // kv_heads / heads_per_cta
  int32_t row_tiles;      // tiles of query rows a request may have
  float scale_log2;
  int32_t window;
  int32_t sinks;
  int split;  // units are split over CTAs (one row tile a request)
  float* part;         // [2 * grid][heads_per_cta][rows][D + 2]
  int32_t* prefix;     // [batch + 1] tiles before each request (split)
  unsigned int* status;
};

// What a CTA knows of one request.
struct Request {
  int32_t row0;  // first query row in q
  int32_t n;     // query tokens
  int32_t len;   // visible cache length (the last query's position + 1)
};

__device__ __forceinline__ Request load_request(const AttnParams& p, int b, bool flag) {
  Request r;
  int32_t lo = b, hi = b + 1;
  if (p.query_start != nullptr) {
    lo = p.query_start[b];
    hi = p.query_start[b + 1];
  }
  bool bad = lo < 0 || hi < lo || hi > p.num_rows;
  if (bad) lo = hi = 0;
  r.row0 = lo;
  r.n = hi - lo;
  if (r.n > p.max_query) {
    bad = true;
    r.n = 0;
  }
  r.len = p.seq_lens[b];
  const int64_t cap = static_cast<int64_t>(p.table_cols) * p.div_block.d;
  if (r.len < 0 || r.len > cap) {
    bad = true;
    r.len = 0;
  }
  if (bad && flag) raise_flag(p.status, LMCB_DEVICE_FLAG_LENGTH_OUT_OF_RANGE);
  return r;
}

// The keys that any query of a run of positions [p0, p1] sees, as one virtual
// range [0, count): first `head` first tokens, then the tokens from `first` on.
struct KeyRange {
  int32_t count, head, first;
};

__device__ __forceinline__ KeyRange key_range(const AttnParams& p, int32_t p0, int32_t p1) {
  KeyRange k;
  if (p1 < 0) return KeyRange{0, 0, 0};
  k.first = p.window > 0 && p0 - p.window + 1 > 0 ? p0 - p.window + 1 : 0;
  k.head = min(p.sinks, k.first);
  k.count = k.head + p1 + 1 - k.first;
  return k;
}

__device__ __forceinline__ int32_t tiles_of(const KeyRange& k) {
  // A unit without visible keys still has one (empty) tile: its rows are written.
  return k.count <= 0 ? 1 : (k.count + kTile - 1) / kTile;
}

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

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float half_lo(uint32_t v) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(v)));
}
__device__ __forceinline__ float half_hi(uint32_t v) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(v >> 16)));
}

// 2^e for |e| <= 126.
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const int32_t* src) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + i);
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  } else if constexpr (N == 2) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
    w[0] = v.x, w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = static_cast<uint32_t>(__ldg(src + i));
  }
}

template <typename T> __device__ __forceinline__ float elem_to_float(T v);
template <> __device__ __forceinline__ float elem_to_float<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <> __device__ __forceinline__ float elem_to_float<__half>(__half v) {
  return __half2float(v);
}

// N consecutive query elements as floats.
template <typename T, int N>
__device__ __forceinline__ void load_query(const T* src, bool vec, float (&x)[N]) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + i);
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[8 * i + j] = elem_to_float(e[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = elem_to_float(src[i]);
  }
}

// One warp's running softmax over the tiles it has taken, for 8 * NT query
// rows of one KV head. Lane (g, t) holds, for query columns 2 t and 2 t + 1 of
// each group of eight: the running maximum m (log2), its own tokens' parts of
// the sum l and of z = sum p zv, and the output values g * D / 8 ...
template <int D, int NT>
struct Running {
  static constexpr int MT = D / 16;
  float acc[MT][NT][4];
  float m[NT][2], l[NT][2], z[NT][2];
  int vexp;  // acc is in units of 2^(vexp - 15 - 6) 2^24 ... (see value_unit)

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int i = 0; i < MT; ++i)
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
  // p sv goes into the matrix instruction as p sv 2^(21 - vexp), vexp the
  // largest biased fp16 exponent of the sv so far: at most 2^7 for p <= 1.
  __device__ __forceinline__ float value_factor() const { return pow2i(21 - vexp); }
  __device__ __forceinline__ float value_unit() const { return pow2i(24 + vexp - 21); }
};

// Query operands of a unit: B fragments of q . k, and per column the factors
//   s = acc * a * sk + zk * b  (log2 units).
template <int D, int NT>
struct Query {
  static constexpr int KS = D / 16;
  uint32_t frag[NT][KS][2];
  float a[NT][2], b[NT][2];
  int32_t pos[NT][2];  // position of the column's query token, -1: no such row
};

template <typename T, int D, int NT>
__device__ __forceinline__ void load_unit_query(const AttnParams& p, const Request& rq, int tile,
                                                int kv_head, Query<D, NT>& q) {
  const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  constexpr int N = D / 4;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int flat = tile * (8 * NT) + n * 8 + g;
    const int tok = static_cast<int>(p.div_group.div(static_cast<uint32_t>(flat)));
    const int head = kv_head * p.group + (flat - tok * p.group);
    float x[N];
    if (tok < rq.n) {
      load_query<T, N>(static_cast<const T*>(p.q) + (rq.row0 + static_cast<int64_t>(tok)) * p.q_stride +
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
    // 2^e <= big < 2^(e + 1); all zero or subnormal: as 2^-100
    int e = ((__float_as_int(big) >> 23) & 255) - 127;
    e = max(e, -100);
    const float up = pow2i(13 - min(e, 100)), down = pow2i(min(e, 100) - 13);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = __half2float(__float2half_rn(x[i] * up));
      sum += x[i];
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
    for (int w = 0; w < N / 8; ++w)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        q.frag[n][2 * w + j / 2][j % 2] = pack_half2(x[8 * w + j], x[8 * w + j + 4]);
      }
    const float unit = down * p.scale_log2;
    // columns 2 t and 2 t + 1 of the score tile are rows held by lanes of g = 2 t, 2 t + 1
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int src = (2 * t + c) * 4;
      q.a[n][c] = __shfl_sync(0xffffffffu, unit, src) * 16777216.0f;
      q.b[n][c] = __shfl_sync(0xffffffffu, unit * sum, src);
      const int ps = tok < rq.n ? rq.len - rq.n + tok : -1;
      q.pos[n][c] = __shfl_sync(0xffffffffu, ps, src);
    }
  }
}

// One tile of kTile virtual tokens starting at v0.
template <int D, int NT>
__device__ __forceinline__ void take_tile(const AttnParams& p, const KeyRange& range, int32_t v0,
                                          const int32_t* table, int kv_head, bool mask,
                                          const Query<D, NT>& q, Running<D, NT>& st) {
  constexpr int KW = D / 32;  // code words of K a lane holds of a token
  constexpr int VW = D / 64;  // code words of V
  constexpr int MT = D / 16;
  const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;

  // Lane i finds virtual token v0 + i: its key index and its row in the cache.
  int32_t row = -1, key = -1;
  if (lane < kTile && v0 + lane < range.count) {
    const int32_t v = v0 + lane;
    key = v < range.head ? v : range.first + (v - range.head);
    const int32_t blk = static_cast<int32_t>(p.div_block.div(static_cast<uint32_t>(key)));
    const int32_t page = __ldg(table + blk);
    if (page >= 0 && page < p.num_blocks) {
      row = page * static_cast<int32_t>(p.div_block.d) +
            (key - blk * static_cast<int32_t>(p.div_block.d));
    } else {
      raise_flag(p.status, LMCB_DEVICE_FLAG_SLOT_OUT_OF_RANGE);  // the token is not seen
    }
  }

  const int64_t head_off = static_cast<int64_t>(kv_head) * (D / 8);
  const int64_t par_off = static_cast<int64_t>(p.kv_heads) * (D / 8) + kv_head;
  uint32_t kw[2][KW], kpar[2], vpar[2], vw[4][VW];
  int32_t krow[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    krow[i] = __shfl_sync(0xffffffffu, row, g + 8 * i);
    if (krow[i] >= 0) {
      const int32_t* base = p.cache + krow[i] * p.row_words;
      load_words<KW>(kw[i], base + head_off + t * KW);
      kpar[i] = static_cast<uint32_t>(__ldg(base + par_off));
      vpar[i] = static_cast<uint32_t>(__ldg(base + p.half_words + par_off));
    } else {
#pragma unroll
      for (int w = 0; w < KW; ++w) kw[i][w] = 0;
      kpar[i] = vpar[i] = 0;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int32_t r = __shfl_sync(0xffffffffu, row, 2 * t + (i & 1) + 8 * (i >> 1));
    if (r >= 0) {
      load_words<VW>(vw[i], p.cache + p.half_words + r * p.row_words + head_off + g * VW);
    } else {
#pragma unroll
      for (int w = 0; w < VW; ++w) vw[i][w] = 0;
    }
  }
  int32_t kkey[2] = {0, 0};
  if (mask) {
    kkey[0] = __shfl_sync(0xffffffffu, key, g);
    kkey[1] = __shfl_sync(0xffffffffu, key, g + 8);
  }

  // Scores.
  float s[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) s[n][c] = 0.0f;
#pragma unroll
  for (int w = 0; w < KW; ++w) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const uint32_t a0 = (kw[0][w] >> (4 * j)) & 0x000f000fu;
      const uint32_t a1 = (kw[1][w] >> (4 * j)) & 0x000f000fu;
      const uint32_t a2 = (kw[0][w] >> (4 * j + 4)) & 0x000f000fu;
      const uint32_t a3 = (kw[1][w] >> (4 * j + 4)) & 0x000f000fu;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma_f16(s[n], a0, a1, a2, a3, q.frag[n][2 * w + j / 2][0], q.frag[n][2 * w + j / 2][1]);
      }
    }
  }

  // The largest value exponent of the tile rescales the sums when it grows.
  const int vexp = static_cast<int>(
      __reduce_max_sync(0xffffffffu, max((vpar[0] >> 10) & 31u, (vpar[1] >> 10) & 31u)));
  float rescale = 1.0f;
  if (vexp > st.vexp) {
    rescale = pow2i(st.vexp - vexp);
    st.vexp = vexp;
  }
  const float vfac = st.value_factor();
  uint32_t pf[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int i = c >> 1, col = c & 1;
      float v = fmaf(s[n][c] * q.a[n][col], half_lo(kpar[i]), half_hi(kpar[i]) * q.b[n][col]);
      bool seen = krow[i] >= 0;
      if (mask) {
        const int32_t ps = q.pos[n][col];
        seen = seen && kkey[i] <= ps &&
               (p.window == 0 || kkey[i] > ps - p.window || kkey[i] < p.sinks);
      }
      v = seen ? v : -INFINITY;
      s[n][c] = v;
      top[col] = fmaxf(top[col], v);
    }
    float grow[2];
#pragma unroll
    for (int col = 0; col < 2; ++col) {
      top[col] = fmaxf(top[col], __shfl_xor_sync(0xffffffffu, top[col], 4));
      top[col] = fmaxf(top[col], __shfl_xor_sync(0xffffffffu, top[col], 8));
      top[col] = fmaxf(top[col], __shfl_xor_sync(0xffffffffu, top[col], 16));
      const float m = fmaxf(st.m[n][col], top[col]);
      const float ref = m == -INFINITY ? 0.0f : m;
      grow[col] = exp2f(st.m[n][col] - ref);  // 0 for the first keys
      st.m[n][col] = m;
      st.l[n][col] *= grow[col];
      st.z[n][col] *= grow[col];
      top[col] = ref;
    }
    float ps[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int i = c >> 1, col = c & 1;
      const float e = exp2f(s[n][c] - top[col]);
      st.l[n][col] += e;
      st.z[n][col] = fmaf(e, half_hi(vpar[i]), st.z[n][col]);
      ps[c] = e * (half_lo(vpar[i]) * vfac);
    }
    pf[n][0] = transpose_8x8(pack_half2(ps[0], ps[1]));
    pf[n][1] = transpose_8x8(pack_half2(ps[2], ps[3]));
    const float f0 = grow[0] * rescale, f1 = grow[1] * rescale;
    if (__any_sync(0xffffffffu, f0 != 1.0f || f1 != 1.0f)) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        st.acc[i][n][0] *= f0;
        st.acc[i][n][1] *= f1;
        st.acc[i][n][2] *= f0;
        st.acc[i][n][3] *= f1;
      }
    }
  }

  // Values: rows of the A operand are two of the lane's D / 8 values, columns
  // its four tokens.
#pragma unroll
  for (int w = 0; w < VW; ++w) {
    const uint32_t lo0 = __byte_perm(vw[0][w], vw[1][w], 0x5410);
    const uint32_t hi0 = __byte_perm(vw[0][w], vw[1][w], 0x7632);
    const uint32_t lo1 = __byte_perm(vw[2][w], vw[3][w], 0x5410);
    const uint32_t hi1 = __byte_perm(vw[2][w], vw[3][w], 0x7632);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x0 = i < 2 ? lo0 : hi0, x1 = i < 2 ? lo1 : hi1;
      const int sh = 8 * (i & 1);
      const uint32_t a0 = (x0 >> sh) & 0x000f000fu, a1 = (x0 >> (sh + 4)) & 0x000f000fu;
      const uint32_t a2 = (x1 >> sh) & 0x000f000fu, a3 = (x1 >> (sh + 4)) & 0x000f000fu;
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_f16(st.acc[4 * w + i][n], a0, a1, a2, a3, pf[n][0], pf[n][1]);
    }
  }
}

// Output of one row: `o` holds unnormalised sums; l = 0 (nothing seen) gives 0.
template <typename T>
__device__ __forceinline__ T out_elem(float v);
template <> __device__ __forceinline__ __nv_bfloat16 out_elem<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half out_elem<__half>(float v) {
  return __float2half_rn(v);
}

// Shared memory that finish_unit merges warps in.
template <int D, int NT>
__host__ __device__ constexpr size_t merge_bytes(int heads_per_cta) {
  return static_cast<size_t>(heads_per_cta) * 8 * NT * D * 4 +
         static_cast<size_t>(kWarps + heads_per_cta) * 8 * NT * 4;
}

// Merges the warps of each KV head through shared memory and writes the
// unit's rows: the output itself (slot < 0) or this CTA's part of it.
template <typename T, int D, int NT>
__device__ __forceinline__ void finish_unit(const AttnParams& p, const Request& rq, int tile,
                                            int hg, int slot, Running<D, NT>& st, float* smem) {
  constexpr int R = 8 * NT;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const int hw = p.heads_per_cta, tw = kWarps / hw;
  const int head = warp % hw, turn = warp / hw;
  float* s_o = smem;                         // [hw][R][D]
  float* s_m = s_o + hw * R * D;             // [kWarps][R]
  float* s_l = s_m + kWarps * R;             // [hw][R]
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
      if (g == 0) s_m[(turn * hw + head) * R + n * 8 + 2 * t + c] = st.m[n][c];
    }
  __syncthreads();
  const float unit = st.value_unit();
  float f[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float m = -INFINITY;
      for (int w = 0; w < tw; ++w) m = fmaxf(m, s_m[(w * hw + head) * R + n * 8 + 2 * t + c]);
      f[n][c] = m == -INFINITY ? 0.0f : exp2f(st.m[n][c] - m);
    }
  for (int w = 0; w < tw; ++w) {
    if (w == turn) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int col = n * 8 + 2 * t + c;
          float* o = s_o + (head * R + col) * D + g * (D / 8);
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            float2 v;
            v.x = fmaf(st.acc[i][n][c], unit, st.z[n][c]) * f[n][c];
            v.y = fmaf(st.acc[i][n][c + 2], unit, st.z[n][c]) * f[n][c];
            float2* at = reinterpret_cast<float2*>(o + 2 * i);
            if (w > 0) {
              const float2 old = *at;
              v.x += old.x;
              v.y += old.y;
            }
            *at = v;
          }
          if (g == 0) {
            const float l = st.l[n][c] * f[n][c];
            s_l[head * R + col] = w > 0 ? s_l[head * R + col] + l : l;
          }
        }
    }
    __syncthreads();
  }
  // Rows out.
  for (int i = threadIdx.x; i < hw * R * (D / 4); i += kThreads) {
    const int row = i / (D / 4), e = (i % (D / 4)) * 4;
    const int h = row / R, col = row % R;
    const int flat = tile * R + col;
    const int tok = static_cast<int>(p.div_group.div(static_cast<uint32_t>(flat)));
    if (tok >= rq.n) continue;
    const float4 v = *reinterpret_cast<const float4*>(s_o + row * D + e);
    if (slot < 0) {
      const float l = s_l[row];
      const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // NaN stays NaN
      const int hq = (hg * hw + h) * p.group + (flat - tok * p.group);
      T* dst = static_cast<T*>(p.out) + (rq.row0 + static_cast<int64_t>(tok)) * p.out_stride +
               static_cast<int64_t>(hq) * D + e;
      dst[0] = out_elem<T>(v.x * inv);
      dst[1] = out_elem<T>(v.y * inv);
      dst[2] = out_elem<T>(v.z * inv);
      dst[3] = out_elem<T>(v.w * inv);
    } else {
      float* dst = p.part + (static_cast<int64_t>(slot) * hw * R + row) * (D + 4);
      *reinterpret_cast<float4*>(dst + 4 + e) = v;
      if (e == 0) {
        float m = -INFINITY;
        for (int w = 0; w < tw; ++w) m = fmaxf(m, s_m[(w * hw + h) * R + col]);
        dst[0] = m;
        dst[1] = s_l[row];
      }
    }
  }
  __syncthreads();  // smem is used again by the next unit
}

template <typename T, int D, int NT>
__device__ __forceinline__ void run_unit(const AttnParams& p, int b, int tile, int hg,
                                         const Request& rq, int32_t tile0, int32_t tile1,
                                         int slot, float* smem) {
  constexpr int R = 8 * NT;
  const int warp = threadIdx.x / 32;
  const int hw = p.heads_per_cta, tw = kWarps / hw;
  const int kv_head = hg * hw + warp % hw;
  const int first_tok = static_cast<int>(p.div_group.div(static_cast<uint32_t>(tile * R)));
  const int last_tok =
      min(rq.n - 1, static_cast<int>(p.div_group.div(static_cast<uint32_t>(tile * R + R - 1))));
  const KeyRange range = key_range(p, rq.len - rq.n + first_tok, rq.len - rq.n + last_tok);
  const bool mask = last_tok > first_tok;
  tile1 = min(tile1, tiles_of(range));
  Query<D, NT> q;
  load_unit_query<T, D, NT>(p, rq, tile, kv_head, q);
  Running<D, NT> st;
  st.reset();
  const int32_t* table = p.table + static_cast<int64_t>(b) * p.table_stride;
  for (int32_t i = tile0 + warp / hw; i < tile1; i += tw) {
    if (i * kTile < range.count) take_tile<D, NT>(p, range, i * kTile, table, kv_head, mask, q, st);
  }
  finish_unit<T, D, NT>(p, rq, tile, hg, slot, st, smem);
}

// Tiles of request b when it is split (one row tile a request).
__device__ __forceinline__ int32_t request_tiles(const AttnParams& p, const Request& r) {
  return r.n == 0 ? 0 : tiles_of(key_range(p, r.len - r.n, r.len - 1));
}

// Split: the tiles of all requests and head groups are one line, (head group,
// request, tile), cut into gridDim.x equal pieces, whatever the lengths. A CTA
// writes whole units to the output and at most two pieces of units (its first
// and its last) to the workspace. Not split: a CTA takes one unit.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads) kv4_attention_kernel(const __grid_constant__ AttnParams p) {
  extern __shared__ float attn_smem[];
  if (!p.split) {
    const int tile = blockIdx.x, hg = blockIdx.y, b = blockIdx.z;
    const Request rq = load_request(p, b, tile == 0 && hg == 0 && threadIdx.x == 0);
    if (static_cast<int64_t>(tile) * (8 * NT) >= static_cast<int64_t>(rq.n) * p.group) return;
    run_unit<T, D, NT>(p, b, tile, hg, rq, 0, INT_MAX, -1, attn_smem);
    return;
  }
  __shared__ int32_t s_warp[kWarps];
  int32_t* s_prefix = reinterpret_cast<int32_t*>(  // [batch + 1]
      reinterpret_cast<char*>(attn_smem) + merge_bytes<D, NT>(p.heads_per_cta));
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int32_t base = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    int32_t own = 0;
    if (b < p.batch) own = request_tiles(p, load_request(p, b, blockIdx.x == 0));
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
    if (b < p.batch) s_prefix[b] = before + sum - own;
    __syncthreads();
  }
  if (threadIdx.x == 0) s_prefix[p.batch] = base;
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i <= p.batch; i += kThreads) p.prefix[i] = s_prefix[i];
  }
  const int64_t total = static_cast<int64_t>(base) * p.head_groups;
  const int64_t begin = total * blockIdx.x / gridDim.x;
  const int64_t end = total * (blockIdx.x + 1) / gridDim.x;
  bool first = true;
  for (int64_t at = begin; at < end;) {
    const int hg = static_cast<int>(at / base);
    const int32_t in_group = static_cast<int32_t>(at - static_cast<int64_t>(hg) * base);
    int lo = 0, hi = p.batch;  // s_prefix[lo] <= in_group < s_prefix[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_prefix[mid] <= in_group) lo = mid; else hi = mid;
    }
    const int32_t unit_tiles = s_prefix[lo + 1] - s_prefix[lo];
    const int32_t t0 = in_group - s_prefix[lo];
    const int64_t left = end - at;
    const int32_t t1 = left < unit_tiles - t0 ? t0 + static_cast<int32_t>(left) : unit_tiles;
    const bool whole = t0 == 0 && t1 == unit_tiles;
    const int slot = whole ? -1 : 2 * static_cast<int>(blockIdx.x) + (first ? 0 : 1);
    run_unit<T, D, NT>(p, lo, 0, hg, load_request(p, lo, false), t0, t1, slot, attn_smem);
    first = false;
    at += t1 - t0;
  }
}

// Joins the pieces of every unit that more than one CTA worked on. One CTA of
// 128 threads a query row: four groups of lanes share the pieces, always in
// the same order.
constexpr int kJoinThreads = 128;

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kJoinThreads)
kv4_attention_join_kernel(const __grid_constant__ AttnParams p, const int num_ctas) {
  constexpr int R = 8 * NT;
  constexpr int kLanes = D / 4;
  constexpr int kParts = kJoinThreads / kLanes;
  __shared__ float4 s_o[kParts][kLanes];
  __shared__ float s_l[kParts], s_m[kParts];
  const int b = blockIdx.y, kv_head = blockIdx.x / R, col = blockIdx.x % R;
  const int hg = kv_head / p.heads_per_cta, h = kv_head % p.heads_per_cta;
  const int tok = static_cast<int>(p.div_group.div(static_cast<uint32_t>(col)));
  const Request rq = load_request(p, b, false);
  if (tok >= rq.n) return;
  const int64_t per_group = p.prefix[p.batch];
  const int64_t total = per_group * p.head_groups;
  const int64_t u0 = hg * per_group + p.prefix[b], u1 = hg * per_group + p.prefix[b + 1];
  const auto bound = [&](int64_t c) { return total * c / num_ctas; };
  const auto cta_of = [&](int64_t x) {  // bound(c) <= x < bound(c + 1)
    int64_t c = x * num_ctas / total;
    while (bound(c + 1) <= x) ++c;
    while (bound(c) > x) --c;
    return c;
  };
  const int64_t c0 = cta_of(u0), c1 = cta_of(u1 - 1);
  if (c0 == c1) return;  // written by its CTA
  const int part = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const auto piece = [&](int64_t c) {
    const int64_t slot = 2 * c + (bound(c) >= u0 ? 0 : 1);
    return p.part + ((slot * p.heads_per_cta + h) * R + col) * (D + 4);
  };
  float m = -INFINITY, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int64_t c = c0 + part; c <= c1; c += kParts) {
    if (bound(c) == bound(c + 1)) continue;  // fewer tiles than CTAs: took none
    const float* src = piece(c);
    const float pm = src[0], pl = src[1];
    const float4 v = *reinterpret_cast<const float4*>(src + 4 + lane * 4);
    const float nm = fmaxf(m, pm);
    const float ref = nm == -INFINITY ? 0.0f : nm;
    const float fa = exp2f(m - ref), fb = exp2f(pm - ref);
    m = nm;
    l = l * fa + pl * fb;
    o.x = o.x * fa + v.x * fb;
    o.y = o.y * fa + v.y * fb;
    o.z = o.z * fa + v.z * fb;
    o.w = o.w * fa + v.w * fb;
  }
  s_o[part][lane] = o;
  if (lane == 0) s_l[part] = l, s_m[part] = m;
  __syncthreads();
  if (part != 0) return;
  for (int i = 1; i < kParts; ++i) {
    const float nm = fmaxf(m, s_m[i]);
    const float ref = nm == -INFINITY ? 0.0f : nm;
    const float fa = exp2f(m - ref), fb = exp2f(s_m[i] - ref);
    const float4 v = s_o[i][lane];
    m = nm;
    l = l * fa + s_l[i] * fb;
    o.x = o.x * fa + v.x * fb;
    o.y = o.y * fa + v.y * fb;
    o.z = o.z * fa + v.z * fb;
    o.w = o.w * fa + v.w * fb;
  }
  const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
  const int hq = kv_head * p.group + (col - tok * p.group);
  T* dst = static_cast<T*>(p.out) + (rq.row0 + static_cast<int64_t>(tok)) * p.out_stride +
           static_cast<int64_t>(hq) * D + lane * 4;
  dst[0] = out_elem<T>(o.x * inv);
  dst[1] = out_elem<T>(o.y * inv);
  dst[2] = out_elem<T>(o.z * inv);
  dst[3] = out_elem<T>(o.w * inv);
}

// ---------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------

// How a call is cut up; the same for the workspace size and the launch.
struct Plan {
  int nt;  // groups of eight query rows a unit holds
  int heads_per_cta;
  bool split;
  int ctas;
  int64_t part_bytes;    // partial rows
  int64_t prefix_bytes;
};

int pick_nt(int64_t rows, int64_t head_size) {
  const int most = head_size == 256 ? 2 : 4;
  int nt = 1;
  while (nt < most && nt * 8 < rows) nt *= 2;
  return nt;
}

Plan make_plan(int64_t batch, int64_t max_query, int64_t max_len, int64_t kv_heads, int64_t group,
               int64_t head_size, int64_t window, int64_t sinks) {
  Plan pl;
  const int64_t rows = max_query * group;
  pl.nt = pick_nt(rows, head_size);
  pl.heads_per_cta = 1;
  while (pl.heads_per_cta < kWarps && kv_heads % (pl.heads_per_cta * 2) == 0) pl.heads_per_cta *= 2;
  const int64_t head_groups = kv_heads / pl.heads_per_cta;
  int64_t seen = max_len;
  if (window > 0 && window + sinks + max_query < seen) seen = window + sinks + max_query;
  const int64_t tiles = batch * head_groups * ((seen + kTile - 1) / kTile);
  const int64_t per_step = kWarps / pl.heads_per_cta;
  const int64_t most = static_cast<int64_t>(current_sm_count()) * (pl.nt == 1 ? 2 : 1);
  int64_t ctas = (tiles + per_step - 1) / per_step;
  if (ctas > most) ctas = most;
  if (ctas < 1) ctas = 1;
  pl.split = rows <= pl.nt * 8 && batch <= kMaxSplitUnits && seen > kTile * per_step;
  pl.ctas = static_cast<int>(ctas);
  pl.prefix_bytes = (batch + 1 + 63) / 64 * 256;
  pl.part_bytes = 2 * ctas * pl.heads_per_cta * pl.nt * 8 * (head_size + 4) * 4;
  return pl;
}

template <typename T, int D, int NT>
cudaError_t launch(const AttnParams& p, const Plan& pl, cudaStream_t stream) {
  constexpr size_t kPrefixBytes = (kMaxSplitUnits + 1) * 4;
  const size_t smem = merge_bytes<D, NT>(p.heads_per_cta) +
                      (p.split ? (static_cast<size_t>(p.batch) + 1) * 4 : 0);
  // 47 KB: the static shared memory counts towards the 48 KB that need no limit
  cudaError_t err = ensure_smem_limit<kv4_attention_kernel<T, D, NT>>(
      smem > 47 * 1024 ? smem + 1024 : smem, merge_bytes<D, NT>(kWarps) + kPrefixBytes);
  if (err != cudaSuccess) return err;
  if (p.split) {
    kv4_attention_kernel<T, D, NT><<<pl.ctas, kThreads, smem, stream>>>(p);
    err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    const dim3 grid(static_cast<unsigned>(p.kv_heads * 8 * NT), static_cast<unsigned>(p.batch));
    kv4_attention_join_kernel<T, D, NT><<<grid, kJoinThreads, 0, stream>>>(p, pl.ctas);
  } else {
    const dim3 grid(static_cast<unsigned>(p.row_tiles), static_cast<unsigned>(p.head_groups),
                    static_cast<unsigned>(p.batch));
    kv4_attention_kernel<T, D, NT><<<grid, kThreads, smem, stream>>>(p);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_size(const AttnParams& p, const Plan& pl, int64_t head_size,
                        cudaStream_t stream) {
  if (head_size == 64) {
    if (pl.nt == 1) return launch<T, 64, 1>(p, pl, stream);
    if (pl.nt == 2) return launch<T, 64, 2>(p, pl, stream);
    return launch<T, 64, 4>(p, pl, stream);
  }
  if (head_size == 128) {
    if (pl.nt == 1) return launch<T, 128, 1>(p, pl, stream);
    if (pl.nt == 2) return launch<T, 128, 2>(p, pl, stream);
    return launch<T, 128, 4>(p, pl, stream);
  }
  if (pl.nt == 1) return launch<T, 256, 1>(p, pl, stream);
  return launch<T, 256, 2>(p, pl, stream);
}

int check_shape(const std::string& who, int64_t batch, int64_t max_query, int64_t max_len,
                int64_t kv_heads, int64_t query_heads, int64_t head_size, int64_t window,
                int64_t sinks) {
  if (head_size != 64 && head_size != 128 && head_size != 256) {
    return fail(LMCB_ERR_INVALID_ARGUMENT, who + ": head_size must be 64, 128 or 256.");
  }
  if (batch < 0 || batch > 65535 || max_query < 0 || max_len < 0 || kv_heads <= 0 ||
      query_heads <= 0 || query_heads % kv_heads != 0 || query_heads > 4096 || window < 0 ||
      sinks < 0 || window > INT_MAX || sinks > INT_MAX || max_len > INT_MAX ||
      max_query > (INT_MAX / 2) / query_heads) {
    return fail(LMCB_ERR_INVALID_ARGUMENT, who + ": invalid shape.");
  }
  return LMCB_OK;
}

}  // namespace
}  // namespace lmcb

extern "C" {

int lmcb_kv4_attention_workspace(int64_t batch, int64_t maxQueryLen, int64_t maxSeqLen,
                                 int64_t numKvHeads, int64_t numQueryHeads, int64_t headSize,
                                 int64_t window, int64_t sinks, size_t* bytesOut) {
  lmcb::clear_error();
  const std::string who = "kv4_attention_workspace";
  if (bytesOut == nullptr) {
    return lmcb::fail(LMCB_ERR_INVALID_ARGUMENT, who + ": bytesOut is NULL.");
  }
  const int st = lmcb::check_shape(who, batch, maxQueryLen, maxSeqLen, numKvHeads, numQueryHeads,
                                   headSize, window, sinks);
  if (st != LMCB_OK) return st;
  const lmcb::Plan pl = lmcb::make_plan(batch, maxQueryLen, maxSeqLen, numKvHeads,
                                        numQueryHeads / numKvHeads, headSize, window, sinks);
  *bytesOut = pl.split ? static_cast<size_t>(pl.part_bytes + pl.prefix_bytes) : 0;
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
  lmcb::clear_error();
  const std::string who = "kv4_attention";
  if (type != LMCB_DTYPE_BF16 && type != LMCB_DTYPE_FP16) {
    return lmcb::fail(LMCB_ERR_UNSUPPORTED_DTYPE, who + ": queries must be bf16 or fp16.");
  }
  int st = lmcb::check_shape(who, batch, maxQueryLen, maxSeqLen, numKvHeads, numQueryHeads,
                             headSize, window, sinks);
  if (st != LMCB_OK) return st;
  if (numQueryRows < 0 || numQueryRows > INT_MAX / 2 || numBlocks < 0 || blockSize <= 0 ||
      (numBlocks > 0 && blockSize > INT_MAX / numBlocks) || tableCols < 0 ||
      tableStride < tableCols || (tableCols > 0 && blockSize > INT_MAX / tableCols) ||
      queryTokenStride < numQueryHeads * headSize || outTokenStride < numQueryHeads * headSize ||
      (queryStart == nullptr && (maxQueryLen < 1 || numQueryRows < batch))) {
    return lmcb::fail(LMCB_ERR_INVALID_ARGUMENT, who + ": invalid shape.");
  }
  if (batch == 0 || numQueryRows == 0 || maxQueryLen == 0) return LMCB_OK;
  if (query == nullptr || out == nullptr || seqLens == nullptr ||
      (tableCols > 0 && blockTable == nullptr) || (numBlocks > 0 && kvCache == nullptr)) {
    return lmcb::fail(LMCB_ERR_INVALID_ARGUMENT, who + ": NULL pointer.");
  }
  if (reinterpret_cast<uintptr_t>(kvCache) % 16 != 0) {
    return lmcb::fail(LMCB_ERR_INVALID_ARGUMENT, who + ": the cache must be 16-byte aligned.");
  }
  const lmcb::Plan pl = lmcb::make_plan(batch, maxQueryLen, maxSeqLen, numKvHeads,
                                        numQueryHeads / numKvHeads, headSize, window, sinks);
  if (pl.split && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 ||
                   workspaceBytes < static_cast<size_t>(pl.part_bytes + pl.prefix_bytes))) {
    return lmcb::fail(LMCB_ERR_CAPACITY, who + ": the workspace is too small or not aligned.");
  }
  lmcb::AttnParams p;
  p.q = query;
  p.q_type = type;
  p.q_vec = reinterpret_cast<uintptr_t>(query) % 16 == 0 && queryTokenStride % 8 == 0;
  p.q_stride = queryTokenStride;
  p.out = out;
  p.out_stride = outTokenStride;
  p.cache = kvCache;
  p.row_words = lmcb::kv4_row_words(numKvHeads, headSize);
  p.half_words = numBlocks * blockSize * p.row_words;
  p.num_blocks = static_cast<int32_t>(numBlocks);
  p.div_block = lmcb::FastDiv(static_cast<uint32_t>(blockSize));
  p.table = blockTable;
  p.table_stride = tableStride;
  p.table_cols = static_cast<int32_t>(tableCols);
  p.seq_lens = seqLens;
  p.query_start = queryStart;
  p.num_rows = static_cast<int32_t>(numQueryRows);
  p.batch = static_cast<int32_t>(batch);
  p.max_query = static_cast<int32_t>(maxQueryLen);
  p.kv_heads = static_cast<int32_t>(numKvHeads);
  p.group = static_cast<int32_t>(numQueryHeads / numKvHeads);
  p.div_group = lmcb::FastDiv(static_cast<uint32_t>(p.group));
  p.heads_per_cta = pl.heads_per_cta;
  p.head_groups = p.kv_heads / pl.heads_per_cta;
  p.row_tiles = static_cast<int32_t>((maxQueryLen * p.group + pl.nt * 8 - 1) / (pl.nt * 8));
  p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  p.window = static_cast<int32_t>(window);
  p.sinks = static_cast<int32_t>(sinks);
  p.split = pl.split ? 1 : 0;
  p.part = static_cast<float*>(workspace);
  p.prefix = pl.split ? reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + pl.part_bytes)
                      : nullptr;
  p.status = lmcb::device_status_ptr();
  if (p.status == nullptr) return LMCB_ERR_CUDA;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = type == LMCB_DTYPE_BF16
                              ? lmcb::launch_size<__nv_bfloat16>(p, pl, headSize, s)
                              : lmcb::launch_size<__half>(p, pl, headSize, s);
  if (err != cudaSuccess) return lmcb::cuda_fail(err, who.c_str());
  return LMCB_OK;
}

}  // extern "C"
