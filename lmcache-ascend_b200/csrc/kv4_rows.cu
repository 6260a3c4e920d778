// kv4_rows.cu -- attention over the 4-bit paged cache for many query rows a
// KV head (several query tokens a request).
#include <climits>

#include "kv4_attention.cuh"
#include "kv4_plan.h"

namespace lmcb {
namespace kv4 {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 16;  // cache tokens a warp takes at once

struct RowsParams : AttnParams {
  int32_t heads_per_cta;  // KV heads a CTA works on, a power of two <= kWarps
};

__device__ __forceinline__ int32_t tiles_of(const KeyRange& k) {
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
__device__ __forceinline__ void load_unit_query(const RowsParams& p, const Request& rq, int tile,
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
__device__ __forceinline__ void take_tile(const RowsParams& p, const KeyRange& range, int32_t v0,
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

// Shared memory that finish_unit merges warps in.
template <int D, int NT>
__host__ __device__ constexpr size_t merge_bytes(int heads_per_cta) {
  return static_cast<size_t>(heads_per_cta) * 8 * NT * D * 4 +
         static_cast<size_t>(kWarps + heads_per_cta) * 8 * NT * 4;
}

// Merges the warps of each KV head through shared memory and writes the
// unit's rows: the output itself (slot < 0) or this CTA's part of it.
template <typename T, int D, int NT>
__device__ __forceinline__ void finish_unit(const RowsParams& p, const Request& rq, int tile,
                                            int hg, Running<D, NT>& st, float* smem) {
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
    const float inv = inverse_sum(s_l[row]);
    const int hq = (hg * hw + h) * p.group + (flat - tok * p.group);
    const float x[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
    store_out<T, 4>(static_cast<T*>(p.out) + (rq.row0 + static_cast<int64_t>(tok)) * p.out_stride +
                        static_cast<int64_t>(hq) * D + e,
                    p.out_vec != 0, x);
  }
}

template <typename T, int D, int NT>
__device__ __forceinline__ void run_unit(const RowsParams& p, int b, int tile, int hg,
                                         const Request& rq, float* smem) {
  constexpr int R = 8 * NT;
  const int warp = threadIdx.x / 32;
  const int hw = p.heads_per_cta, tw = kWarps / hw;
  const int kv_head = hg * hw + warp % hw;
  const int first_tok = static_cast<int>(p.div_group.div(static_cast<uint32_t>(tile * R)));
  const int last_tok =
      min(rq.n - 1, static_cast<int>(p.div_group.div(static_cast<uint32_t>(tile * R + R - 1))));
  const KeyRange range = key_range(p, rq.len - rq.n + first_tok, rq.len - rq.n + last_tok);
  const bool mask = last_tok > first_tok;
  const int32_t tile1 = tiles_of(range);
  Query<D, NT> q;
  load_unit_query<T, D, NT>(p, rq, tile, kv_head, q);
  Running<D, NT> st;
  st.reset();
  const int32_t* table = p.table + static_cast<int64_t>(b) * p.table_stride;
  for (int32_t i = warp / hw; i < tile1; i += tw) {
    if (i * kTile < range.count) take_tile<D, NT>(p, range, i * kTile, table, kv_head, mask, q, st);
  }
  finish_unit<T, D, NT>(p, rq, tile, hg, st, smem);
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads) kv4_rows_kernel(const __grid_constant__ RowsParams p) {
  extern __shared__ float rows_smem[];
  const int tile = blockIdx.x, hg = blockIdx.y, b = blockIdx.z;
  const Request rq = load_request(p, b, tile == 0 && hg == 0 && threadIdx.x == 0);
  if (static_cast<int64_t>(tile) * (8 * NT) >= static_cast<int64_t>(rq.n) * p.group) return;
  run_unit<T, D, NT>(p, b, tile, hg, rq, rows_smem);
}

template <typename T, int D, int NT>
cudaError_t launch(const RowsParams& p, cudaStream_t stream) {
  const size_t smem = merge_bytes<D, NT>(p.heads_per_cta);
  cudaError_t err =
      ensure_smem_limit<kv4_rows_kernel<T, D, NT>>(smem, merge_bytes<D, NT>(kWarps));
  if (err != cudaSuccess) return err;
  const int64_t rows = static_cast<int64_t>(p.max_query) * p.group;
  const dim3 grid(static_cast<unsigned>((rows + NT * 8 - 1) / (NT * 8)),
                  static_cast<unsigned>(p.kv_heads / p.heads_per_cta),
                  static_cast<unsigned>(p.batch));
  kv4_rows_kernel<T, D, NT><<<grid, kThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_size(const RowsParams& p, int64_t head_size, cudaStream_t stream) {
  if (head_size == 64) return launch<T, 64, 4>(p, stream);
  if (head_size == 128) return launch<T, 128, 4>(p, stream);
  return launch<T, 256, 2>(p, stream);
}

}  // namespace

size_t rows_workspace(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) {
  return 0;
}

cudaError_t launch_rows(const AttnParams& a, int type, int64_t head_size, int64_t, void*,
                        cudaStream_t stream) {
  RowsParams p;
  static_cast<AttnParams&>(p) = a;
  p.heads_per_cta = 1;
  while (p.heads_per_cta < kWarps && a.kv_heads % (p.heads_per_cta * 2) == 0) p.heads_per_cta *= 2;
  return type == LMCB_DTYPE_BF16 ? launch_size<__nv_bfloat16>(p, head_size, stream)
                                 : launch_size<__half>(p, head_size, stream);
}

}  // namespace kv4
}  // namespace lmcb
