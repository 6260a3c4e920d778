// pos_kernels.cu -- fused K re-rotation for CacheBlend (rotary_embedding_k_fused).
//
// The reference exports rotary_embedding_k_fused (csrc/pybind.cpp:25) but its
// body raises NotImplementedError (csrc/pos_kernels.cpp:7-14). Its caller
// (lmcache_ascend/v1/blend/positional_encoding.py:57-77) moves cached K rows
// from the positions they were encoded at to new positions; the unfused
// equivalent there (DummyFusedRope, :80-101) undoes the rotary embedding at
// the old positions and applies it at the new ones. This kernel does both in
// one pass: for each rotated pair (x1, x2) with angles a (old) and b (new),
//   (x1, x2) <- R(b - a) (x1, x2),
//   cos(b - a) = cos b cos a + sin b sin a,  sin(b - a) = sin b cos a - cos b sin a,
// in fp32, rounding once to the key's type. Pairs follow the rotary layouts
// of the cos/sin cache [max_position, rot_dim] = [cos | sin]: neox style pairs
// dims (i, i + rot_dim/2), GPT-J style pairs (2i, 2i + 1); dims at and beyond
// rot_dim are left unchanged.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <cstdlib>
#include <cstring>
#include <string>

#include "common.cuh"
#include "lmcache_b200.h"

namespace lmcb {
namespace {

constexpr int kRopeThreads = 128;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// The rotation of one pair, with every rounding explicit: products by
// __fmul_rn and sums by __fmaf_rn leave the compiler no multiply-add to
// contract on its own, so the three kernels below compute bit-identical
// results whatever their instruction schedule.
//   c = cos(b - a) = cos b cos a + sin b sin a,  s = sin(b - a) = sin b cos a - cos b sin a
//   y1 = x1 c - x2 s,                             y2 = x2 c + x1 s
__device__ __forceinline__ void angle_diff(float cos_a, float sin_a, float cos_b, float sin_b,
                                           float& c, float& s) {
  c = __fmaf_rn(cos_b, cos_a, __fmul_rn(sin_b, sin_a));
  s = __fmaf_rn(sin_b, cos_a, -__fmul_rn(cos_b, sin_a));
}

__device__ __forceinline__ void rotate_pair(float x1, float x2, float c, float s, float& y1,
                                            float& y2) {
  y1 = __fmaf_rn(x1, c, -__fmul_rn(x2, s));
  y2 = __fmaf_rn(x2, c, __fmul_rn(x1, s));
}

struct RopeParams {
  const void* old_pos;
  const void* new_pos;
  void* key;
  const void* cache;
  int64_t num_tokens;
  int64_t num_heads;
  int64_t head_size;
  int64_t token_stride;  // elements between consecutive tokens of `key`
  int64_t rot_dim;
  int64_t max_position;
  int is_neox;
  unsigned int* status;
  FastDiv div_half;  // pair index -> head: by rot_dim / 2 (rot_dim / 4 in the vec2 kernel)
};

// A CTA walks tokens in a grid-stride loop (one launch of up to
// kRopeBlocksPerSm CTAs per SM, instead of a tiny CTA per token); within a
// token, thread q handles rotated pairs q, q + blockDim.x, ... with 32-bit
// pair arithmetic (pairs per token = num_heads * rot_dim / 2 < 2^31, checked
// by the entry point).
template <typename KeyT, typename CacheT, typename PosT>
__global__ void __launch_bounds__(kRopeThreads) rope_k_fused_kernel(const RopeParams p) {
  const int half = static_cast<int>(p.rot_dim / 2);
  const int pairs = static_cast<int>(p.num_heads) * half;
  for (int64_t token = blockIdx.x; token < p.num_tokens; token += gridDim.x) {
    const int64_t a = static_cast<int64_t>(static_cast<const PosT*>(p.old_pos)[token]);
    const int64_t b = static_cast<int64_t>(static_cast<const PosT*>(p.new_pos)[token]);
    if (a < 0 || a >= p.max_position || b < 0 || b >= p.max_position) {
      if (threadIdx.x == 0) raise_flag(p.status, LMCB_DEVICE_FLAG_POSITION_OUT_OF_RANGE);
      continue;  // uniform across the CTA
    }
    const CacheT* ca = static_cast<const CacheT*>(p.cache) + a * p.rot_dim;
    const CacheT* cb = static_cast<const CacheT*>(p.cache) + b * p.rot_dim;
    KeyT* k = static_cast<KeyT*>(p.key) + token * p.token_stride;
    for (int q = threadIdx.x; q < pairs; q += blockDim.x) {
      const int h = static_cast<int>(p.div_half.div(static_cast<uint32_t>(q)));
      const int i = q - h * half;
      const float cos_a = to_f(ca[i]), sin_a = to_f(ca[half + i]);
      const float cos_b = to_f(cb[i]), sin_b = to_f(cb[half + i]);
      float c, s;
      angle_diff(cos_a, sin_a, cos_b, sin_b, c, s);
      KeyT* row = k + static_cast<int64_t>(h) * p.head_size;
      const int i1 = p.is_neox ? i : 2 * i;
      const int i2 = p.is_neox ? i + half : 2 * i + 1;
      float y1, y2;
      rotate_pair(to_f(row[i1]), to_f(row[i2]), c, s, y1, y2);
      row[i1] = from_f<KeyT>(y1);
      row[i2] = from_f<KeyT>(y2);
    }
  }
}

// Same rotation, two adjacent pairs per step with 2-element vector accesses:
// neox pairs (i, i + half) and (i + 1, i + 1 + half), GPT-J pairs (2i, 2i + 1)
// and (2i + 2, 2i + 3), i even; cos/sin of both pairs come in one 2-element
// load each. The per-pair arithmetic is that of rope_k_fused_kernel, so the
// results are identical. Launched only when the host has checked that every
// access is aligned to its vector width (rope_vec_ok).
template <typename T, int N>
struct alignas(sizeof(T) * N) RopeVec {
  T v[N];
};

template <typename KeyT, typename CacheT, typename PosT>
__global__ void __launch_bounds__(kRopeThreads) rope_k_fused_vec2_kernel(const RopeParams p) {
  const int half = static_cast<int>(p.rot_dim / 2);
  const int quads = static_cast<int>(p.num_heads) * (half / 2);  // pair pairs per token
  const FastDiv& div_q = p.div_half;  // here: division by half / 2
  for (int64_t token = blockIdx.x; token < p.num_tokens; token += gridDim.x) {
    const int64_t a = static_cast<int64_t>(static_cast<const PosT*>(p.old_pos)[token]);
    const int64_t b = static_cast<int64_t>(static_cast<const PosT*>(p.new_pos)[token]);
    if (a < 0 || a >= p.max_position || b < 0 || b >= p.max_position) {
      if (threadIdx.x == 0) raise_flag(p.status, LMCB_DEVICE_FLAG_POSITION_OUT_OF_RANGE);
      continue;  // uniform across the CTA
    }
    const CacheT* ca = static_cast<const CacheT*>(p.cache) + a * p.rot_dim;
    const CacheT* cb = static_cast<const CacheT*>(p.cache) + b * p.rot_dim;
    KeyT* k = static_cast<KeyT*>(p.key) + token * p.token_stride;
    for (int q = threadIdx.x; q < quads; q += blockDim.x) {
      const int h = static_cast<int>(div_q.div(static_cast<uint32_t>(q)));
      const int i = 2 * (q - h * (half / 2));
      using C2 = RopeVec<CacheT, 2>;
      const C2 cos_a = *reinterpret_cast<const C2*>(ca + i);
      const C2 sin_a = *reinterpret_cast<const C2*>(ca + half + i);
      const C2 cos_b = *reinterpret_cast<const C2*>(cb + i);
      const C2 sin_b = *reinterpret_cast<const C2*>(cb + half + i);
      float c[2], sn[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float ca_j = to_f(cos_a.v[j]), sa_j = to_f(sin_a.v[j]);
        const float cb_j = to_f(cos_b.v[j]), sb_j = to_f(sin_b.v[j]);
        angle_diff(ca_j, sa_j, cb_j, sb_j, c[j], sn[j]);
      }
      KeyT* row = k + static_cast<int64_t>(h) * p.head_size;
      if (p.is_neox) {
        using K2 = RopeVec<KeyT, 2>;
        K2* p1 = reinterpret_cast<K2*>(row + i);
        K2* p2 = reinterpret_cast<K2*>(row + half + i);
        K2 x1 = *p1, x2 = *p2;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float y1, y2;
          rotate_pair(to_f(x1.v[j]), to_f(x2.v[j]), c[j], sn[j], y1, y2);
          x1.v[j] = from_f<KeyT>(y1);
          x2.v[j] = from_f<KeyT>(y2);
        }
        *p1 = x1;
        *p2 = x2;
      } else {
        using K4 = RopeVec<KeyT, 4>;
        K4* px = reinterpret_cast<K4*>(row + 2 * i);
        K4 x = *px;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float y1, y2;
          rotate_pair(to_f(x.v[2 * j]), to_f(x.v[2 * j + 1]), c[j], sn[j], y1, y2);
          x.v[2 * j] = from_f<KeyT>(y1);
          x.v[2 * j + 1] = from_f<KeyT>(y2);
        }
        *px = x;
      }
    }
  }
}

// Same rotation with 16-byte key vectors, the angles computed once per token
// for all heads. An item is (token, vector v): v selects E = 16 /
// sizeof(KeyT) key elements -- for neox the E dims at v * E of the first
// rotary half, paired with the E dims at half + v * E; for GPT-J E / 2
// adjacent pairs at v * E -- and the item rotates that vector of every head.
// The cos/sin runs the vector needs are loaded once per item and the angle
// differences computed once, not once per head (heads of a token share its
// positions): cache traffic per token is one pass over its two cache rows
// against two passes over its key rows. Items are numbered token-major with
// v fastest, so the threads of a warp read and write whole 128-byte segments
// of each head. A thread loads eight key vectors (kRopeHeadsInFlight heads,
// half as many for neox, whose heads take two vectors each) and, for the
// first group, the positions before it uses any, then rotates and stores
// them. The per-pair arithmetic is angle_diff / rotate_pair, as in the
// other kernels, so the results are identical. Launched only when the host
// has checked alignment and that the item count is below 2^31 (rope_v16_ok).
constexpr int kRopeV16Threads = 256;
constexpr int kRopeHeadsInFlight = 8;

template <typename T>
struct alignas(16) Vec16 {
  T v[16 / sizeof(T)];
};

// N consecutive cache values at `src` as floats: 16-byte loads when the run
// is at least 16 bytes (src 16-byte aligned), else one load of the run.
template <typename CacheT, int N>
__device__ __forceinline__ void load_cache_run(const CacheT* src, float (&out)[N]) {
  constexpr int kBytes = N * static_cast<int>(sizeof(CacheT));
  if constexpr (kBytes >= 16) {
    constexpr int kPer = 16 / sizeof(CacheT);
#pragma unroll
    for (int c = 0; c < N / kPer; ++c) {
      const Vec16<CacheT> piece = reinterpret_cast<const Vec16<CacheT>*>(src)[c];
#pragma unroll
      for (int j = 0; j < kPer; ++j) out[c * kPer + j] = to_f(piece.v[j]);
    }
  } else {
    const RopeVec<CacheT, N> piece = *reinterpret_cast<const RopeVec<CacheT, N>*>(src);
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = to_f(piece.v[j]);
  }
}

template <typename KeyT, typename CacheT, typename PosT, bool kNeox>
__global__ void __launch_bounds__(kRopeV16Threads, 2)
rope_k_fused_v16_kernel(const RopeParams p, const uint32_t num_items, const FastDiv div_vec) {
  constexpr int E = 16 / sizeof(KeyT);   // key elements per vector
  constexpr int NP = kNeox ? E : E / 2;  // pairs per vector
  constexpr int HF = kNeox ? kRopeHeadsInFlight / 2 : kRopeHeadsInFlight;  // vectors in flight: 8
  using KV = Vec16<KeyT>;
  const int half = static_cast<int>(p.rot_dim / 2);
  const int heads = static_cast<int>(p.num_heads);
  for (uint32_t item = blockIdx.x * kRopeV16Threads + threadIdx.x; item < num_items;
       item += gridDim.x * kRopeV16Threads) {
    const uint32_t t = div_vec.div(item);
    const int v = static_cast<int>(item - t * div_vec.d);
    const int e0 = v * E;                 // first key element of the vector
    const int col = kNeox ? e0 : e0 / 2;  // its first cache column (pair index)
    KeyT* row0 = static_cast<KeyT*>(p.key) + static_cast<int64_t>(t) * p.token_stride + e0;
    float c[NP], sn[NP];
    for (int h0 = 0; h0 < heads; h0 += HF) {
      KV x1[HF], x2[HF];
      // 1. this group's key vectors (and, for the first group, the positions)
#pragma unroll
      for (int hh = 0; hh < HF; ++hh) {
        if (h0 + hh < heads) {
          const KeyT* r = row0 + static_cast<int64_t>(h0 + hh) * p.head_size;
          x1[hh] = *reinterpret_cast<const KV*>(r);
          if constexpr (kNeox) x2[hh] = *reinterpret_cast<const KV*>(r + half);
        }
      }
      if (h0 == 0) {
        const int64_t a = static_cast<int64_t>(static_cast<const PosT*>(p.old_pos)[t]);
        const int64_t b = static_cast<int64_t>(static_cast<const PosT*>(p.new_pos)[t]);
        if (a < 0 || a >= p.max_position || b < 0 || b >= p.max_position) {
          if (v == 0) raise_flag(p.status, LMCB_DEVICE_FLAG_POSITION_OUT_OF_RANGE);
          break;  // the token is left unchanged
        }
        const CacheT* ca = static_cast<const CacheT*>(p.cache) + a * p.rot_dim + col;
        const CacheT* cb = static_cast<const CacheT*>(p.cache) + b * p.rot_dim + col;
        float cos_a[NP], sin_a[NP], cos_b[NP], sin_b[NP];
        load_cache_run<CacheT, NP>(ca, cos_a);
        load_cache_run<CacheT, NP>(ca + half, sin_a);
        load_cache_run<CacheT, NP>(cb, cos_b);
        load_cache_run<CacheT, NP>(cb + half, sin_b);
#pragma unroll
        for (int j = 0; j < NP; ++j) angle_diff(cos_a[j], sin_a[j], cos_b[j], sin_b[j], c[j], sn[j]);
      }
      // 2. rotate and store
#pragma unroll
      for (int hh = 0; hh < HF; ++hh) {
        if (h0 + hh >= heads) continue;
        KeyT* r = row0 + static_cast<int64_t>(h0 + hh) * p.head_size;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          float y1, y2;
          if constexpr (kNeox) {
            rotate_pair(to_f(x1[hh].v[j]), to_f(x2[hh].v[j]), c[j], sn[j], y1, y2);
            x1[hh].v[j] = from_f<KeyT>(y1);
            x2[hh].v[j] = from_f<KeyT>(y2);
          } else {
            rotate_pair(to_f(x1[hh].v[2 * j]), to_f(x1[hh].v[2 * j + 1]), c[j], sn[j], y1, y2);
            x1[hh].v[2 * j] = from_f<KeyT>(y1);
            x1[hh].v[2 * j + 1] = from_f<KeyT>(y2);
          }
        }
        *reinterpret_cast<KV*>(r) = x1[hh];
        if constexpr (kNeox) *reinterpret_cast<KV*>(r + half) = x2[hh];
      }
    }
  }
}

// True when every access of rope_k_fused_v16_kernel is aligned and its item
// count fits: E = 16 / sizeof(KeyT); neox needs rot_dim a multiple of 2E,
// GPT-J of E; the key base, token stride and head size multiples of 16 bytes;
// the cache base 16-byte aligned.
template <typename KeyT, typename CacheT>
bool rope_v16_ok(const RopeParams& p, uint32_t* vecs_per_head) {
  constexpr int64_t E = 16 / sizeof(KeyT);
  const int64_t unit = p.is_neox ? 2 * E : E;
  if (p.rot_dim % unit != 0) return false;
  if (reinterpret_cast<uintptr_t>(p.key) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(p.cache) % 16 != 0) {
    return false;
  }
  if ((p.token_stride * static_cast<int64_t>(sizeof(KeyT))) % 16 != 0 ||
      (p.head_size * static_cast<int64_t>(sizeof(KeyT))) % 16 != 0) {
    return false;
  }
  const int64_t vph = p.is_neox ? p.rot_dim / 2 / E : p.rot_dim / E;
  if (p.num_tokens * vph >= (int64_t(1) << 31)) return false;
  *vecs_per_head = static_cast<uint32_t>(vph);
  return true;
}

constexpr int kRopeBlocksPerSm = 16;

// True when every access of rope_k_fused_vec2_kernel is aligned: rot_dim a
// multiple of 4 (so i and half + i are even), the key base, token stride and
// head size multiples of the key vector (2 elements neox, 4 GPT-J) and the
// cache base a multiple of 2 cache elements.
template <typename KeyT, typename CacheT>
bool rope_vec_ok(const RopeParams& p) {
  if (p.rot_dim % 4 != 0) return false;
  const int64_t kv = p.is_neox ? 2 : 4;
  const uint64_t kbytes = static_cast<uint64_t>(kv) * sizeof(KeyT);
  if (reinterpret_cast<uintptr_t>(p.key) % kbytes != 0) return false;
  if ((p.token_stride % kv) != 0 || (p.head_size % kv) != 0) return false;
  return reinterpret_cast<uintptr_t>(p.cache) % (2 * sizeof(CacheT)) == 0;
}

template <typename KeyT, typename CacheT, typename PosT>
void launch_rope_v16(const RopeParams& p, uint32_t vph, cudaStream_t stream) {
  const uint32_t items = static_cast<uint32_t>(p.num_tokens) * vph;
  const int64_t blocks = (static_cast<int64_t>(items) + kRopeV16Threads - 1) / kRopeV16Threads;
  const int64_t max_grid = static_cast<int64_t>(current_sm_count()) * 2;
  const dim3 grid(static_cast<unsigned>(blocks < max_grid ? blocks : max_grid));
  const FastDiv div_vec(vph);
  if (p.is_neox) {
    rope_k_fused_v16_kernel<KeyT, CacheT, PosT, true>
        <<<grid, kRopeV16Threads, 0, stream>>>(p, items, div_vec);
  } else {
    rope_k_fused_v16_kernel<KeyT, CacheT, PosT, false>
        <<<grid, kRopeV16Threads, 0, stream>>>(p, items, div_vec);
  }
}

template <typename KeyT, typename CacheT>
cudaError_t launch_rope_pos(RopeParams p, int pos_type, cudaStream_t stream) {
  const int64_t max_grid = static_cast<int64_t>(current_sm_count()) * kRopeBlocksPerSm;
  const dim3 grid(static_cast<unsigned>(p.num_tokens < max_grid ? p.num_tokens : max_grid));
  uint32_t vph = 0;
  const char* force = std::getenv("LMCB_ROPE_KERNEL");  // "vec2" or "pair": tests, tuning
  const bool allow_v16 = force == nullptr || std::strcmp(force, "v16") == 0;
  const bool allow_vec2 = force == nullptr || std::strcmp(force, "pair") != 0;
  if (allow_v16 && rope_v16_ok<KeyT, CacheT>(p, &vph)) {
    if (pos_type == LMCB_DTYPE_INT64) {
      launch_rope_v16<KeyT, CacheT, int64_t>(p, vph, stream);
    } else {
      launch_rope_v16<KeyT, CacheT, int32_t>(p, vph, stream);
    }
  } else if (allow_vec2 && rope_vec_ok<KeyT, CacheT>(p)) {
    p.div_half = FastDiv(static_cast<uint32_t>(p.rot_dim / 4));
    if (pos_type == LMCB_DTYPE_INT64) {
      rope_k_fused_vec2_kernel<KeyT, CacheT, int64_t><<<grid, kRopeThreads, 0, stream>>>(p);
    } else {
      rope_k_fused_vec2_kernel<KeyT, CacheT, int32_t><<<grid, kRopeThreads, 0, stream>>>(p);
    }
  } else if (pos_type == LMCB_DTYPE_INT64) {
    rope_k_fused_kernel<KeyT, CacheT, int64_t><<<grid, kRopeThreads, 0, stream>>>(p);
  } else {
    rope_k_fused_kernel<KeyT, CacheT, int32_t><<<grid, kRopeThreads, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

template <typename KeyT>
cudaError_t launch_rope_cache(const RopeParams& p, int cache_type, int pos_type,
                              cudaStream_t stream) {
  switch (cache_type) {
    case LMCB_DTYPE_FP32: return launch_rope_pos<KeyT, float>(p, pos_type, stream);
    case LMCB_DTYPE_BF16: return launch_rope_pos<KeyT, __nv_bfloat16>(p, pos_type, stream);
    default: return launch_rope_pos<KeyT, __half>(p, pos_type, stream);
  }
}

bool float_type(int t) {
  return t == LMCB_DTYPE_FP32 || t == LMCB_DTYPE_BF16 || t == LMCB_DTYPE_FP16;
}


// ---------------------------------------------------------------------------
// Per-head norm of queries and keys with the rotation in the same pass
// (qk_norm_rope)
// ---------------------------------------------------------------------------
//
// Every head row x of D values becomes
//   y = x / sqrt(mean(x^2) + eps) * w,
// and its first rot_dim values are rotated by the angles of the token's
// position: y1' = y1 cos - y2 sin, y2' = y2 cos + y1 sin, in the pairs of the
// rotary layouts above. Squares, sum, scale and rotation are fp32; the result
// is rounded once to the row's type, where a norm and a rotation run one after
// the other round twice.

struct QkNormParams {
  const void* in[2];   // q, k
  void* out[2];
  const void* weight[2];  // NULL: no weight
  int weight_type[2];
  int64_t in_stride[2];  // elements between tokens
  int64_t out_stride[2];
  const void* positions;
  int pos64;
  const void* cache;
  int cache_type;
  int64_t num_tokens;
  int32_t heads[2];
  int32_t head_size;
  int32_t rot_dim;
  int64_t max_position;
  float eps;
  unsigned int* status;
};

// N consecutive values of a tensor whose type is known at run time only (the
// weights and the cos/sin rows: once per row or token, the branch is uniform).
template <int N>
__device__ __forceinline__ void load_run_typed(const void* base, int type, int64_t at,
                                               float (&out)[N]) {
  if (type == LMCB_DTYPE_FP32) {
    load_cache_run<float, N>(static_cast<const float*>(base) + at, out);
  } else if (type == LMCB_DTYPE_BF16) {
    load_cache_run<__nv_bfloat16, N>(static_cast<const __nv_bfloat16*>(base) + at, out);
  } else {
    load_cache_run<__half, N>(static_cast<const __half*>(base) + at, out);
  }
}

__device__ __forceinline__ float load_typed(const void* base, int type, int64_t at) {
  if (type == LMCB_DTYPE_FP32) return static_cast<const float*>(base)[at];
  if (type == LMCB_DTYPE_BF16) return to_f(static_cast<const __nv_bfloat16*>(base)[at]);
  return to_f(static_cast<const __half*>(base)[at]);
}

__device__ __forceinline__ int64_t qk_position(const QkNormParams& p, int64_t token) {
  return p.pos64 ? static_cast<const int64_t*>(p.positions)[token]
                 : static_cast<int64_t>(static_cast<const int32_t*>(p.positions)[token]);
}

constexpr int kQkThreads = 256;

// kLanes lanes share a head row; a lane holds two 16-byte vectors of it: for
// neox a vector of the first rotary half and its partner in the second (so a
// pair never leaves its lane), else two vectors of adjacent pairs; lanes behind
// the rotated part hold two vectors of the rest. A warp takes one token and a
// run of its heads (q heads, then k heads), 32 / kLanes heads a step. With r = 1 / sqrt(mean + eps), a pair's results are
//   y1 = r (x1 (w1 cos) - x2 (w2 sin)),  y2 = r (x2 (w2 cos) + x1 (w1 sin)),
// (cos = 1 and sin = 0 where nothing is rotated), and the four products with
// the weights are the same for every q head of the token, and every k head: a
// lane makes them once for the run.
template <typename T>
struct QkFactors {
  static constexpr int E = 16 / sizeof(T);  // pairs of a lane
  float c1[E], s2[E], c2[E], s1[E];         // w1 cos, w2 sin, w2 cos, w1 sin
};

// A lane's two vectors of a row: their first elements, and whether they are
// rotated.
struct QkLane {
  int e0, e1;
  bool turn0, turn1;
};

// Where the factors of a row come from: weights (NULL: none) and a row [cos |
// sin] of `half` values each.
struct QkSource {
  const void* weight;
  int weight_type;
  const void* cache;
  int cache_type;
  int64_t row;
  int half;
};

template <typename T, bool kNeox>
__device__ __forceinline__ void qk_factors(const QkSource& src, const QkLane& ln,
                                           QkFactors<T>& f) {
  constexpr int E = 16 / sizeof(T);
  float wa[E], wb[E], cs[E], sn[E];
#pragma unroll
  for (int j = 0; j < E; ++j) wa[j] = wb[j] = cs[j] = 1.0f, sn[j] = 0.0f;
  if (src.weight != nullptr) {
    load_run_typed<E>(src.weight, src.weight_type, ln.e0, wa);
    load_run_typed<E>(src.weight, src.weight_type, ln.e1, wb);
  }
  if constexpr (kNeox) {
    if (ln.turn0) {
      load_run_typed<E>(src.cache, src.cache_type, src.row + ln.e0, cs);
      load_run_typed<E>(src.cache, src.cache_type, src.row + src.half + ln.e0, sn);
    }
  } else {
    float c[E / 2], s[E / 2];
    if (ln.turn0) {
      load_run_typed<E / 2>(src.cache, src.cache_type, src.row + ln.e0 / 2, c);
      load_run_typed<E / 2>(src.cache, src.cache_type, src.row + src.half + ln.e0 / 2, s);
#pragma unroll
      for (int j = 0; j < E / 2; ++j) cs[j] = c[j], sn[j] = s[j];
    }
    if (ln.turn1) {
      load_run_typed<E / 2>(src.cache, src.cache_type, src.row + ln.e1 / 2, c);
      load_run_typed<E / 2>(src.cache, src.cache_type, src.row + src.half + ln.e1 / 2, s);
#pragma unroll
      for (int j = 0; j < E / 2; ++j) cs[E / 2 + j] = c[j], sn[E / 2 + j] = s[j];
    }
  }
#pragma unroll
  for (int j = 0; j < E; ++j) {
    float w1, w2;
    if constexpr (kNeox) {
      w1 = wa[j];
      w2 = wb[j];
    } else {
      w1 = j < E / 2 ? wa[2 * j] : wb[2 * j - E];
      w2 = j < E / 2 ? wa[2 * j + 1] : wb[2 * j - E + 1];
    }
    const bool turn = kNeox || j < E / 2 ? ln.turn0 : ln.turn1;
    f.c1[j] = w1 * cs[j];
    f.s1[j] = turn ? w1 * sn[j] : 0.0f;  // an infinite weight times 0 is NaN
    f.c2[j] = w2 * cs[j];
    f.s2[j] = turn ? w2 * sn[j] : 0.0f;
  }
}

template <bool kNeox, int E>
__device__ __forceinline__ QkLane qk_lane(int l, int rot) {
  QkLane ln;
  if constexpr (kNeox) {
    const int pairs = rot / 2 / E;  // lanes that hold rotated vectors
    ln.turn0 = ln.turn1 = l < pairs;
    ln.e0 = l < pairs ? l * E : rot + (l - pairs) * 2 * E;
    ln.e1 = l < pairs ? rot / 2 + l * E : ln.e0 + E;
  } else {
    ln.e0 = l * 2 * E;
    ln.e1 = ln.e0 + E;
    ln.turn0 = ln.e0 < rot;
    ln.turn1 = ln.e1 < rot;
  }
  return ln;
}

// One head row, in a lane's two vectors: x becomes the result. All lanes of a
// warp take part; `live` lanes hold something. Where nothing is rotated the partner
// is left out, not multiplied by 0: it may be infinite. (A choice an element: two
// paths, by lane or for rows with an infinity only, took 3 to 8% longer.)
template <typename T, bool kNeox, int kLanes>
__device__ __forceinline__ void qk_row(Vec16<T> (&x)[2], const QkFactors<T>& f, const QkLane& ln,
                                       float mean, float eps, bool live) {
  constexpr int E = 16 / sizeof(T);
  float x1[E], x2[E];  // the pairs
  float ss = 0.0f;
  if (live) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if constexpr (kNeox) {
        x1[j] = to_f(x[0].v[j]);
        x2[j] = to_f(x[1].v[j]);
      } else {
        x1[j] = to_f(j < E / 2 ? x[0].v[2 * j] : x[1].v[2 * j - E]);
        x2[j] = to_f(j < E / 2 ? x[0].v[2 * j + 1] : x[1].v[2 * j - E + 1]);
      }
      ss = fmaf(x1[j], x1[j], ss);
      ss = fmaf(x2[j], x2[j], ss);
    }
  }
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (!live) return;
  const float r = rsqrtf(fmaf(ss, mean, eps));
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const bool turn = kNeox || j < E / 2 ? ln.turn0 : ln.turn1;
    const float from2 = turn ? x2[j] * f.s2[j] : 0.0f, from1 = turn ? x1[j] * f.s1[j] : 0.0f;
    const T y1 = from_f<T>(r * fmaf(x1[j], f.c1[j], -from2));
    const T y2 = from_f<T>(r * fmaf(x2[j], f.c2[j], from1));
    if constexpr (kNeox) {
      x[0].v[j] = y1;
      x[1].v[j] = y2;
    } else if (j < E / 2) {
      x[0].v[2 * j] = y1;
      x[0].v[2 * j + 1] = y2;
    } else {
      x[1].v[2 * j - E] = y1;
      x[1].v[2 * j - E + 1] = y2;
    }
  }
}

// An item is a token and a run of its heads. The factors' registers leave an SM
// 16 warps, and a step is 1 KB a warp: less than memory has to have under way.
// So a lane brings its vectors of the next kQkAhead steps, of the next items
// too, by asynchronous copies into places of its own in shared memory, which
// nobody else reads: there is nothing to wait for but its own copies.
// Measured for 16384 tokens of 64 + 8 heads of 128 (bf16, 604 MB): 107 us, 0.88
// of the copy bandwidth; with two steps ahead in registers, or a ring of whole
// tokens by bulk copies, 147 us. Bound by memory.
constexpr int kQkAhead = 6;

// 16 bytes, asynchronously.
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <typename T, bool kNeox, int kLanes>
__global__ void __launch_bounds__(kQkThreads, 2)
qk_norm_rope_vec_kernel(const __grid_constant__ QkNormParams p, const uint32_t num_items,
                        const FastDiv div_runs, const int heads_per_run) {
  constexpr int E = 16 / sizeof(T);
  constexpr int kHeadsPerStep = 32 / kLanes;
  using V = Vec16<T>;
  __shared__ V ring[kQkAhead][2][kQkThreads];
  const int lane = threadIdx.x % 32;
  const int D = p.head_size;
  const QkLane ln = qk_lane<kNeox, E>(lane % kLanes, p.rot_dim);
  const bool active = lane % kLanes * 2 * E < D;
  const int q_heads = p.heads[0], all_heads = p.heads[0] + p.heads[1];
  const float mean = 1.0f / static_cast<float>(D);
  const uint32_t warps = gridDim.x * (kQkThreads / 32);
  const uint32_t first = blockIdx.x * (kQkThreads / 32) + threadIdx.x / 32;
  const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(&ring[0][0][threadIdx.x]));

  // The step that is brought next: its item, and this lane's head.
  uint32_t far_item = first;
  int far_h = 0, far_last = 0;
  const T *far_q = nullptr, *far_k = nullptr;
  const auto far_start = [&]() {
    if (far_item >= num_items) return;
    const uint32_t t = div_runs.div(far_item);
    const int h_first = static_cast<int>(far_item - t * div_runs.d) * heads_per_run;
    far_h = h_first + lane / kLanes;
    far_last = min(h_first + heads_per_run, all_heads);
    far_q = static_cast<const T*>(p.in[0]) + t * p.in_stride[0];
    far_k = static_cast<const T*>(p.in[1]) + t * p.in_stride[1] -
            static_cast<int64_t>(q_heads) * D;
  };
  const auto bring = [&](int slot) {
    if (far_item < num_items) {
      if (far_h < far_last && active) {
        const T* row = (far_h < q_heads ? far_q : far_k) + static_cast<int64_t>(far_h) * D;
        const uint32_t to = mine + slot * static_cast<uint32_t>(sizeof(ring[0]));
        copy_async16(to, row + ln.e0);
        copy_async16(to + static_cast<uint32_t>(sizeof(ring[0][0])), row + ln.e1);
      }
      far_h += kHeadsPerStep;
      if (far_h - lane / kLanes >= far_last) {  // uniform: the item's last step
        far_item += warps;
        far_start();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  far_start();
#pragma unroll
  for (int u = 0; u + 1 < kQkAhead; ++u) bring(u);

  int slot = 0;
  int64_t next_pos = first < num_items ? qk_position(p, div_runs.div(first)) : 0;
  for (uint32_t item = first; item < num_items; item += warps) {
    const uint32_t t = div_runs.div(item);
    const int h_first = static_cast<int>(item - t * div_runs.d) * heads_per_run;
    const int h_last = min(h_first + heads_per_run, all_heads);
    const int64_t pos = next_pos;
    if (item + warps < num_items) next_pos = qk_position(p, div_runs.div(item + warps));
    const bool ok = pos >= 0 && pos < p.max_position;
    if (!ok && lane == 0 && h_first == 0) {
      raise_flag(p.status, LMCB_DEVICE_FLAG_POSITION_OUT_OF_RANGE);
    }
    QkFactors<T> f;
    int made_for = -1;  // q (0) or k (1) heads
    for (int h0 = h_first; h0 < h_last; h0 += kHeadsPerStep) {
      bring(slot == 0 ? kQkAhead - 1 : slot - 1);
      const int h = h0 + lane / kLanes;
      const bool live = h < h_last && active && ok;
      const int which = h >= q_heads;
      if (live && which != made_for) {
        const QkSource src{which ? p.weight[1] : p.weight[0],
                           which ? p.weight_type[1] : p.weight_type[0], p.cache, p.cache_type,
                           pos * p.rot_dim, p.rot_dim / 2};
        qk_factors<T, kNeox>(src, ln, f);
        made_for = which;
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(kQkAhead - 1) : "memory");
      V x[2] = {ring[slot][0][threadIdx.x], ring[slot][1][threadIdx.x]};
      if (++slot == kQkAhead) slot = 0;
      qk_row<T, kNeox, kLanes>(x, f, ln, mean, p.eps, live);
      if (live) {
        T* row = which ? static_cast<T*>(p.out[1]) + t * p.out_stride[1] +
                             static_cast<int64_t>(h - q_heads) * D
                       : static_cast<T*>(p.out[0]) + t * p.out_stride[0] +
                             static_cast<int64_t>(h) * D;
        *reinterpret_cast<V*>(row + ln.e0) = x[0];
        *reinterpret_cast<V*>(row + ln.e1) = x[1];
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// The same for every other size and alignment: a warp a head row, element by
// element. The second pass reads and writes an element in one lane only, so
// the output may be the input.
template <typename T>
__global__ void __launch_bounds__(kQkThreads)
qk_norm_rope_kernel(const QkNormParams p, const int is_neox, const FastDiv div_heads,
                    const uint32_t num_rows) {
  const int lane = threadIdx.x % 32;
  const int D = p.head_size, rot = p.rot_dim, half = rot / 2;
  for (uint32_t row = blockIdx.x * (kQkThreads / 32) + threadIdx.x / 32; row < num_rows;
       row += gridDim.x * (kQkThreads / 32)) {
    const uint32_t t = div_heads.div(row);
    const int h = static_cast<int>(row - t * div_heads.d);
    const int which = h >= p.heads[0];
    const int64_t head = h - (which ? p.heads[0] : 0);
    const T* in = static_cast<const T*>(p.in[which]) + t * p.in_stride[which] + head * D;
    T* out = static_cast<T*>(p.out[which]) + t * p.out_stride[which] + head * D;
    const int64_t pos = qk_position(p, t);
    if (pos < 0 || pos >= p.max_position) {
      if (lane == 0) raise_flag(p.status, LMCB_DEVICE_FLAG_POSITION_OUT_OF_RANGE);
      continue;  // uniform across the warp
    }
    float ss = 0.0f;
    for (int i = lane; i < D; i += 32) {
      const float v = to_f(in[i]);
      ss = fmaf(v, v, ss);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(ss / static_cast<float>(D) + p.eps);
    const void* w = p.weight[which];
    const int wt = p.weight_type[which];
    for (int i = lane; i < half; i += 32) {
      const int i1 = is_neox ? i : 2 * i;
      const int i2 = is_neox ? i + half : 2 * i + 1;
      const float w1 = w == nullptr ? 1.0f : load_typed(w, wt, i1);
      const float w2 = w == nullptr ? 1.0f : load_typed(w, wt, i2);
      const float c = load_typed(p.cache, p.cache_type, pos * rot + i);
      const float s = load_typed(p.cache, p.cache_type, pos * rot + half + i);
      float y1, y2;
      rotate_pair(to_f(in[i1]) * inv * w1, to_f(in[i2]) * inv * w2, c, s, y1, y2);
      out[i1] = from_f<T>(y1);
      out[i2] = from_f<T>(y2);
    }
    for (int i = rot + lane; i < D; i += 32) {
      const float w1 = w == nullptr ? 1.0f : load_typed(w, wt, i);
      out[i] = from_f<T>(to_f(in[i]) * inv * w1);
    }
  }
}

// True when every access of qk_norm_rope_vec_kernel is a whole aligned vector.
template <typename T>
bool qk_vec_ok(const QkNormParams& p, bool neox) {
  constexpr int E = 16 / sizeof(T);
  const auto aligned = [](const void* a) { return reinterpret_cast<uintptr_t>(a) % 16 == 0; };
  for (int i = 0; i < 2; ++i) {
    if (p.heads[i] == 0) continue;
    if (!aligned(p.in[i]) || !aligned(p.out[i]) || p.in_stride[i] % E != 0 ||
        p.out_stride[i] % E != 0 || (p.weight[i] != nullptr && !aligned(p.weight[i]))) {
      return false;
    }
  }
  if (!aligned(p.cache) || p.head_size % (2 * E) != 0 || p.head_size > 32 * 2 * E) return false;
  // neox: whole vectors in each rotary half and whole vector pairs behind
  // them; else whole vectors rotated. A cache row of any type starts on a
  // vector of the widths read when rot_dim is a multiple of 16 (8 two-byte
  // values, half of a row).
  if (p.rot_dim % 16 != 0) return false;
  return neox ? (p.head_size - p.rot_dim) % (2 * E) == 0 : p.rot_dim % E == 0;
}

template <typename T, bool kNeox, int kLanes>
void launch_qk_vec(const QkNormParams& p, cudaStream_t stream) {
  const int heads = p.heads[0] + p.heads[1];
  const int64_t sms = current_sm_count();
  // A step a warp while warps are left, then longer runs.
  const int64_t steps = (heads + 32 / kLanes - 1) / (32 / kLanes);
  int64_t runs = steps;
  while (runs > 1 && p.num_tokens * (runs / 2) >= sms * 16) runs /= 2;
  int per_run = static_cast<int>((steps + runs - 1) / runs) * (32 / kLanes);
  runs = (heads + per_run - 1) / per_run;
  const int64_t items = p.num_tokens * runs;
  const int64_t want = (items + kQkThreads / 32 - 1) / (kQkThreads / 32);
  const int64_t most = sms * 2;
  qk_norm_rope_vec_kernel<T, kNeox, kLanes>
      <<<static_cast<unsigned>(want < most ? want : most), kQkThreads, 0, stream>>>(
          p, static_cast<uint32_t>(items), FastDiv(static_cast<uint32_t>(runs)), per_run);
}

template <typename T, bool kNeox>
void launch_qk_lanes(const QkNormParams& p, cudaStream_t stream) {
  constexpr int E = 16 / sizeof(T);
  const int lanes = p.head_size / (2 * E);
  if (lanes <= 4) launch_qk_vec<T, kNeox, 4>(p, stream);
  else if (lanes <= 8) launch_qk_vec<T, kNeox, 8>(p, stream);
  else if (lanes <= 16) launch_qk_vec<T, kNeox, 16>(p, stream);
  else launch_qk_vec<T, kNeox, 32>(p, stream);
}

template <typename T>
cudaError_t launch_qk(const QkNormParams& p, bool neox, cudaStream_t stream) {
  if (qk_vec_ok<T>(p, neox)) {
    if (neox) launch_qk_lanes<T, true>(p, stream);
    else launch_qk_lanes<T, false>(p, stream);
  } else {
    const int heads = p.heads[0] + p.heads[1];
    const int64_t rows = p.num_tokens * heads;
    const int64_t want = (rows + kQkThreads / 32 - 1) / (kQkThreads / 32);
    const int64_t most = static_cast<int64_t>(current_sm_count()) * 8;
    qk_norm_rope_kernel<T><<<static_cast<unsigned>(want < most ? want : most), kQkThreads, 0,
                             stream>>>(p, neox ? 1 : 0, FastDiv(static_cast<uint32_t>(heads)),
                                       static_cast<uint32_t>(rows));
  }
  return cudaGetLastError();
}

}  // namespace
}  // namespace lmcb

extern "C" {

int lmcb_rotary_embedding_k_fused(const void* oldPositions, const void* newPositions, int posType,
                                  void* key, int keyType, int64_t numTokens, int64_t numHeads,
                                  int64_t headSize, int64_t keyTokenStride,
                                  const void* cosSinCache, int cacheType, int64_t rotDim,
                                  int64_t maxPosition, int isNeox, void* stream) {
  lmcb::clear_error();
  const char* who = "rotary_embedding_k_fused";
  if (!lmcb::float_type(keyType) || !lmcb::float_type(cacheType)) {
    return lmcb::fail(LMCB_ERR_UNSUPPORTED_DTYPE, std::string(who) + ": ScalarType not supported.");
  }
  if (posType != LMCB_DTYPE_INT64 && posType != LMCB_DTYPE_INT32) {
    return lmcb::fail(LMCB_ERR_UNSUPPORTED_DTYPE,
                      std::string(who) + ": positions must be int64 or int32.");
  }
  if (numTokens < 0 || numHeads < 0 || headSize <= 0 || rotDim <= 0 || rotDim % 2 != 0 ||
      rotDim > headSize || maxPosition <= 0 || keyTokenStride < numHeads * headSize ||
      numTokens > 0x7fffffff || numHeads * (rotDim / 2) > 0x7fffffff) {
    return lmcb::fail(LMCB_ERR_INVALID_ARGUMENT,
                      std::string(who) + ": invalid shape (rot_dim must be even and <= head_size).");
  }
  if (numTokens == 0 || numHeads == 0) return LMCB_OK;
  if (oldPositions == nullptr || newPositions == nullptr || key == nullptr ||
      cosSinCache == nullptr) {
    return lmcb::fail(LMCB_ERR_INVALID_ARGUMENT, std::string(who) + ": NULL pointer.");
  }
  lmcb::RopeParams p;
  p.old_pos = oldPositions;
  p.new_pos = newPositions;
  p.key = key;
  p.cache = cosSinCache;
  p.num_tokens = numTokens;
  p.num_heads = numHeads;
  p.head_size = headSize;
  p.token_stride = keyTokenStride;
  p.rot_dim = rotDim;
  p.max_position = maxPosition;
  p.is_neox = isNeox ? 1 : 0;
  p.div_half = lmcb::FastDiv(static_cast<uint32_t>(rotDim / 2));
  p.status = lmcb::device_status_ptr();
  if (p.status == nullptr) return LMCB_ERR_CUDA;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t err;
  switch (keyType) {
    case LMCB_DTYPE_FP32: err = lmcb::launch_rope_cache<float>(p, cacheType, posType, s); break;
    case LMCB_DTYPE_BF16:
      err = lmcb::launch_rope_cache<__nv_bfloat16>(p, cacheType, posType, s);
      break;
    default: err = lmcb::launch_rope_cache<__half>(p, cacheType, posType, s); break;
  }
  if (err != cudaSuccess) return lmcb::cuda_fail(err, who);
  return LMCB_OK;
}

int lmcb_qk_norm_rope(const void* query, const void* key, int type, int64_t queryTokenStride,
                      int64_t keyTokenStride, const void* queryWeight, int queryWeightType,
                      const void* keyWeight, int keyWeightType, const void* positions, int posType,
                      const void* cosSinCache, int cacheType, int64_t rotDim, int64_t maxPosition,
                      int isNeox, double eps, int64_t numTokens, int64_t numQueryHeads,
                      int64_t numKeyHeads, int64_t headSize, void* queryOut,
                      int64_t queryOutStride, void* keyOut, int64_t keyOutStride, void* stream) {
  lmcb::clear_error();
  const std::string who = "qk_norm_rope";
  if (!lmcb::float_type(type) || !lmcb::float_type(cacheType) ||
      (queryWeight != nullptr && !lmcb::float_type(queryWeightType)) ||
      (keyWeight != nullptr && !lmcb::float_type(keyWeightType))) {
    return lmcb::fail(LMCB_ERR_UNSUPPORTED_DTYPE, who + ": ScalarType not supported.");
  }
  if (posType != LMCB_DTYPE_INT64 && posType != LMCB_DTYPE_INT32) {
    return lmcb::fail(LMCB_ERR_UNSUPPORTED_DTYPE, who + ": positions must be int64 or int32.");
  }
  if (numTokens < 0 || numQueryHeads < 0 || numKeyHeads < 0 || headSize <= 0 ||
      headSize > 65536 || rotDim < 0 || rotDim % 2 != 0 || rotDim > headSize ||
      maxPosition <= 0 || numQueryHeads > 65536 || numKeyHeads > 65536 ||
      queryTokenStride < numQueryHeads * headSize || queryOutStride < numQueryHeads * headSize ||
      keyTokenStride < numKeyHeads * headSize || keyOutStride < numKeyHeads * headSize) {
    return lmcb::fail(LMCB_ERR_INVALID_ARGUMENT,
                      who + ": invalid shape (rot_dim must be even and <= head_size).");
  }
  const int64_t heads = numQueryHeads + numKeyHeads;
  if (numTokens == 0 || heads == 0) return LMCB_OK;
  if (numTokens > 0x7fffffff / heads) {
    return lmcb::fail(LMCB_ERR_INVALID_ARGUMENT, who + ": too many head rows in one call.");
  }
  if ((numQueryHeads > 0 && (query == nullptr || queryOut == nullptr)) ||
      (numKeyHeads > 0 && (key == nullptr || keyOut == nullptr)) || positions == nullptr ||
      (rotDim > 0 && cosSinCache == nullptr)) {
    return lmcb::fail(LMCB_ERR_INVALID_ARGUMENT, who + ": NULL pointer.");
  }
  lmcb::QkNormParams p;
  p.in[0] = query;
  p.in[1] = key;
  p.out[0] = queryOut;
  p.out[1] = keyOut;
  p.weight[0] = queryWeight;
  p.weight[1] = keyWeight;
  p.weight_type[0] = queryWeightType;
  p.weight_type[1] = keyWeightType;
  p.in_stride[0] = queryTokenStride;
  p.in_stride[1] = keyTokenStride;
  p.out_stride[0] = queryOutStride;
  p.out_stride[1] = keyOutStride;
  p.positions = positions;
  p.pos64 = posType == LMCB_DTYPE_INT64;
  p.cache = cosSinCache;
  p.cache_type = cacheType;
  p.num_tokens = numTokens;
  p.heads[0] = static_cast<int32_t>(numQueryHeads);
  p.heads[1] = static_cast<int32_t>(numKeyHeads);
  p.head_size = static_cast<int32_t>(headSize);
  p.rot_dim = static_cast<int32_t>(rotDim);
  p.max_position = maxPosition;
  p.eps = static_cast<float>(eps);
  p.status = lmcb::device_status_ptr();
  if (p.status == nullptr) return LMCB_ERR_CUDA;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t err;
  switch (type) {
    case LMCB_DTYPE_FP32: err = lmcb::launch_qk<float>(p, isNeox != 0, s); break;
    case LMCB_DTYPE_BF16: err = lmcb::launch_qk<__nv_bfloat16>(p, isNeox != 0, s); break;
    default: err = lmcb::launch_qk<__half>(p, isNeox != 0, s); break;
  }
  if (err != cudaSuccess) return lmcb::cuda_fail(err, who.c_str());
  return LMCB_OK;
}

}  // extern "C"
