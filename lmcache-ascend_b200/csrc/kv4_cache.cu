// kv4_cache.cu -- rows into and out of the paged KV cache held in 4 bits
// (kv4_store, kv4_load; layout in kv4.cuh).
//
// A head row x of D values keeps z = fp16(min x), s = fp16((max x - min x) /
// 15) and the codes clamp(rne((x - z) / s), 0, 15); it reads back as z + s c.
// Minimum, difference and quotient are fp32, each rounded once; s and z are
// fp16 because an attention kernel multiplies by them in fp32 anyway and a
// row's 4 bytes are then 1/17 of its 68 (D = 128). NaN counts as 0 and values
// beyond the fp16 range as its ends, so that every row is finite.
//
// The code is the exact one: (x - z) * (1 / s) in fp32 is off by less than
// 2^-17 for quotients up to 17, and a lane whose quotient lies that close to a
// border between two codes repeats it in 64 bits. So the codes depend on no
// rounding of the reciprocal and equal those of any exact computation.
//
// Both kernels are byte movers (2 D bytes of bf16 against D / 2 + 4): D / 8
// lanes share a head row, a lane holds the eight values of one word (one
// 16-byte access of a 16-bit type), and a lane has kRows rows in flight.
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

constexpr int kThreads = 256;
constexpr int kRows = 4;  // head rows in flight per lane

struct Kv4Params {
  const void* src[2];       // store: key, value rows
  void* dst[2];             // load: key, value rows
  int64_t token_stride[2];  // elements between tokens of key, value
  int32_t* cache;           // K half; V half at cache + half_words
  int64_t half_words;
  int64_t row_words;
  int64_t num_rows;  // slots in each half
  const void* slots;
  int slot64;
  int32_t num_tokens;
  int32_t num_heads;
  int32_t head_size;
  uint32_t rows_per_half;  // num_tokens * num_heads
  FastDiv div_heads;
  unsigned int* status;
};

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_float<__half>(float v) {
  return __float2half_rn(v);
}

// Eight consecutive elements: 16-byte pieces where the host has checked the
// alignment (kVec), else one element at a time.
template <typename T>
struct alignas(16) Eight {
  T v[8];
};

template <typename T, bool kVec>
__device__ __forceinline__ Eight<T> load8(const T* src) {
  Eight<T> out;
  if constexpr (kVec) {
    constexpr int kPieces = sizeof(T) / 2;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      reinterpret_cast<uint4*>(&out)[i] = reinterpret_cast<const uint4*>(src)[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) out.v[i] = src[i];
  }
  return out;
}

template <typename T, bool kVec>
__device__ __forceinline__ void store8(T* dst, const Eight<T>& in) {
  if constexpr (kVec) {
    constexpr int kPieces = sizeof(T) / 2;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(&in)[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = in.v[i];
  }
}

__device__ __forceinline__ float finite_half_range(float x) {
  // NaN -> 0 first: fmin / fmax would return the bound for it.
  x = x != x ? 0.0f : x;
  return fminf(fmaxf(x, -65504.0f), 65504.0f);
}

// clamp(rne((x - z) / s), 0, 15), exact. `inv` is 1 / s rounded.
__device__ __forceinline__ uint32_t code_of(float x, float z, float s, float inv) {
  const float q = (x - z) * inv;
  const float r = rintf(q);
  if (fabsf(fabsf(q - r) - 0.5f) < 1.0f / 65536.0f) {
    const double exact = (static_cast<double>(x) - static_cast<double>(z)) / static_cast<double>(s);
    return static_cast<uint32_t>(fmin(fmax(rint(exact), 0.0), 15.0));
  }
  return static_cast<uint32_t>(fminf(fmaxf(r, 0.0f), 15.0f));
}

// A row of the work list: rows are numbered half-major (K, then V), then by
// token, then by head, so consecutive rows are consecutive in memory on the
// 16/32-bit side.
struct RowRef {
  int half;
  uint32_t token;
  uint32_t head;
};

__device__ __forceinline__ RowRef row_ref(const Kv4Params& p, uint32_t row) {
  RowRef r;
  r.half = row >= p.rows_per_half;
  const uint32_t in_half = r.half ? row - p.rows_per_half : row;
  r.token = p.div_heads.div(in_half);
  r.head = in_half - r.token * p.div_heads.d;
  return r;
}

__device__ __forceinline__ int64_t slot_of(const Kv4Params& p, uint32_t token) {
  return p.slot64 ? static_cast<const int64_t*>(p.slots)[token]
                  : static_cast<int64_t>(static_cast<const int32_t*>(p.slots)[token]);
}

// kGroup lanes share a head row (D <= 8 * kGroup).
template <typename T, int kGroup, bool kVec>
__global__ void __launch_bounds__(kThreads) kv4_store_kernel(const Kv4Params p) {
  const int lane = threadIdx.x % kGroup;
  const bool active = lane * 8 < p.head_size;
  const uint32_t total = 2 * p.rows_per_half;
  constexpr uint32_t kGroups = kThreads / kGroup;
  const int words = p.head_size / 8;
  for (uint64_t r0 = static_cast<uint64_t>(blockIdx.x) * (kGroups * kRows) + threadIdx.x / kGroup;
       r0 - threadIdx.x / kGroup < total; r0 += static_cast<uint64_t>(gridDim.x) * kGroups * kRows) {
    Eight<T> x[kRows];
    int64_t slot[kRows];
    RowRef ref[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const uint64_t row = r0 + k * kGroups;
      slot[k] = -1;
      if (row < total) {
        ref[k] = row_ref(p, static_cast<uint32_t>(row));
        slot[k] = slot_of(p, ref[k].token);
        if (active) {
          const T* src = static_cast<const T*>(p.src[ref[k].half]) +
                         static_cast<int64_t>(ref[k].token) * p.token_stride[ref[k].half] +
                         static_cast<int64_t>(ref[k].head) * p.head_size + lane * 8;
          x[k] = load8<T, kVec>(src);
        }
        if (slot[k] >= p.num_rows) {
          if (lane == 0) raise_flag(p.status, LMCB_DEVICE_FLAG_SLOT_OUT_OF_RANGE);
          slot[k] = -1;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      float v[8];
      float lo = INFINITY, hi = -INFINITY;
      if (active && slot[k] >= 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[i] = finite_half_range(to_float(x[k].v[i]));
          lo = fminf(lo, v[i]);
          hi = fmaxf(hi, v[i]);
        }
      }
#pragma unroll
      for (int o = kGroup / 2; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      if (!active || slot[k] < 0) continue;
      const __half sh = __float2half_rn(__fdiv_rn(hi - lo, 15.0f));
      // + 0: a zero of either sign is kept as +0, so equal rows have equal words
      const float z = __half2float(__float2half_rn(lo)) + 0.0f;
      const __half zh = __float2half_rn(z);
      const float s = __half2float(sh);
      uint32_t word = 0;
      if (s > 0.0f) {
        const float inv = __frcp_rn(s);
#pragma unroll
        for (int i = 0; i < 8; ++i) word |= code_of(v[i], z, s, inv) << (4 * i);
      }
      int32_t* dst = p.cache + (ref[k].half ? p.half_words : 0) + slot[k] * p.row_words;
      dst[static_cast<int64_t>(ref[k].head) * words + lane] = static_cast<int32_t>(word);
      if (lane == 0) {
        dst[static_cast<int64_t>(p.num_heads) * words + ref[k].head] = static_cast<int32_t>(
            static_cast<uint32_t>(__half_as_ushort(sh)) |
            (static_cast<uint32_t>(__half_as_ushort(zh)) << 16));
      }
    }
  }
}

template <typename T, int kGroup, bool kVec>
__global__ void __launch_bounds__(kThreads) kv4_load_kernel(const Kv4Params p) {
  const int lane = threadIdx.x % kGroup;
  if (lane * 8 >= p.head_size) return;
  const uint32_t total = 2 * p.rows_per_half;
  constexpr uint32_t kGroups = kThreads / kGroup;
  const int words = p.head_size / 8;
  for (uint64_t r0 = static_cast<uint64_t>(blockIdx.x) * (kGroups * kRows) + threadIdx.x / kGroup;
       r0 < total; r0 += static_cast<uint64_t>(gridDim.x) * kGroups * kRows) {
    uint32_t word[kRows], par[kRows];
    int64_t slot[kRows];
    RowRef ref[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const uint64_t row = r0 + k * kGroups;
      slot[k] = -1;
      if (row < total) {
        ref[k] = row_ref(p, static_cast<uint32_t>(row));
        slot[k] = slot_of(p, ref[k].token);
        if (slot[k] >= p.num_rows) {
          if (lane == 0) raise_flag(p.status, LMCB_DEVICE_FLAG_SLOT_OUT_OF_RANGE);
          slot[k] = -1;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (slot[k] >= 0) {
        const int32_t* src = p.cache + (ref[k].half ? p.half_words : 0) + slot[k] * p.row_words;
        word[k] = static_cast<uint32_t>(src[static_cast<int64_t>(ref[k].head) * words + lane]);
        par[k] = static_cast<uint32_t>(
            src[static_cast<int64_t>(p.num_heads) * words + ref[k].head]);
      }
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (slot[k] < 0) continue;
      const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(par[k])));
      const float z = __half2float(__ushort_as_half(static_cast<unsigned short>(par[k] >> 16)));
      Eight<T> out;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        out.v[i] = from_float<T>(__fmaf_rn(static_cast<float>((word[k] >> (4 * i)) & 15u), s, z));
      }
      T* dst = static_cast<T*>(p.dst[ref[k].half]) +
               static_cast<int64_t>(ref[k].token) * p.token_stride[ref[k].half] +
               static_cast<int64_t>(ref[k].head) * p.head_size + lane * 8;
      store8<T, kVec>(dst, out);
    }
  }
}

template <typename T, int kGroup, bool kVec>
void launch(const Kv4Params& p, bool store, cudaStream_t stream) {
  constexpr uint32_t kPerCta = kThreads / kGroup * kRows;
  const uint64_t want = (2ull * p.rows_per_half + kPerCta - 1) / kPerCta;
  const uint64_t most = static_cast<uint64_t>(current_sm_count()) * 8;
  const unsigned grid = static_cast<unsigned>(want < most ? want : most);
  if (store) {
    kv4_store_kernel<T, kGroup, kVec><<<grid, kThreads, 0, stream>>>(p);
  } else {
    kv4_load_kernel<T, kGroup, kVec><<<grid, kThreads, 0, stream>>>(p);
  }
}

template <typename T>
cudaError_t dispatch(const Kv4Params& p, bool store, cudaStream_t stream) {
  bool vec = true;
  for (int h = 0; h < 2; ++h) {
    const void* base = store ? p.src[h] : p.dst[h];
    vec = vec && reinterpret_cast<uintptr_t>(base) % 16 == 0 &&
          (p.token_stride[h] * static_cast<int64_t>(sizeof(T))) % 16 == 0;
  }
  // head_size is a multiple of 8, so head rows keep the base's 16-byte alignment.
  if (p.head_size <= 64) {
    vec ? launch<T, 8, true>(p, store, stream) : launch<T, 8, false>(p, store, stream);
  } else if (p.head_size <= 128) {
    vec ? launch<T, 16, true>(p, store, stream) : launch<T, 16, false>(p, store, stream);
  } else {
    vec ? launch<T, 32, true>(p, store, stream) : launch<T, 32, false>(p, store, stream);
  }
  return cudaGetLastError();
}

int run(const char* name, const void* key_in, const void* value_in, void* key_out, void* value_out,
        int type, int64_t key_stride, int64_t value_stride, int32_t* cache, int64_t num_blocks,
        int64_t block_size, const void* slots, int slot_type, int64_t num_tokens,
        int64_t num_heads, int64_t head_size, bool store, void* stream) {
  clear_error();
  const std::string who = name;
  if (type != LMCB_DTYPE_FP32 && type != LMCB_DTYPE_BF16 && type != LMCB_DTYPE_FP16) {
    return fail(LMCB_ERR_UNSUPPORTED_DTYPE, who + ": ScalarType not supported.");
  }
  if (slot_type != LMCB_DTYPE_INT64 && slot_type != LMCB_DTYPE_INT32) {
    return fail(LMCB_ERR_UNSUPPORTED_DTYPE, who + ": slots must be int64 or int32.");
  }
  if (num_tokens < 0 || num_heads < 0 || num_blocks < 0 || block_size < 0 || head_size < 8 ||
      head_size > 256 || head_size % 8 != 0) {
    return fail(LMCB_ERR_INVALID_ARGUMENT,
                who + ": head_size must be a multiple of 8, at most 256.");
  }
  if (num_tokens == 0 || num_heads == 0) return LMCB_OK;
  if (num_heads > INT_MAX / 2 || num_tokens > INT_MAX / 2 / num_heads ||
      key_stride < num_heads * head_size || value_stride < num_heads * head_size ||
      (num_blocks > 0 && block_size > INT_MAX / num_blocks)) {
    return fail(LMCB_ERR_INVALID_ARGUMENT, who + ": invalid shape.");
  }
  if ((store ? key_in == nullptr || value_in == nullptr
             : key_out == nullptr || value_out == nullptr) ||
      slots == nullptr || cache == nullptr) {
    return fail(LMCB_ERR_INVALID_ARGUMENT, who + ": NULL pointer.");
  }
  Kv4Params p;
  p.src[0] = key_in;
  p.src[1] = value_in;
  p.dst[0] = key_out;
  p.dst[1] = value_out;
  p.token_stride[0] = key_stride;
  p.token_stride[1] = value_stride;
  p.cache = cache;
  p.row_words = kv4_row_words(num_heads, head_size);
  p.num_rows = num_blocks * block_size;
  p.half_words = p.num_rows * p.row_words;
  p.slots = slots;
  p.slot64 = slot_type == LMCB_DTYPE_INT64;
  p.num_tokens = static_cast<int32_t>(num_tokens);
  p.num_heads = static_cast<int32_t>(num_heads);
  p.head_size = static_cast<int32_t>(head_size);
  p.rows_per_half = static_cast<uint32_t>(num_tokens * num_heads);
  p.div_heads = FastDiv(static_cast<uint32_t>(num_heads));
  p.status = device_status_ptr();
  if (p.status == nullptr) return LMCB_ERR_CUDA;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t err;
  switch (type) {
    case LMCB_DTYPE_FP32: err = dispatch<float>(p, store, s); break;
    case LMCB_DTYPE_BF16: err = dispatch<__nv_bfloat16>(p, store, s); break;
    default: err = dispatch<__half>(p, store, s); break;
  }
  if (err != cudaSuccess) return cuda_fail(err, name);
  return LMCB_OK;
}

}  // namespace
}  // namespace lmcb

extern "C" {

int64_t lmcb_kv4_row_words(int64_t numHeads, int64_t headSize) {
  if (numHeads <= 0 || numHeads > INT_MAX / 2 || headSize < 8 || headSize > 256 ||
      headSize % 8 != 0) {
    return 0;
  }
  return lmcb::kv4_row_words(numHeads, headSize);
}

int lmcb_kv4_store(const void* key, const void* value, int type, int64_t keyTokenStride,
                   int64_t valueTokenStride, int32_t* kvCache, int64_t numBlocks,
                   int64_t blockSize, const void* slotMapping, int slotType, int64_t numTokens,
                   int64_t numHeads, int64_t headSize, void* stream) {
  return lmcb::run("kv4_store", key, value, nullptr, nullptr, type, keyTokenStride,
                   valueTokenStride, kvCache, numBlocks, blockSize, slotMapping, slotType,
                   numTokens, numHeads, headSize, true, stream);
}

int lmcb_kv4_load(const int32_t* kvCache, int64_t numBlocks, int64_t blockSize,
                  const void* slotMapping, int slotType, void* key, void* value, int type,
                  int64_t keyTokenStride, int64_t valueTokenStride, int64_t numTokens,
                  int64_t numHeads, int64_t headSize, void* stream) {
  return lmcb::run("kv4_load", nullptr, nullptr, key, value, type, keyTokenStride,
                   valueTokenStride, const_cast<int32_t*>(kvCache), numBlocks, blockSize,
                   slotMapping, slotType, numTokens, numHeads, headSize, false, stream);
}

}  // extern "C"
