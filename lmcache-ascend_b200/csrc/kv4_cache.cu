// kv4_cache.cu -- rows into and out of the paged KV cache held in 4 bits
// (kv4_store, kv4_load; layout in kv4.cuh).
//
// A head row x of D values keeps z = fp16(min x), s = fp16((max x - min x) r), r the
// fp32 number nearest to 1 / 15, and the codes clamp(rne((x - z) / s), 0, 15); it
// reads back as z + s c. Difference and product are fp32, each rounded once (a
// quotient by 15 gives another fp16 number for one fp32 row in 8,700); s and z are
// fp16 because an attention kernel multiplies by them in fp32 anyway and a row's 4
// bytes are then 1/17 of its 68 (D = 128). NaN counts as 0 and values beyond the
// fp16 range as its ends, so that s and z are finite, and with them every value in
// fp32 and bf16 (in fp16 z + 15 s of a row that spans the whole range may round to
// infinity).
//
// The code is the exact one, see word_of: it depends on no rounding of a
// reciprocal and equals that of any exact computation.
//
// Both kernels are byte movers (2 D bytes of bf16 against D / 2 + 4): D / 8
// lanes share a head row, a lane holds the eight values of one word (one
// 16-byte access of a 16-bit type), and a lane has up to kMost rows in flight.
//
// Measured, 40001 tokens of 8 heads of 128 in bf16 (208 MB each way): load 37 us,
// 5.6 TB/s, bound by memory; store 73 us, 2.8 TB/s, bound by issue slots (76%
// of them used: 176 instructions a warp for two head rows, of which half find the
// codes and the sixth part the row's minimum and maximum). With a division per
// element instead of the corrected product it took 215 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <climits>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "kv4.cuh"
#include "lmcache_b200.h"

namespace lmcb {
namespace {

constexpr int kThreads = 256;
constexpr int kMost = 4;  // head rows in flight per lane

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
  uint32_t items_per_half;  // items of a group of lanes in K, or in V
  FastDiv div_items;        // by items per token
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

// Eight elements as floats; bf16 are the high halves of theirs.
template <typename T>
__device__ __forceinline__ void floats_of(const Eight<T>& x, float (&v)[8]) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float(x.v[i]);
  }
}

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

// Smallest and largest of a head row over the lanes that share it, both NaN
// where the row holds one. 16-bit types compare two values an instruction,
// and (min, -max) is one register on its way through the lanes.
template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };
template <> struct Pair<__half> { using type = __half2; };

template <typename T, int kGroup>
__device__ __forceinline__ void row_range(const Eight<T>& x, bool active, float& lo, float& hi) {
  if constexpr (sizeof(T) == 2) {
    using P = typename Pair<T>::type;
    const P* v = reinterpret_cast<const P*>(&x);
    const P small = __hmin2_nan(__hmin2_nan(v[0], v[1]), __hmin2_nan(v[2], v[3]));
    const P large = __hmax2_nan(__hmax2_nan(v[0], v[1]), __hmax2_nan(v[2], v[3]));
    P both;
    both.x = __hmin_nan(small.x, small.y);
    both.y = __hneg(__hmax_nan(large.x, large.y));
    if (!active) both.x = both.y = from_float<T>(INFINITY);
#pragma unroll
    for (int o = kGroup / 2; o > 0; o >>= 1) {
      both = __hmin2_nan(both, __shfl_xor_sync(0xffffffffu, both, o));
    }
    lo = to_float(both.x);
    hi = -to_float(both.y);
  } else {
    lo = INFINITY;
    hi = -INFINITY;
    bool nan = false;
    if (active) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        nan = nan || x.v[i] != x.v[i];
        lo = fminf(lo, x.v[i]);
        hi = fmaxf(hi, x.v[i]);
      }
    }
    if (nan) hi = INFINITY;  // out of range all the same
#pragma unroll
    for (int o = kGroup / 2; o > 0; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
  }
}

// One word of codes clamp(rne((x - z) / s), 0, 15).
//
// In fp32, y = x / (15 s) - z / (15 s) with an approximate reciprocal, clamped to
// [0, 1] by the multiply-add itself, is off by less than (|x| + |z|) / (15 s)
// 2^-22 <= (2 |z| / s / 15 + 1) 2^-22, so 15 y by (|z| / s + 8) 2^-21. Adding
// 1.5 2^23 rounds 15 y to an integer, ties to even, in the sum's low bits; a
// multiply-add by 16^i puts it in its place, and what the eight exponent fields
// add up to is one constant. Only a word with an element that lies that close to
// the border between two codes is taken again, in 64 bits.
struct Coder {
  float inv, shift, sure;  // 1 / (15 s), -z / (15 s), and how close is too close

  __device__ __forceinline__ Coder(float z, float s) {
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(15.0f * s));
    shift = -z * inv;
    sure = 0.5f - fmaf(fabsf(shift), 15.0f, 8.0f) * 4.7683716e-7f;
  }
};

constexpr float kMagic = 12582912.0f;

// `off` grows to how far the word's elements are from their codes, in steps.
__device__ __forceinline__ uint32_t word_of(const float (&v)[8], const Coder& c, float& off) {
  constexpr uint32_t kBias = 0x4B400000u * 0x11111111u;
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = __saturatef(fmaf(v[i], c.inv, c.shift));
    const float r = fmaf(y, 15.0f, kMagic);
    off = fmaxf(off, fabsf(fmaf(y, 15.0f, kMagic - r)));
    word += __float_as_uint(r) << (4 * i);
  }
  return word - kBias;
}

// z and s of a head row whose values are in [lo, hi].
__device__ __forceinline__ void row_params(float lo, float hi, float& z, float& s) {
  s = __half2float(__float2half_rn(__fmul_rn(hi - lo, 1.0f / 15.0f)));
  // + 0: a zero of either sign is kept as +0, so equal rows have equal words
  z = __half2float(__float2half_rn(lo)) + 0.0f;
}

// A word with elements too close to a border, again, from global memory: their x - z,
// in 64 bits, against a border (k + 1/2) s, which is exact in fp32. k is the
// quotient's floor, or off by one only where the quotient is within an fp32
// rounding of a whole number and both its borders are far. It is at most 14: a
// row that is narrow against its offset has quotients far beyond 15. Out of line
// and apart from the rest, so that the common path keeps its registers.
template <typename T>
__device__ __noinline__ void exact_word(const T* src, float z, float s, int32_t* dst) {
  const Coder c(z, s);
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = finite_half_range(to_float(src[i]));
    const float q = __saturatef(fmaf(x, c.inv, c.shift)) * 15.0f;
    uint32_t code = static_cast<uint32_t>(q + 0.5f);
    if (fabsf(q - rintf(q)) >= c.sure) {
      const double d = static_cast<double>(x) - static_cast<double>(z);
      const float low = fminf(fmaxf(floorf(static_cast<float>(d) / s), 0.0f), 14.0f);
      const double border = static_cast<double>((low + 0.5f) * s);
      const uint32_t k = static_cast<uint32_t>(low);
      code = d > border ? k + 1 : (d < border ? k : (k + 1) & ~1u);
    }
    word |= code << (4 * i);
  }
  *dst = static_cast<int32_t>(word);
}

__device__ __forceinline__ int64_t slot_of(const Kv4Params& p, uint32_t token) {
  return p.slot64 ? static_cast<const int64_t*>(p.slots)[token]
                  : static_cast<int64_t>(static_cast<const int32_t*>(p.slots)[token]);
}

// What a group of lanes takes at once: kHeads consecutive heads of one token's
// K or V row. Items are numbered half-major, then by token, so consecutive
// groups read consecutive memory, and the slot and all addresses are found
// once for kHeads head rows.
struct Item {
  int half;
  uint32_t token;
  int32_t head;   // the first one
  int32_t count;  // heads of it, 0: nothing to do
  int64_t slot;
};

template <int kHeads>
__device__ __forceinline__ Item item_of(const Kv4Params& p, uint64_t at, bool flag) {
  Item it;
  it.half = it.count = 0;
  it.token = it.head = 0;
  it.slot = -1;
  if (at >= 2ull * p.items_per_half) return it;
  it.half = at >= p.items_per_half;
  const uint32_t in_half = static_cast<uint32_t>(at) - (it.half ? p.items_per_half : 0);
  it.token = p.div_items.div(in_half);
  it.head = static_cast<int32_t>(in_half - it.token * p.div_items.d) * kHeads;
  it.slot = slot_of(p, it.token);
  if (it.slot >= p.num_rows) {
    if (flag) raise_flag(p.status, LMCB_DEVICE_FLAG_SLOT_OUT_OF_RANGE);
    it.slot = -1;
  }
  if (it.slot >= 0) it.count = min(kHeads, p.num_heads - it.head);
  return it;
}

// The head rows x of a group into the cache. kWild: some row of the warp holds
// NaN or a value beyond the fp16 range. Returns a bit for each row whose word
// of this lane has an element too close to a border.
template <typename T, int kGroup, int kHeads, bool kFull, bool kWild>
__device__ __forceinline__ uint32_t store_rows(const Eight<T> (&x)[kHeads], float (&lo)[kHeads],
                                               float (&hi)[kHeads], bool active, int count,
                                               int lane, int words, int32_t* codes,
                                               int32_t* params) {
  uint32_t close = 0;
#pragma unroll
  for (int k = 0; k < kHeads; ++k) {
    float v[8];
    floats_of(x[k], v);
    if constexpr (kWild) {
      lo[k] = INFINITY;
      hi[k] = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = finite_half_range(v[i]);
        if (active) {
          lo[k] = fminf(lo[k], v[i]);
          hi[k] = fmaxf(hi[k], v[i]);
        }
      }
#pragma unroll
      for (int o = kGroup / 2; o > 0; o >>= 1) {
        lo[k] = fminf(lo[k], __shfl_xor_sync(0xffffffffu, lo[k], o));
        hi[k] = fmaxf(hi[k], __shfl_xor_sync(0xffffffffu, hi[k], o));
      }
    }
    float z, s;
    row_params(lo[k], hi[k], z, s);
    const Coder c(z, s);
    float off = 0.0f;
    uint32_t word = word_of(v, c, off);
    if (s == 0.0f) word = 0;  // one value only: z
    if ((kFull ? count > 0 : k < count) && active) {
      codes[k * words] = static_cast<int32_t>(word);
      if (s > 0.0f && off >= c.sure) close |= 1u << k;
      if (lane == 0) {
        params[k] = static_cast<int32_t>(
            static_cast<uint32_t>(__half_as_ushort(__float2half_rn(s))) |
            (static_cast<uint32_t>(__half_as_ushort(__float2half_rn(z))) << 16));
      }
    }
  }
  return close;
}

// kGroup lanes share a head row (D <= 8 * kGroup).
// kFull: kHeads divides the heads.
template <typename T, int kGroup, int kHeads, bool kVec, bool kFull>
__global__ void __launch_bounds__(kThreads, 4)
kv4_store_kernel(const __grid_constant__ Kv4Params p) {
  const int lane = threadIdx.x % kGroup;
  const int D = p.head_size;
  const bool active = lane * 8 < D;
  constexpr uint32_t kGroups = kThreads / kGroup;
  for (uint64_t base = static_cast<uint64_t>(blockIdx.x) * kGroups; base < 2ull * p.items_per_half;
       base += static_cast<uint64_t>(gridDim.x) * kGroups) {
    const Item it = item_of<kHeads>(p, base + threadIdx.x / kGroup, lane == 0);
    Eight<T> x[kHeads] = {};
    const T* src = static_cast<const T*>(it.half ? p.src[1] : p.src[0]) +
                   static_cast<int64_t>(it.token) *
                       (it.half ? p.token_stride[1] : p.token_stride[0]) +
                   static_cast<int64_t>(it.head) * D + lane * 8;
    if (it.count > 0 && active) {
#pragma unroll
      for (int k = 0; k < kHeads; ++k) {
        if (kFull || k < it.count) x[k] = load8<T, kVec>(src + k * D);
      }
    }
    int32_t* row = p.cache + (it.half ? p.half_words : 0) + it.slot * p.row_words;
    int32_t* codes = row + static_cast<int64_t>(it.head) * (D / 8) + lane;
    int32_t* params = row + static_cast<int64_t>(p.num_heads) * (D / 8) + it.head;
    float lo[kHeads], hi[kHeads];
    bool tame = true;
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
      row_range<T, kGroup>(x[k], active, lo[k], hi[k]);
      tame = tame && lo[k] >= -65504.0f && hi[k] <= 65504.0f;
    }
    uint32_t close;
    if (__all_sync(0xffffffffu, tame)) {
      close = store_rows<T, kGroup, kHeads, kFull, false>(x, lo, hi, active, it.count, lane, D / 8,
                                                          codes, params);
    } else {
      close = store_rows<T, kGroup, kHeads, kFull, true>(x, lo, hi, active, it.count, lane, D / 8,
                                                         codes, params);
    }
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
      if (close & (1u << k)) {
        float z, s;
        row_params(lo[k], hi[k], z, s);
        exact_word<T>(src + k * D, z, s, codes + k * (D / 8));
      }
    }
  }
}

template <typename T, int kGroup, int kHeads, bool kVec>
__global__ void __launch_bounds__(kThreads) kv4_load_kernel(const __grid_constant__ Kv4Params p) {
  const int lane = threadIdx.x % kGroup;
  const int D = p.head_size;
  if (lane * 8 >= D) return;
  constexpr uint32_t kGroups = kThreads / kGroup;
  for (uint64_t at = static_cast<uint64_t>(blockIdx.x) * kGroups + threadIdx.x / kGroup;
       at < 2ull * p.items_per_half; at += static_cast<uint64_t>(gridDim.x) * kGroups) {
    const Item it = item_of<kHeads>(p, at, lane == 0);
    if (it.count == 0) continue;
    const int32_t* row = p.cache + (it.half ? p.half_words : 0) + it.slot * p.row_words;
    const int32_t* codes = row + static_cast<int64_t>(it.head) * (D / 8) + lane;
    const int32_t* params = row + static_cast<int64_t>(p.num_heads) * (D / 8) + it.head;
    uint32_t word[kHeads], par[kHeads];
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
      if (k < it.count) {
        word[k] = static_cast<uint32_t>(codes[k * (D / 8)]);
        par[k] = static_cast<uint32_t>(params[k]);
      }
    }
    T* dst = static_cast<T*>(it.half ? p.dst[1] : p.dst[0]) +
             static_cast<int64_t>(it.token) * (it.half ? p.token_stride[1] : p.token_stride[0]) +
             static_cast<int64_t>(it.head) * D + lane * 8;
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
      if (k >= it.count) continue;
      const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(par[k])));
      const float z = __half2float(__ushort_as_half(static_cast<unsigned short>(par[k] >> 16)));
      Eight<T> out;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // 2^23 + code as a float's bits, less 2^23: the code, exactly
        const float c = __uint_as_float(((word[k] >> (4 * i)) & 15u) | 0x4B000000u) - 8388608.0f;
        out.v[i] = from_float<T>(__fmaf_rn(c, s, z));
      }
      store8<T, kVec>(dst + k * D, out);
    }
  }
}

template <typename T, int kGroup, int kHeads, bool kVec>
void launch_items(Kv4Params p, bool store, cudaStream_t stream) {
  const uint32_t per_token = static_cast<uint32_t>((p.num_heads + kHeads - 1) / kHeads);
  p.items_per_half = static_cast<uint32_t>(p.num_tokens) * per_token;
  p.div_items = FastDiv(per_token);
  constexpr uint32_t kPerCta = kThreads / kGroup;
  const uint64_t want = (2ull * p.items_per_half + kPerCta - 1) / kPerCta;
  const uint64_t most = static_cast<uint64_t>(current_sm_count()) * 8;
  const unsigned grid = static_cast<unsigned>(want < most ? want : most);
  if (store) {
    if (p.num_heads % kHeads == 0) {
      kv4_store_kernel<T, kGroup, kHeads, kVec, true><<<grid, kThreads, 0, stream>>>(p);
    } else {
      kv4_store_kernel<T, kGroup, kHeads, kVec, false><<<grid, kThreads, 0, stream>>>(p);
    }
  } else {
    kv4_load_kernel<T, kGroup, kHeads, kVec><<<grid, kThreads, 0, stream>>>(p);
  }
}

template <typename T, int kGroup, bool kVec>
void launch(const Kv4Params& p, bool store, cudaStream_t stream) {
  // Few head rows are spread over the lanes; many are taken kMost at a time.
  const int64_t rows = static_cast<int64_t>(p.num_tokens) * p.num_heads * 2;
  const int64_t lanes = static_cast<int64_t>(current_sm_count()) * 1024;
  if (p.num_heads == 1 || rows * kGroup <= lanes) {
    launch_items<T, kGroup, 1, kVec>(p, store, stream);
  } else {
    launch_items<T, kGroup, kMost, kVec>(p, store, stream);
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
