// kv4_attention.cuh -- what the attention kernels over the 4-bit paged cache
// share: their parameters, what a request and its visible keys are, and small
// wrappers of PTX instructions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "kv4.cuh"
#include "lmcache_b200.h"

namespace lmcb {
namespace kv4 {

struct AttnParams {
  const void* q;
  int q_vec;         // query rows are 16-byte aligned
  int64_t q_stride;  // elements between query tokens
  void* out;
  int out_vec;       // output rows are 16-byte aligned
  int64_t out_stride;
  const int32_t* cache;
  int64_t half_words;  // words from a K row to its V row
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
  int32_t group;  // query heads a KV head
  FastDiv div_group;
  float scale_log2;
  int32_t window;
  int32_t sinks;
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
  r.len = p.seq_lens[b];
  bool bad = lo < 0 || hi < lo || hi > p.num_rows;
  if (bad) lo = hi = 0;
  r.row0 = lo;
  r.n = hi - lo;
  if (r.n > p.max_query) {
    bad = true;
    r.n = 0;
  }
  const int64_t cap = static_cast<int64_t>(p.table_cols) * p.div_block.d;
  if (r.len < 0 || r.len > cap) {
    bad = true;
    r.len = 0;
  }
  if (bad && flag) raise_flag(p.status, LMCB_DEVICE_FLAG_LENGTH_OUT_OF_RANGE);
  return r;
}

// The last key that a query at `pos` (which may lie before the first key) does
// not see for its window; -1: none. Never below -1, whatever the two are.
__device__ __forceinline__ int32_t window_end(const AttnParams& p, int32_t pos) {
  return p.window > 0 && pos >= p.window ? pos - p.window : -1;
}

// The keys that any query of a run of positions [p0, p1] sees, as one virtual
// range [0, count): first `head` first tokens, then the tokens from `first` on.
struct KeyRange {
  int32_t count, head, first;
};

__device__ __forceinline__ KeyRange key_range(const AttnParams& p, int32_t p0, int32_t p1) {
  KeyRange k;
  if (p1 < 0) return KeyRange{0, 0, 0};
  k.first = window_end(p, p0) + 1;
  k.head = min(p.sinks, k.first);
  k.count = k.head + p1 + 1 - k.first;
  return k;
}

__device__ __forceinline__ int32_t key_of(const KeyRange& k, int32_t v) {
  return v < k.head ? v : k.first + (v - k.head);
}

// The cache row of virtual token v, or -1 where v is behind the range or its
// page is not in the cache (flagged: the key is not seen).
__device__ __forceinline__ int32_t row_of(const AttnParams& p, const int32_t* table,
                                          const KeyRange& k, int32_t v) {
  if (v >= k.count) return -1;
  const int32_t key = key_of(k, v);
  const int32_t size = static_cast<int32_t>(p.div_block.d);
  const int32_t blk = static_cast<int32_t>(p.div_block.div(static_cast<uint32_t>(key)));
  const int32_t page = __ldg(table + blk);
  if (page < 0 || page >= p.num_blocks) {
    raise_flag(p.status, LMCB_DEVICE_FLAG_SLOT_OUT_OF_RANGE);
    return -1;
  }
  return page * size + (key - blk * size);
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

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T> __device__ __forceinline__ float elem_to_float(T v);
template <> __device__ __forceinline__ float elem_to_float<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <> __device__ __forceinline__ float elem_to_float<__half>(__half v) {
  return __half2float(v);
}

template <typename T> __device__ __forceinline__ uint32_t pack_out(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack_out<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack_out<__half>(float lo, float hi) {
  return pack_half2(lo, hi);
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

// N consecutive output elements (N even).
template <typename T, int N>
__device__ __forceinline__ void store_out(T* dst, bool vec, const float (&x)[N]) {
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) w[i] = pack_out<T>(x[2 * i], x[2 * i + 1]);
  if (vec && N % 8 == 0) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      reinterpret_cast<uint4*>(dst)[i] =
          make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  } else if (vec && N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      reinterpret_cast<uint2*>(dst)[i] = make_uint2(w[2 * i], w[2 * i + 1]);
    }
  } else {
    const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < N; ++i) dst[i] = e[i];
  }
}

// 1 / l for a row's sum of probabilities: a row that saw nothing (l = 0) has
// zeros for an output, and a NaN stays one.
__device__ __forceinline__ float inverse_sum(float l) {
  return l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
}

// ---------------------------------------------------------------------------
// PTX
// ---------------------------------------------------------------------------

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count)
               : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void mbar_arrive_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)),
               "r"(bytes)
               : "memory");
}

__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}

// Every wait is bounded: after the limit it gives up, and its caller raises
// LMCB_DEVICE_FLAG_WAIT_TIMEOUT and leaves.
constexpr uint32_t kWaitLimit = 1u << 22;

__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity,
                                          uint32_t limit = kWaitLimit) {
  for (uint32_t i = 0; i < limit; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
  }
  return false;
}

// The same for a whole warp, whose lanes are told the same: were each to poll for
// itself, a phase that ends as the last polls go out could send them different
// ways, in front of instructions that take the whole warp. `limit` is the same for
// all.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity,
                                          uint32_t limit = kWaitLimit) {
  for (uint32_t i = 0; i < limit; ++i) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  }
  return false;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace kv4
}  // namespace lmcb
