// paged_batch.cu -- block tables, slot maps, positions and lengths of a batch
// from its request lengths, on the GPU (build_slot_mapping).
//
// Request b has c_b tokens in the paged cache and brings n_b new ones; pages
// hold s tokens. With has_b = ceil(c_b / s) and need_b = ceil((c_b + n_b) / s)
// - has_b, the request takes free pages [f_b, f_b + need_b), f_b the exclusive
// prefix sum of need, and its tokens are tokens [q_b, q_b + n_b) of the batch,
// q_b the exclusive prefix sum of n. Both sums are short (one entry a
// request), so every CTA computes them for itself into shared memory: one
// launch, no wait of one CTA for another. New pages' numbers are then read
// from the free list and not from the table, which other CTAs may still be
// writing; the thread that has a new page's first token writes it there. What is
// left is one search over the prefix sums for each group of consecutive tokens
// and the writes of slots and positions.
//
// Measured: 1021 requests with 765,000 tokens 14.0 us, where writing and reading
// the 12.9 MB takes 2.0. Nearly all of it is time in the kernel (13.7 us in a
// profile): 584 instructions a warp at 40% of the issue slots, in 191 CTAs of 1024
// threads. SMs are busy for 8.7 us on average and 11.8 where they have two CTAs, 43
// of the 148; the stalls are loads (the lengths, table and free list) and shared
// memory (scans and searches). 8 requests with a token each 6.4 us, which is the
// call itself (256 threads there; 1024 cost 2 us more, and nothing from 96 requests
// on).
#include <cuda_runtime.h>
#include <stdint.h>

#include <climits>
#include <string>

#include "common.cuh"
#include "lmcache_b200.h"

namespace lmcb {
namespace {

constexpr int kBatchThreads = 1024;  // 256 where they cover requests and tokens
constexpr int kBatchMaxRequests = 16384;  // 12 bytes of shared memory each
constexpr int kTokensPerThread = 4;

struct BatchParams {
  const void* context_lens;
  const void* query_lens;
  int len64;  // lengths are int64 (else int32)
  int32_t num_requests;
  int32_t* table;
  int64_t table_stride;
  int32_t table_cols;
  int32_t row_tokens;  // table_cols * block size
  const int32_t* free_blocks;
  int32_t num_free;
  FastDiv div_block;
  int32_t num_tokens;
  void* slots;
  void* positions;
  int aligned;  // slots and positions start on 16 bytes
  int32_t* query_start;
  int32_t* seq_lens;
  int32_t* blocks_used;
  unsigned int* status;
};

// A length as an int32; what does not fit counts as 0 (negative) or the
// largest int32 and raises the flag.
__device__ __forceinline__ int32_t load_len(const void* p, int len64, int i, unsigned int* status) {
  const int64_t v = len64 ? static_cast<const int64_t*>(p)[i]
                          : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
  if (v < 0 || v >= INT_MAX) {
    raise_flag(status, LMCB_DEVICE_FLAG_LENGTH_OUT_OF_RANGE);
    return v < 0 ? 0 : INT_MAX - 1;
  }
  return static_cast<int32_t>(v);
}

__device__ __forceinline__ int32_t clamp31(int64_t v) {
  return v > INT_MAX ? INT_MAX : static_cast<int32_t>(v);
}

// Pages that `tokens` (< 2^32) tokens fill, at most the table's width.
__device__ __forceinline__ int32_t pages_of(uint32_t tokens, const BatchParams& p) {
  if (tokens >= static_cast<uint32_t>(p.row_tokens)) return p.table_cols;
  return tokens == 0 ? 0 : static_cast<int32_t>(p.div_block.div(tokens - 1)) + 1;
}

// Index of the last entry <= key in ascending a[0..n) (a[0] <= key).
__device__ __forceinline__ int last_le(const int32_t* a, int n, int32_t key) {
  int lo = 0, hi = n;  // a[lo] <= key < a[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= key) lo = mid; else hi = mid;
  }
  return lo;
}

// Sums that stop at INT_MAX: what lies behind it is behind every table and
// every token too.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) {
  return min(a + b, static_cast<uint32_t>(INT_MAX));
}

// Inclusive sums over a warp.
__device__ __forceinline__ void warp_sums(uint32_t& a, uint32_t& b, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, a, o);
    const uint32_t y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) {
      a = add_sat(a, x);
      b = add_sat(b, y);
    }
  }
}

template <typename SlotT>
__global__ void __launch_bounds__(kBatchThreads) build_slot_mapping_kernel(const BatchParams p) {
  extern __shared__ int32_t batch_smem[];
  const int B = p.num_requests;
  int32_t* s_start = batch_smem;  // [B] first token of the request
  int32_t* s_first = s_start + B; // [B] first free-list entry of the request
  int32_t* s_ctx = s_first + B;   // [B] tokens in the cache
  __shared__ uint32_t s_warp[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;

  // Prefix sums, a request a thread and round.
  uint32_t base_tok = 0, base_page = 0;
  for (int b0 = 0; b0 < B; b0 += threads) {
    const int b = b0 + tid;
    int32_t ctx = 0, fresh = 0, need = 0;
    if (b < B) {
      ctx = load_len(p.context_lens, p.len64, b, p.status);
      fresh = load_len(p.query_lens, p.len64, b, p.status);
      need = pages_of(static_cast<uint32_t>(ctx) + fresh, p) - pages_of(ctx, p);
    }
    uint32_t tok = fresh, page = need;
    warp_sums(tok, page, lane);
    if (lane == 31) {
      s_warp[0][warp] = tok;
      s_warp[1][warp] = page;
    }
    __syncthreads();
    if (warp == 0) {
      uint32_t t = lane < threads / 32 ? s_warp[0][lane] : 0;
      uint32_t g = lane < threads / 32 ? s_warp[1][lane] : 0;
      warp_sums(t, g, lane);
      s_warp[0][lane] = t;
      s_warp[1][lane] = g;
    }
    __syncthreads();
    const uint32_t before_tok = warp > 0 ? add_sat(base_tok, s_warp[0][warp - 1]) : base_tok;
    const uint32_t before_page = warp > 0 ? add_sat(base_page, s_warp[1][warp - 1]) : base_page;
    if (b < B) {
      // this thread's own come off again, but for sums that have stopped
      const uint32_t tok_sum = add_sat(before_tok, tok), page_sum = add_sat(before_page, page);
      const uint32_t st = tok_sum == INT_MAX ? tok_sum : tok_sum - fresh;
      s_ctx[b] = ctx;
      s_start[b] = static_cast<int32_t>(min(st, static_cast<uint32_t>(p.num_tokens)));
      s_first[b] = static_cast<int32_t>(page_sum == INT_MAX ? page_sum : page_sum - need);
      if (blockIdx.x == 0) {
        p.query_start[b] = s_start[b];
        p.seq_lens[b] = clamp31(static_cast<int64_t>(ctx) + fresh);
      }
    }
    base_tok = add_sat(base_tok, s_warp[0][31]);
    base_page = add_sat(base_page, s_warp[1][31]);
    __syncthreads();  // s_warp is rewritten by the next round
  }
  const int32_t total_tok =
      static_cast<int32_t>(min(base_tok, static_cast<uint32_t>(p.num_tokens)));
  const int32_t total_page = static_cast<int32_t>(base_page);
  if (blockIdx.x == 0 && tid == 0) {
    p.query_start[B] = total_tok;
    p.blocks_used[0] = total_page;
    if (base_tok > static_cast<uint32_t>(p.num_tokens)) {
      raise_flag(p.status, LMCB_DEVICE_FLAG_LENGTH_OUT_OF_RANGE);
    }
    if (total_page > p.num_free) raise_flag(p.status, LMCB_DEVICE_FLAG_PAGES_EXHAUSTED);
  }

  const int64_t stride = static_cast<int64_t>(gridDim.x) * threads;
  const int64_t me = static_cast<int64_t>(blockIdx.x) * threads + tid;

  // The page of block `blk` of request r, from the table where the request had
  // it and else from the free list.
  const uint32_t size = p.div_block.d;
  const auto page_of = [&](int r, uint32_t ctx, uint32_t blk) {
    if (blk * size < ctx) return p.table[r * p.table_stride + blk];
    const uint32_t f = s_first[r] + (blk - pages_of(ctx, p));
    return f < static_cast<uint32_t>(p.num_free) ? p.free_blocks[f] : -1;
  };
  const auto slot_at = [&](int32_t page, uint32_t off) {
    const int64_t at = static_cast<int64_t>(page) * size + off;
    if (page < 0) return static_cast<SlotT>(-1);
    if (sizeof(SlotT) == 4 && at > INT_MAX) {
      raise_flag(p.status, LMCB_DEVICE_FLAG_SLOT_OUT_OF_RANGE);
      return static_cast<SlotT>(-1);
    }
    return static_cast<SlotT>(at);
  };
  // The token at a new page's start enters the page in the table.
  const auto enter = [&](int r, uint32_t ctx, uint32_t blk, uint32_t off, int32_t page) {
    if (off == 0 && blk * size >= ctx) p.table[r * p.table_stride + blk] = page;
  };

  // kTokensPerThread consecutive tokens a thread.
  SlotT* slots = static_cast<SlotT*>(p.slots);
  SlotT* positions = static_cast<SlotT*>(p.positions);
  for (int64_t t0 = me * kTokensPerThread; t0 < p.num_tokens; t0 += stride * kTokensPerThread) {
    const int32_t t = static_cast<int32_t>(t0);
    int r = 0;
    int32_t r_end = 0;
    uint32_t ctx = 0, pos = 0;
    if (t < total_tok) {
      r = last_le(s_start, B, t);
      r_end = r + 1 < B ? s_start[r + 1] : total_tok;
      ctx = s_ctx[r];
      pos = ctx + static_cast<uint32_t>(t - s_start[r]);
    }
    if (p.aligned && size >= kTokensPerThread && t + kTokensPerThread <= r_end &&
        pos + kTokensPerThread <= static_cast<uint32_t>(p.row_tokens)) {
      // of one request and inside its row: one page, or the end of one and the
      // start of the next
      alignas(16) SlotT slot[kTokensPerThread], position[kTokensPerThread];
      const uint32_t blk = p.div_block.div(pos), off = pos - blk * size;
      const int32_t page = page_of(r, ctx, blk);
      enter(r, ctx, blk, off, page);
      const uint32_t in_page = size - off;
      int32_t after = -1;
      if (in_page < kTokensPerThread) {
        after = page_of(r, ctx, blk + 1);
        enter(r, ctx, blk + 1, 0, after);
      }
#pragma unroll
      for (uint32_t k = 0; k < kTokensPerThread; ++k) {
        slot[k] = k < in_page ? slot_at(page, off + k) : slot_at(after, k - in_page);
        position[k] = static_cast<SlotT>(pos + k);
      }
      constexpr int kVecs = sizeof(slot) / 16;
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        reinterpret_cast<uint4*>(slots + t0)[v] = reinterpret_cast<const uint4*>(slot)[v];
        reinterpret_cast<uint4*>(positions + t0)[v] = reinterpret_cast<const uint4*>(position)[v];
      }
      continue;
    }
#pragma unroll 1
    for (int32_t u = t; u < t + kTokensPerThread && u < p.num_tokens; ++u) {
      SlotT slot = -1, position = 0;
      if (u < total_tok) {
        if (u >= r_end) {
          r = last_le(s_start, B, u);
          r_end = r + 1 < B ? s_start[r + 1] : total_tok;
          ctx = s_ctx[r];
        }
        pos = ctx + static_cast<uint32_t>(u - s_start[r]);
        position = static_cast<SlotT>(pos);
        if (pos < static_cast<uint32_t>(p.row_tokens)) {
          const uint32_t blk = p.div_block.div(pos), off = pos - blk * size;
          const int32_t page = page_of(r, ctx, blk);
          enter(r, ctx, blk, off, page);
          slot = slot_at(page, off);
        } else {
          raise_flag(p.status, LMCB_DEVICE_FLAG_PAGES_EXHAUSTED);  // beyond the table's row
        }
      }
      slots[u] = slot;
      positions[u] = position;
    }
  }
}

}  // namespace
}  // namespace lmcb

extern "C" {

int lmcb_build_slot_mapping(const void* contextLens, const void* queryLens, int lenType,
                            int32_t numRequests, int32_t* blockTable, int64_t tableStride,
                            int32_t tableCols, const int32_t* freeBlocks, int64_t numFree,
                            int32_t blockSize, int64_t numTokens, void* slotMapping,
                            void* positions, int slotType, int32_t* queryStart, int32_t* seqLens,
                            int32_t* blocksUsed, void* stream) {
  lmcb::clear_error();
  const std::string who = "build_slot_mapping";
  if ((lenType != LMCB_DTYPE_INT64 && lenType != LMCB_DTYPE_INT32) ||
      (slotType != LMCB_DTYPE_INT64 && slotType != LMCB_DTYPE_INT32)) {
    return lmcb::fail(LMCB_ERR_UNSUPPORTED_DTYPE, who + ": lengths and slots must be int64 or int32.");
  }
  if (numRequests < 0 || tableCols < 0 || tableStride < tableCols || numFree < 0 ||
      numFree > INT_MAX || blockSize <= 0 || numTokens < 0 || numTokens > INT_MAX - 4 ||
      static_cast<int64_t>(tableCols) * blockSize > INT_MAX) {
    return lmcb::fail(LMCB_ERR_INVALID_ARGUMENT, who + ": invalid shape.");
  }
  if (numRequests > lmcb::kBatchMaxRequests) {
    return lmcb::fail(LMCB_ERR_CAPACITY, who + ": at most " +
                                             std::to_string(lmcb::kBatchMaxRequests) +
                                             " requests a call.");
  }
  if (queryStart == nullptr || blocksUsed == nullptr ||
      (numRequests > 0 && (contextLens == nullptr || queryLens == nullptr || seqLens == nullptr)) ||
      (numRequests > 0 && tableCols > 0 && blockTable == nullptr) ||
      (numFree > 0 && freeBlocks == nullptr) ||
      (numTokens > 0 && (slotMapping == nullptr || positions == nullptr))) {
    return lmcb::fail(LMCB_ERR_INVALID_ARGUMENT, who + ": NULL pointer.");
  }
  lmcb::BatchParams p;
  p.context_lens = contextLens;
  p.query_lens = queryLens;
  p.len64 = lenType == LMCB_DTYPE_INT64;
  p.num_requests = numRequests;
  p.table = blockTable;
  p.table_stride = tableStride;
  p.table_cols = tableCols;
  p.row_tokens = tableCols * blockSize;
  p.free_blocks = freeBlocks;
  p.num_free = static_cast<int32_t>(numFree);
  p.div_block = lmcb::FastDiv(static_cast<uint32_t>(blockSize));
  p.num_tokens = static_cast<int32_t>(numTokens);
  p.slots = slotMapping;
  p.positions = positions;
  p.aligned = reinterpret_cast<uintptr_t>(slotMapping) % 16 == 0 &&
              reinterpret_cast<uintptr_t>(positions) % 16 == 0;
  p.query_start = queryStart;
  p.seq_lens = seqLens;
  p.blocks_used = blocksUsed;
  p.status = lmcb::device_status_ptr();
  if (p.status == nullptr) return LMCB_ERR_CUDA;
  const int64_t groups =
      (numTokens + lmcb::kTokensPerThread - 1) / lmcb::kTokensPerThread;
  const int threads = groups <= 256 && numRequests <= 256 ? 256 : lmcb::kBatchThreads;
  const int64_t want = (groups + threads - 1) / threads;
  const int64_t most = lmcb::current_sm_count() * 2;
  const unsigned grid = static_cast<unsigned>(want < 1 ? 1 : want < most ? want : most);
  const size_t smem = static_cast<size_t>(numRequests) * 12;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  constexpr size_t kCap = size_t(lmcb::kBatchMaxRequests) * 12;
  if (slotType == LMCB_DTYPE_INT64) {
    LMCB_CUDA_TRY((lmcb::ensure_smem_limit<lmcb::build_slot_mapping_kernel<int64_t>>(smem, kCap)));
    lmcb::build_slot_mapping_kernel<int64_t><<<grid, threads, smem, s>>>(p);
  } else {
    LMCB_CUDA_TRY((lmcb::ensure_smem_limit<lmcb::build_slot_mapping_kernel<int32_t>>(smem, kCap)));
    lmcb::build_slot_mapping_kernel<int32_t><<<grid, threads, smem, s>>>(p);
  }
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return lmcb::cuda_fail(err, who.c_str());
  return LMCB_OK;
}

}  // extern "C"
