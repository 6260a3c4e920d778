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
// writing. What is left is one search over the prefix sums for each group of
// consecutive tokens and the writes of slots and positions, so a large batch
// is bound by those writes and a small one by one launch and three dependent
// loads (lengths, prefix sums, page).
#include <cuda_runtime.h>
#include <stdint.h>

#include <climits>
#include <string>

#include "common.cuh"
#include "lmcache_b200.h"

namespace lmcb {
namespace {

constexpr int kBatchThreads = 512;
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
  const int32_t* free_blocks;
  int32_t num_free;
  FastDiv div_block;
  int32_t num_tokens;
  void* slots;
  void* positions;
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

// Pages that `tokens` tokens fill, at most the table's width.
__device__ __forceinline__ int32_t pages_of(int64_t tokens, const FastDiv& d, int32_t cols) {
  // tokens < 2^32: the quotient of tokens - 1 in two steps would lose nothing,
  // but a clamp to the largest table first keeps the numerator below 2^31.
  const int64_t cap = static_cast<int64_t>(cols) * d.d;
  if (tokens >= cap) return cols;
  return tokens == 0 ? 0 : static_cast<int32_t>(d.div(static_cast<uint32_t>(tokens - 1))) + 1;
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

template <typename SlotT>
__global__ void __launch_bounds__(kBatchThreads) build_slot_mapping_kernel(const BatchParams p) {
  extern __shared__ int32_t batch_smem[];
  const int B = p.num_requests;
  int32_t* s_start = batch_smem;      // [B] first token of the request
  int32_t* s_first = s_start + B;     // [B] first free-list entry of the request
  int32_t* s_ctx = s_first + B;       // [B] tokens in the cache
  __shared__ int64_t s_warp[2][kBatchThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  // Prefix sums, kBatchThreads requests at a time, in 64 bits.
  int64_t base_tok = 0, base_page = 0;
  for (int b0 = 0; b0 < B; b0 += kBatchThreads) {
    const int b = b0 + tid;
    int32_t ctx = 0, fresh = 0, need = 0;
    if (b < B) {
      ctx = load_len(p.context_lens, p.len64, b, p.status);
      fresh = load_len(p.query_lens, p.len64, b, p.status);
      need = pages_of(static_cast<int64_t>(ctx) + fresh, p.div_block, p.table_cols) -
             pages_of(ctx, p.div_block, p.table_cols);
    }
    int64_t tok = fresh, page = need;  // inclusive sums of the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t a = __shfl_up_sync(0xffffffffu, tok, o);
      const int64_t c = __shfl_up_sync(0xffffffffu, page, o);
      if (lane >= o) {
        tok += a;
        page += c;
      }
    }
    if (lane == 31) {
      s_warp[0][warp] = tok;
      s_warp[1][warp] = page;
    }
    __syncthreads();
    int64_t before_tok = base_tok, before_page = base_page;
    for (int w = 0; w < kBatchThreads / 32; ++w) {
      if (w < warp) {
        before_tok += s_warp[0][w];
        before_page += s_warp[1][w];
      }
      base_tok += s_warp[0][w];
      base_page += s_warp[1][w];
    }
    if (b < B) {
      s_ctx[b] = ctx;
      const int64_t st = before_tok + tok - fresh;
      s_start[b] = static_cast<int32_t>(st < p.num_tokens ? st : p.num_tokens);
      s_first[b] = clamp31(before_page + page - need);
      if (blockIdx.x == 0) {
        p.query_start[b] = s_start[b];
        p.seq_lens[b] = clamp31(static_cast<int64_t>(ctx) + fresh);
      }
    }
    __syncthreads();  // s_warp is rewritten by the next round
  }
  const int32_t total_tok =
      static_cast<int32_t>(base_tok < p.num_tokens ? base_tok : p.num_tokens);
  const int32_t total_page = clamp31(base_page);
  if (blockIdx.x == 0 && tid == 0) {
    p.query_start[B] = total_tok;
    p.blocks_used[0] = total_page;
    if (base_tok > p.num_tokens) raise_flag(p.status, LMCB_DEVICE_FLAG_LENGTH_OUT_OF_RANGE);
    if (total_page > p.num_free) raise_flag(p.status, LMCB_DEVICE_FLAG_PAGES_EXHAUSTED);
  }

  const int64_t stride = static_cast<int64_t>(gridDim.x) * kBatchThreads;
  const int64_t me = static_cast<int64_t>(blockIdx.x) * kBatchThreads + tid;

  // New table entries, one a thread.
  for (int64_t e = me; e < total_page; e += stride) {
    const int r = last_le(s_first, B, static_cast<int32_t>(e));
    const int32_t col = pages_of(s_ctx[r], p.div_block, p.table_cols) +
                        static_cast<int32_t>(e - s_first[r]);
    // Inside the row by construction; the test also covers sums beyond 2^31.
    if (col < p.table_cols) {
      p.table[r * p.table_stride + col] = e < p.num_free ? p.free_blocks[e] : -1;
    }
  }

  // Slots and positions, kTokensPerThread consecutive tokens a thread.
  SlotT* slots = static_cast<SlotT*>(p.slots);
  SlotT* positions = static_cast<SlotT*>(p.positions);
  for (int64_t t0 = me * kTokensPerThread; t0 < p.num_tokens; t0 += stride * kTokensPerThread) {
    int r = 0;
    int32_t r_end = 0;  // first token behind request r
    int32_t cached_blk = -1, cached_page = -1;
#pragma unroll
    for (int k = 0; k < kTokensPerThread; ++k) {
      const int32_t t = static_cast<int32_t>(t0) + k;
      if (t0 + k >= p.num_tokens) break;
      if (t >= total_tok) {
        slots[t] = -1;
        positions[t] = 0;
        continue;
      }
      if (k == 0 || t >= r_end) {
        r = last_le(s_start, B, t);
        r_end = r + 1 < B ? s_start[r + 1] : total_tok;
        cached_blk = -1;
      }
      const int64_t pos = static_cast<int64_t>(s_ctx[r]) + (t - s_start[r]);
      int64_t slot = -1;
      if (pos < static_cast<int64_t>(p.table_cols) * p.div_block.d) {
        const int32_t blk = static_cast<int32_t>(p.div_block.div(static_cast<uint32_t>(pos)));
        if (blk != cached_blk) {
          cached_blk = blk;
          const int32_t has = pages_of(s_ctx[r], p.div_block, p.table_cols);
          if (blk < has) {
            cached_page = p.table[r * p.table_stride + blk];
          } else {
            const int64_t f = static_cast<int64_t>(s_first[r]) + (blk - has);
            cached_page = f < p.num_free ? p.free_blocks[f] : -1;
          }
        }
        if (cached_page >= 0) {
          slot = static_cast<int64_t>(cached_page) * p.div_block.d +
                 (pos - static_cast<int64_t>(blk) * p.div_block.d);
          if (sizeof(SlotT) == 4 && slot > INT_MAX) {
            raise_flag(p.status, LMCB_DEVICE_FLAG_SLOT_OUT_OF_RANGE);
            slot = -1;
          }
        }
      } else {
        raise_flag(p.status, LMCB_DEVICE_FLAG_PAGES_EXHAUSTED);  // beyond the table's row
      }
      slots[t] = static_cast<SlotT>(slot);
      positions[t] = static_cast<SlotT>(pos);
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
  p.free_blocks = freeBlocks;
  p.num_free = static_cast<int32_t>(numFree);
  p.div_block = lmcb::FastDiv(static_cast<uint32_t>(blockSize));
  p.num_tokens = static_cast<int32_t>(numTokens);
  p.slots = slotMapping;
  p.positions = positions;
  p.query_start = queryStart;
  p.seq_lens = seqLens;
  p.blocks_used = blocksUsed;
  p.status = lmcb::device_status_ptr();
  if (p.status == nullptr) return LMCB_ERR_CUDA;
  const int64_t per_cta = int64_t(lmcb::kBatchThreads) * lmcb::kTokensPerThread;
  const int64_t want = (numTokens + per_cta - 1) / per_cta;
  const int64_t most = static_cast<int64_t>(lmcb::current_sm_count()) * 2;
  const unsigned grid = static_cast<unsigned>(want < 1 ? 1 : want < most ? want : most);
  const size_t smem = static_cast<size_t>(numRequests) * 12;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  constexpr size_t kCap = size_t(lmcb::kBatchMaxRequests) * 12;
  if (slotType == LMCB_DTYPE_INT64) {
    LMCB_CUDA_TRY((lmcb::ensure_smem_limit<lmcb::build_slot_mapping_kernel<int64_t>>(smem, kCap)));
    lmcb::build_slot_mapping_kernel<int64_t><<<grid, lmcb::kBatchThreads, smem, s>>>(p);
  } else {
    LMCB_CUDA_TRY((lmcb::ensure_smem_limit<lmcb::build_slot_mapping_kernel<int32_t>>(smem, kCap)));
    lmcb::build_slot_mapping_kernel<int32_t><<<grid, lmcb::kBatchThreads, smem, s>>>(p);
  }
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return lmcb::cuda_fail(err, who.c_str());
  return LMCB_OK;
}

}  // extern "C"
