// kv4_plan.h -- the kernel for many query rows a KV head, as the entry point
// calls it.
#pragma once

#include "kv4_attention.cuh"

namespace lmcb {
namespace kv4 {

// Bytes of workspace launch_rows needs for these sizes.
size_t rows_workspace(int64_t batch, int64_t max_query, int64_t max_len, int64_t kv_heads,
                      int64_t group, int64_t head_size, int64_t window, int64_t sinks);

cudaError_t launch_rows(const AttnParams& a, int type, int64_t head_size, int64_t max_len,
                        void* workspace, cudaStream_t stream);

}  // namespace kv4
}  // namespace lmcb
