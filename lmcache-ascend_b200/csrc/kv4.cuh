// kv4.cuh -- the paged KV cache held in 4 bits: layout shared by the store,
// the load and the attention that reads it.
//
// A layer's cache is int32 [2, num_blocks, block_size, W]: K rows, then V
// rows, one row of W words a slot. A row of H heads of D values holds
//   words [0, H * D / 8)            codes; word h * D / 8 + w carries values
//                                   8 w ... 8 w + 7 of head h, value 8 w + j in
//                                   bits [4 j, 4 j + 4)
//   words [H * D / 8, + H)          one word a head: fp16 scale s in the low
//                                   half, fp16 zero z in the high half
// and is padded to W, a multiple of four words (16 bytes), with words that are
// neither written nor read. A code c stands for z + s c. Scale and zero sit in
// the token's own row, so a row is a row of int32 like any other to the paged
// transfers: a 4-bit cache is stored to and retrieved from LMCache objects by
// the same launches, with W words for its hidden size.
#pragma once

#include <stdint.h>

namespace lmcb {

inline int64_t kv4_row_words(int64_t heads, int64_t head_size) {
  return (heads * (head_size / 8 + 1) + 3) / 4 * 4;
}

}  // namespace lmcb
