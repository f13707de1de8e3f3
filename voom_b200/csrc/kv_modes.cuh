// What the call's plan and the attention kernels both know of the kernels' tiles.
#pragma once

#include <stdint.h>

namespace voom {
namespace kv {

// attn_tc's modes (kv_tc.cuh).
constexpr int kPair = 0, kAlternate = 1, kSingle = 2;

// attn_rows: keys of a tile, 8 KB of keys and 8 KB of values.
__host__ __device__ constexpr uint32_t row_keys(uint32_t dp) { return 4096u / dp; }

}  // namespace kv
}  // namespace voom
