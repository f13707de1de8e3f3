// What the call's plan and the attention kernels both know of the kernels' tiles.
#pragma once

#include <stdint.h>

namespace voom {
namespace kv {

// Which kernel a call takes: attn_tc's modes (kv_tc.cuh), attn_rows, attn_few.
constexpr int kPair = 0, kAlternate = 1, kSingle = 2, kRows = -1, kFew = -2;
constexpr uint32_t kFewRows = 8;  // rows that attn_few takes

// attn_rows: warps of a block, and bytes of a tile, half of them keys.  Scored
// calls do more for a score, and a warp's tile is bound by its instructions'
// latency: two warps to a scheduler with tiles half as large (heads of 256 would
// be left with 8 keys, too few for a matrix instruction).
__host__ __device__ constexpr bool row_wide(uint32_t dp, bool scored) { return scored && dp <= 128; }
__host__ __device__ constexpr uint32_t row_warps(uint32_t dp, bool scored) { return row_wide(dp, scored) ? 8 : 4; }
__host__ __device__ constexpr uint32_t row_tile(uint32_t dp, bool scored) { return row_wide(dp, scored) ? 8192 : 16384; }
__host__ __device__ constexpr uint32_t row_keys(uint32_t dp, bool scored) { return row_tile(dp, scored) / (4 * dp); }

}  // namespace kv
}  // namespace voom
