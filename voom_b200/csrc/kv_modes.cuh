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
// latency: two warps to a scheduler with tiles half as large (16 rows over 32
// requests of up to 16000 positions, heads of 128: 261 us against 284, of 64: 157
// against 200; heads of 256 would be left with 8 keys, too few for a matrix instruction).
__host__ __device__ constexpr bool row_wide(uint32_t dp, bool scored) { return scored && dp <= 128; }
__host__ __device__ constexpr uint32_t row_warps(uint32_t dp, bool scored) { return row_wide(dp, scored) ? 8 : 4; }
__host__ __device__ constexpr uint32_t row_tile(uint32_t dp, bool scored) { return row_wide(dp, scored) ? 8192 : 16384; }
__host__ __device__ constexpr uint32_t row_keys(uint32_t dp, bool scored) { return row_tile(dp, scored) / (4 * dp); }

// Rows that attn_rows takes; attn_tc takes more.  Scored, 25 to 32 rows of heads of 128
// are attn_tc's too: 32 rows over 32 requests of up to 16000 positions 354 us against
// 407, 16 of up to 1000 47 against 70, but one of 131072 208 against 198; 24 rows there
// 204 against 184.  Heads of 64 stay at 32 rows: 236 us over the 32 requests against 348.
__host__ __device__ constexpr uint32_t row_most(uint32_t dp, bool scored) { return dp == 256 ? 16 : scored && dp == 128 ? 24 : 32; }

}  // namespace kv
}  // namespace voom
