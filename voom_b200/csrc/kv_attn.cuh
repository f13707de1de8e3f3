// Shared pieces of the cache attention kernels: the call, how its work is cut
// into steps and spread over the blocks, and the partial results.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "kv_view.cuh"

namespace voom {
namespace kv {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Rows: the n new tokens of a request times the g query heads that share a key
// head, row r = token r / g, head h * g + r % g.  A unit is a block of `rows`
// rows of one key head of one request; its steps are the tiles of `keys`
// cached positions, then those of the new tokens.  The blocks of the grid
// either take one unit each (direct), or equal shares of all units' steps in
// order, so that a long request is spread over many blocks and short ones
// share a block; a block then leaves at most two units unfinished, its first
// and its last, as partial sums in its two slots.
struct alignas(64) Attn {
  CUtensorMap k_map, v_map;  // the cache (head values, positions, heads, pages or requests), boxes of 64 values x `box` positions
  uint32_t box;              // 0: the cache cannot be read with TMA
  View c;
  voom_tree_attention_args a;
  float* lse;       // B x n x hq: the caller's, or scratch, or NULL
  float* scores;    // scratch, or NULL: unit rows x score_ld, log2 units
  float* partial;   // scratch: 2 slots per block, each rows x ld_o sums, rows x (maximum, sum)
  uint32_t g, R, words;      // query heads per key head, rows, mask words of a row
  uint32_t keys, rows, ld_o; // tile sizes
  uint32_t mblocks, tails;   // blocks of rows of a key head; their steps over the new tokens
  uint32_t ctas;             // 0: direct
  uint32_t score_ld, score_new; // score row length; where the new tokens' scores start
  float scale2;              // scale * log2(e)
  float cap_in, cap_out;     // of capped scores: 2 scale log2(e) / cap, and cap log2(e); 0: not capped
  float cap_small;           // products up to it take the polynomial: its coefficients, twice each
  float2 poly[5];
  int32_t tc;                // which kernel (kv_modes.cuh): at least 0 for attn_tc
};

struct Seg {
  uint32_t b, h, m, s0, s1, steps, len;  // unit (request, key head, block of rows), steps [s0, s1) of `steps`
  uint64_t at, end;                      // this block's place in the list of steps, and its end
};

__host__ __device__ __forceinline__ uint32_t ceil_div(uint32_t a, uint32_t b) { return (a + b - 1) / b; }

// The first tile of cached positions that any of a request's rows sees: a window
// ends `window` positions before the row, and no row stands before position len.
// (SCORED false: the call is known to have no window; nothing is asked)
template <bool SCORED = true>
__device__ __forceinline__ uint32_t first_tile(const Attn& P, uint32_t len) {
  return SCORED && P.a.window && len >= P.a.window ? (len - P.a.window + 1) / P.keys : 0u;
}

// A window's edge moves with the rows: no row sees a cached position below
// `none`, all see those from `all` on (the last of n rows stands at len + n - 1 at
// most).  Values between must not reach the rows that do not see them, not even
// times 0: tiles below `all` are looked through for values that are not finite.
template <bool SCORED = true>
__device__ __forceinline__ uint32_t window_none(const Attn& P, uint32_t len) {
  return SCORED && P.a.window && len >= P.a.window ? len - P.a.window + 1 : 0u;
}
__device__ __forceinline__ uint32_t window_all(const Attn& P, uint32_t len) {
  return P.a.window && len + P.a.n > P.a.window ? len + P.a.n - P.a.window : 0u;
}

template <bool SCORED = true>
__device__ __forceinline__ uint32_t cache_steps(const Attn& P, uint32_t len) { return ceil_div(len, P.keys) - first_tile<SCORED>(P, len); }

// Steps over the new tokens of the m-th block of rows: in a chain, up to its last token.
__host__ __device__ __forceinline__ uint32_t tail_of(const Attn& P, uint32_t m) {
  if (P.a.d_mask) return ceil_div(P.a.n, P.keys);
  const uint32_t rows = (m + 1) * P.rows;
  return ceil_div(((rows < P.R ? rows : P.R) - 1) / P.g + 1, P.keys);
}

// Those of the first m blocks (m < mblocks, or all but the last of them).  In a
// chain block i takes floor(((i + 1) rows - 1) / (g keys)) + 1 steps: a sum of
// floors of an arithmetic progression, by the reciprocity that swaps slope and
// modulus as Euclid's algorithm does.
__host__ __device__ __forceinline__ uint64_t tails_before(const Attn& P, uint32_t m) {
  if (P.a.d_mask) return uint64_t(m) * ceil_div(P.a.n, P.keys);
  uint64_t sum = m, n = m, a = P.rows, b = P.rows - 1, q = uint64_t(P.g) * P.keys;
  if (!m) return 0;
  for (;;) {  // sum of floor((a i + b) / q) over i < n
    sum += n * (n - 1) / 2 * (a / q) + n * (b / q);
    a %= q;
    b %= q;
    const uint64_t top = a * n + b;
    if (top < q) return sum;
    n = top / q;
    b = top % q;
    const uint64_t t = q;
    q = a;
    a = t;
  }
}

// Steps of one key head of a request.
template <bool SCORED = true>
__device__ __forceinline__ uint64_t head_steps(const Attn& P, uint32_t len) {
  return uint64_t(P.mblocks) * cache_steps<SCORED>(P, len) + P.tails;
}

// Steps of all units before request b (warp-collective); b = B: of all.
template <bool SCORED = true>
__device__ __forceinline__ uint64_t steps_before(const Attn& P, uint32_t b) {
  uint64_t sum = 0;
  for (uint32_t i = threadIdx.x & 31u; i < b; i += 32) sum += head_steps<SCORED>(P, P.c.length(i));
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  return sum * P.c.v.hk;
}

// Blocks that share `total` steps.  The grid is laid out for max_len; where the
// lengths on the device leave fewer steps than blocks, the blocks past the last
// step take none, so that every block between a unit's first and last has left
// a partial sum.
__device__ __forceinline__ uint32_t sharers(const Attn& P, uint64_t total) {
  return total < P.ctas ? uint32_t(total) : P.ctas;
}

// First segment of grid block `cta` (warp-collective); false: it has none.
template <bool SCORED>
__device__ __forceinline__ bool first_seg(const Attn& P, uint32_t cta, Seg& s) {
  if (!P.ctas) {  // the units of a request with the most steps first
    const uint32_t hk = P.c.v.hk, U = hk * P.mblocks, r = cta % U;
    s.b = cta / U;
    s.h = r % hk;
    s.m = P.mblocks - 1 - r / hk;
    s.len = P.c.length(s.b);
    s.steps = s.s1 = cache_steps<SCORED>(P, s.len) + tail_of(P, s.m);
    s.s0 = 0;
    s.at = 0;
    s.end = s.steps;
    return true;
  }
  const uint64_t total = steps_before<SCORED>(P, P.c.v.B);
  const uint32_t ctas = sharers(P, total);
  if (cta >= ctas) return false;
  const uint64_t top = total * (cta + 1);
  s.at = top >> 32 ? (top - total) / ctas : uint32_t(top - total) / ctas;
  s.end = top >> 32 ? top / ctas : uint32_t(top) / ctas;
  uint64_t base = 0;
  const uint32_t lane = threadIdx.x & 31u;
  for (uint32_t b0 = 0;; b0 += 32) {
    if (b0 >= P.c.v.B) return false;  // not reached: at < total
    const uint32_t b = b0 + lane;
    const uint64_t mine = b < P.c.v.B ? head_steps<SCORED>(P, P.c.length(b)) * P.c.v.hk : 0;
    uint64_t upto = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
      if (int(lane) >= o) upto += x;
    }
    const uint32_t hit = __ballot_sync(0xFFFFFFFFu, base + upto > s.at);
    if (hit) {
      const int k = __ffs(hit) - 1;
      s.b = b0 + uint32_t(k);
      base += __shfl_sync(0xFFFFFFFFu, upto - mine, k);
      break;
    }
    base += __shfl_sync(0xFFFFFFFFu, upto, 31);
  }
  s.len = P.c.length(s.b);
  const uint32_t cs = cache_steps<SCORED>(P, s.len);
  const uint64_t per = head_steps<SCORED>(P, s.len);
  uint64_t off = s.at - base;
  s.h = uint32_t(off / per);
  off -= s.h * per;
  uint32_t lo = 0, hi = P.mblocks - 1;  // the last block of rows that starts at off or before
  while (lo < hi) {
    const uint32_t mid = (lo + hi + 1) / 2;
    if (uint64_t(mid) * cs + tails_before(P, mid) <= off) lo = mid;
    else hi = mid - 1;
  }
  s.m = lo;
  off -= uint64_t(lo) * cs + tails_before(P, lo);
  s.steps = cs + tail_of(P, lo);
  s.s0 = uint32_t(off);
  s.s1 = uint32_t(min(uint64_t(s.steps), off + (s.end - s.at)));
  return true;
}

template <bool SCORED>
__device__ __forceinline__ bool next_seg(const Attn& P, Seg& s) {
  s.at += s.s1 - s.s0;
  if (s.at >= s.end) return false;
  if (++s.m == P.mblocks) {
    s.m = 0;
    if (++s.h == P.c.v.hk) {
      s.h = 0;
      s.len = P.c.length(++s.b);
    }
  }
  s.steps = cache_steps<SCORED>(P, s.len) + tail_of(P, s.m);
  s.s0 = 0;
  s.s1 = uint32_t(min(uint64_t(s.steps), s.end - s.at));
  return true;
}

// The blocks that hold partial sums of a unit whose steps are [at, at + steps)
// of the list: first .. last, and first's slot is its second one.
__device__ __forceinline__ void owners(const Attn& P, uint64_t total, uint64_t at, uint32_t steps, uint32_t& first,
                                       uint32_t& last) {
  // block c covers [total * c / ctas, total * (c + 1) / ctas), one step at least:
  // x is in the largest c with total * c / ctas <= x, that is total * c < ctas * (x + 1)
  const uint32_t ctas = sharers(P, total);
  auto holder = [&](uint64_t x) {
    const uint64_t top = uint64_t(ctas) * (x + 1) - 1;
    return top >> 32 ? uint32_t(top / total) : uint32_t(top) / uint32_t(total);
  };
  first = holder(at);
  last = holder(at + steps - 1);
}

__device__ __forceinline__ float* slot_of(const Attn& P, uint32_t slot) {
  return P.partial + uint64_t(slot) * P.rows * (P.ld_o + 2);
}

__device__ __forceinline__ bool sees(const Attn& P, uint32_t b, uint32_t i, uint32_t j) {
  if (!P.a.d_mask) return j <= i;
  return P.a.d_mask[(uint64_t(b) * P.a.n + i) * P.words + (j >> 5)] >> (j & 31u) & 1u;
}

// Bits [j0, j0 + 32) of row i's mask.
__device__ __forceinline__ uint32_t sees32(const Attn& P, uint32_t b, uint32_t i, uint32_t j0) {
  if (i >= P.a.n || j0 >= P.a.n) return 0u;
  if (P.a.d_mask) {
    const uint32_t* m = P.a.d_mask + (uint64_t(b) * P.a.n + i) * P.words;
    const uint32_t w = j0 >> 5, r = j0 & 31u, lo = __ldg(m + w);
    if (!r) return lo;
    return __funnelshift_r(lo, w + 1 < P.words ? __ldg(m + w + 1) : 0u, r);
  }
  return i < j0 ? 0u : i - j0 >= 31u ? 0xFFFFFFFFu : (2u << (i - j0)) - 1u;
}

// How far behind the cache new token i stands: its depth in the tree.
__device__ __forceinline__ int32_t depth_of(const Attn& P, uint32_t b, uint32_t i) {
  return P.a.d_mask && P.a.d_depth && i < P.a.n ? __ldg(P.a.d_depth + uint64_t(b) * P.a.n + i) : int32_t(i);
}

// Of 32 keys from distance `ahead` of a row on (key position - row position, one
// more for each), those inside the window, at distances above -window.
__device__ __forceinline__ uint32_t window32(const Attn& P, int32_t ahead) {
  if (!P.a.window) return 0xFFFFFFFFu;
  const int64_t out = -int64_t(P.a.window) - ahead + 1;  // keys before the window
  return out <= 0 ? 0xFFFFFFFFu : out >= 32 ? 0u : 0xFFFFFFFFu << out;
}

__device__ __forceinline__ bool in_window(const Attn& P, int32_t ahead) {
  return !P.a.window || -int64_t(ahead) < int64_t(P.a.window);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 values in a register pair: one instruction works on both.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 make2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void take2(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
// Products q . k as scores in log2 units, for calls whose scores are capped,
// biased or windowed ("scored"): two at a time, whose biases are `bias`.
//   kPlain    not capped
//   kSmall    capped, with |z| <= 3/4 cap: cap tanh(z / cap) = z P((z / cap)^2), off by
//             8e-7 of itself at most, no more than the product's own sum.  Six
//             instructions for two scores, none of them on the special-function unit,
//             which the softmax needs for its own exponentials (1000 tokens x 32 heads
//             over 8192 positions, cap 50, window 6000: 224 us; with another term, for
//             1.3e-7, 237)
//   kAny      capped: the same, and past 3/4 cap  cap - 2 cap / (1 + e^(2 z / cap)), off by
//             a few 2^-23 of the cap and no further at either end
constexpr int kPlain = 0, kSmall = 1, kAny = 2;
// P, nearest to tanh(w) / w on [0, 3/4] with P(0) = 1: largest difference 6.0e-7, by
// reweighted least squares.
constexpr double kTanh[5] = {1.0, -0.3332984149456024, 0.132701113820076, -0.05033518746495247, 0.013158644549548626};
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
template <int KIND>
__device__ __forceinline__ F2 scored2(const Attn& P, F2 x, F2 bias) {
  auto both = [](float c) { return make2(c, c); };
  if (KIND == kPlain) return fma2(x, both(P.scale2), bias);
  auto c = [&](int i) { return make2(P.poly[i].x, P.poly[i].y); };
  const F2 s = mul2(x, x);
  const F2 small = fma2(x, fma2(s, fma2(s, fma2(s, fma2(s, c(4), c(3)), c(2)), c(1)), c(0)), bias);
  if (KIND == kSmall) return small;
  float a, b, x0, x1, y0, y1, z0, z1;
  take2(mul2(x, both(P.cap_in)), a, b);
  take2(add2(make2(exp2_fast(a), exp2_fast(b)), both(1.0f)), a, b);
  take2(fma2(make2(rcp_fast(a), rcp_fast(b)), both(-2.0f * P.cap_out), add2(bias, both(P.cap_out))), y0, y1);
  take2(x, x0, x1);
  take2(small, z0, z1);
  return make2(fabsf(x0) <= P.cap_small ? z0 : y0, fabsf(x1) <= P.cap_small ? z1 : y1);
}
__device__ __forceinline__ F2 scored2(const Attn& P, F2 x, F2 bias) {
  return P.cap_in != 0.0f ? scored2<kAny>(P, x, bias) : scored2<kPlain>(P, x, bias);
}
__device__ __forceinline__ float scored(const Attn& P, float x, float slope2, float ahead) {
  float y, unused;
  take2(scored2(P, make2(x, x), make2(slope2 * ahead, 0.0f)), y, unused);
  return y;
}
template <int KIND>
using Kind = std::integral_constant<int, KIND>;

// A query head's slope in log2 units.
__device__ __forceinline__ float slope2_of(const Attn& P, uint32_t head) {
  return P.a.d_slopes ? kLog2e * __ldg(P.a.d_slopes + head) : 0.0f;
}

// sum += x with what the addition lost kept in `rest`: beside one large term, a
// long cache's small ones would be lost one by one (2^-25 of a row's largest
// does not change a 1 at all).  Both are at least 0.
__device__ __forceinline__ void add_kept(float& sum, float& rest, float x) {
  const float t = sum + x;
  rest += fminf(sum, x) - (t - fmaxf(sum, x));
  sum = t;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Probabilities are rounded to the cache's type for the value product (the tensor
// cores want both operands in one), half a unit each of a sum that is rounded
// to that type anyway; the denominator adds them up unrounded.  What is rounded
// is 2^kLift p.  FP16 ends at 2^-24: beside a position that takes nearly all of a
// row's weight, a long cache's many small ones would vanish, or lose up to half,
// one by one.  Lifted, with p at most 2^SLACK, they are at most 2^14 and keep 11
// bits down to 2^-14 / 2^kLift.  BF16 has fp32's range.
template <typename T, int SLACK>
constexpr float kLift = std::is_same<T, __half>::value ? 14.0f - SLACK : 0.0f;

__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

// Byte offset of 16-byte chunk c of row r in a tile of `rows` rows: blocks of
// 64 values (128 bytes a row) one after another, the chunk turned by the row.
__device__ __forceinline__ uint32_t sw128(uint32_t r, uint32_t c, uint32_t rows) {
  return (c >> 3) * (rows * 128u) + r * 128u + (((c ^ r) & 7u) << 4);
}

// 16 bytes to shared memory without a register, or 16 zero bytes.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16u : 0u) : "memory");
}

// Any of the eight 16-bit values of a chunk infinite or NaN (exponent all ones).
template <typename T>
__device__ __forceinline__ bool odd_values(uint4 c) {
  const uint32_t m = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0x7C007C00u : 0x7F807F80u;
  bool bad = false;
  for (uint32_t w : {c.x, c.y, c.z, c.w}) {
    const uint32_t e = w & m;
    bad |= (e & 0xFFFFu) == (m & 0xFFFFu) || (e >> 16) == (m >> 16);
  }
  return bad;
}

// The attention's kernel, and the rows' weights from the keys again, for caches
// of type T; SCORED: scores are capped, biased or windowed (kv_launch.cuh).
template <typename T, bool SCORED>
int launch_attention(const Attn& P, cudaStream_t s);
template <typename T, bool SCORED>
int launch_sums(const Attn& P, cudaStream_t s);

}  // namespace kv
}  // namespace voom
