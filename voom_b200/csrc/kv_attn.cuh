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
  int32_t tc;                // tensor-core kernel's mode, or -1: attn_rows
};

struct Seg {
  uint32_t b, h, m, s0, s1, steps, len;  // unit (request, key head, block of rows), steps [s0, s1) of `steps`
  uint64_t at, end;                      // this block's place in the list of steps, and its end
};

__host__ __device__ __forceinline__ uint32_t ceil_div(uint32_t a, uint32_t b) { return (a + b - 1) / b; }

__device__ __forceinline__ uint32_t cache_steps(const Attn& P, uint32_t len) { return ceil_div(len, P.keys); }

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
__device__ __forceinline__ uint64_t head_steps(const Attn& P, uint32_t len) {
  return uint64_t(P.mblocks) * cache_steps(P, len) + P.tails;
}

// Steps of all units before request b (warp-collective); b = B: of all.
__device__ __forceinline__ uint64_t steps_before(const Attn& P, uint32_t b) {
  uint64_t sum = 0;
  for (uint32_t i = threadIdx.x & 31u; i < b; i += 32) sum += head_steps(P, P.c.length(i));
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
__device__ __forceinline__ bool first_seg(const Attn& P, uint32_t cta, Seg& s) {
  if (!P.ctas) {  // the units of a request with the most steps first
    const uint32_t hk = P.c.v.hk, U = hk * P.mblocks, r = cta % U;
    s.b = cta / U;
    s.h = r % hk;
    s.m = P.mblocks - 1 - r / hk;
    s.len = P.c.length(s.b);
    s.steps = s.s1 = cache_steps(P, s.len) + tail_of(P, s.m);
    s.s0 = 0;
    s.at = 0;
    s.end = s.steps;
    return true;
  }
  const uint64_t total = steps_before(P, P.c.v.B);
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
    const uint64_t mine = b < P.c.v.B ? head_steps(P, P.c.length(b)) * P.c.v.hk : 0;
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
  const uint32_t cs = cache_steps(P, s.len);
  const uint64_t per = head_steps(P, s.len);
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
  s.steps = cache_steps(P, s.len) + tail_of(P, s.m);
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

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// sum += x with what the addition lost kept in `rest`: beside one large term, a
// long cache's small ones would be lost one by one (2^-25 of a row's largest
// does not change a 1 at all).  Both are at least 0.
__device__ __forceinline__ void add_kept(float& sum, float& rest, float x) {
  const float t = sum + x;
  rest += fminf(sum, x) - (t - fmaxf(sum, x));
  sum = t;
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

}  // namespace kv
}  // namespace voom
