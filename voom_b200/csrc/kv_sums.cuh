// The weight that each position received from many rows: tcgen05.
//
//   sums[s] += sum over rows r of  w_r 2^(scale2 q_r . k_s - lse_r)
//
// after the attention has the rows' denominators.  The product is turned
// around, S^T = K Q^T with 128 keys as M and a block of rows as N, so that a
// thread has one position's scores in its TMEM lane and adds them up by
// itself, row after row: no exchange, no atomics, one order.  It reads the keys
// once more, 2 D bytes a position; keeping the attention's scores instead
// writes and reads 8 bytes per row and position (attn_finish, up to 16 rows).
// Bound by the exponentials with many rows, 16 a clock and SM; by its set-up with
// few tiles a block (26 drafts x 32 heads over 8191 positions: 44 % of the call's 60 us).
#pragma once

#include "kv_attn.cuh"
#include "kv_tc.cuh"
#include "tcgen05.cuh"

namespace voom {
namespace kv {

template <int DP>
struct Sums {
  static constexpr uint32_t KT = 128;
  static constexpr uint32_t NB = DP == 256 ? 128 : 256;  // rows of a block
  static constexpr uint32_t THREADS = 256 + 128 + 32;
  static constexpr uint32_t TILE = KT * DP * 2;
  static constexpr uint32_t Q = NB * DP * 2;
  static constexpr uint32_t RING = (220 * 1024 - Q) / TILE < 12 ? (220 * 1024 - Q) / TILE : 12;
};

struct SumsShared {
  uint64_t full[12], empty[12];
  uint64_t q_full, q_empty, s_full[2], s_empty[2], ready[2], drained;
  uint32_t tmem, failed;
  float2 row[2][256];  // for each softmax warpgroup: minus the row's denominator (log2), its weight
  uint32_t tok[2][256];  // and its token
};

template <int DP>
constexpr uint32_t sums_smem() {
  constexpr uint32_t n = Sums<DP>::Q + Sums<DP>::RING * Sums<DP>::TILE + uint32_t(sizeof(SumsShared));
  static_assert(n <= 227 * 1024 && Sums<DP>::RING >= 2, "shared memory of a block");
  return n;
}

// P: units of all rows of a key head (mblocks = 1), keys = 128.
template <typename T, int DP>
__global__ void __launch_bounds__(Sums<DP>::THREADS, 1) attn_sums(const __grid_constant__ Attn P) {
  using C = Sums<DP>;
  constexpr uint32_t KT = C::KT, NB = C::NB, CH = DP / 8, RING = C::RING, LOAD_WARP = 8, MMA_WARP = 12;
  extern __shared__ __align__(1024) uint8_t smem[];
  SumsShared& sh = *reinterpret_cast<SumsShared*>(smem + C::Q + RING * C::TILE);
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  const uint32_t q_s = smem_addr(smem), ring_s = q_s + C::Q, blocks = ceil_div(P.R, NB);
  auto bar = [](const uint64_t& b) { return smem_addr(&b); };
  auto warp_wait = [&](const uint64_t& b, uint32_t parity) {
    return __all_sync(0xFFFFFFFFu, tc::mbar_wait(smem_addr(&b), parity)) != 0;
  };
  Seg g;
  const bool any = first_seg(P, blockIdx.x, g) && (q_s & 1023u) == 0;
  if (tid == 0) {
    for (uint32_t i = 0; i < RING; i++) {
      tc::mbar_init(bar(sh.full[i]), 128);
      tc::mbar_init(bar(sh.empty[i]), 1);
    }
    tc::mbar_init(bar(sh.q_full), 128);
    tc::mbar_init(bar(sh.q_empty), 1);
    for (int i = 0; i < 2; i++) {
      tc::mbar_init(bar(sh.s_full[i]), 1);
      tc::mbar_init(bar(sh.s_empty[i]), 128);
      tc::mbar_init(bar(sh.ready[i]), 128);
    }
    tc::mbar_init(bar(sh.drained), 1);
    sh.failed = (q_s & 1023u) != 0;
  }
  if (warp == MMA_WARP) tc::tmem_alloc(smem_addr(&sh.tmem), 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = sh.tmem;

  if (any && warp >= LOAD_WARP && warp < MMA_WARP) {
    const uint32_t pw = warp - LOAD_WARP;
    uint32_t it = 0, nq = 0;
    bool ok = true;
    do {
      const uint32_t cs = cache_steps(P, g.len);
      for (uint32_t m = 0; m < blocks && ok; m++) {
        const uint32_t row0 = m * NB, rows = (min(NB, P.R - row0) + 31u) & ~31u;
        if (nq && !(ok = warp_wait(sh.q_empty, (nq - 1) & 1u))) break;
        for (uint32_t r0 = pw * 32; r0 < rows; r0 += 128) {
          const uint32_t row = row0 + r0 + lane, i = row / P.g;
          uint64_t a = 0;
          if (row < P.R && sees(P, g.b, i, i))
            a = reinterpret_cast<uint64_t>(static_cast<const T*>(P.a.d_q) + int64_t(g.b) * P.a.q_b + int64_t(i) * P.a.q_t +
                                           int64_t(g.h * P.g + row % P.g) * P.a.q_h);
#pragma unroll 4
          for (uint32_t k = 0; k < CH; k++) {
            const uint32_t id = k * 32 + lane, r = id / CH, c = id % CH;
            const uint64_t x = __shfl_sync(0xFFFFFFFFu, a, r);
            const bool in = x && c * 8 < P.c.v.D;
            cp16(q_s + sw128(r0 + r, c, NB), in ? reinterpret_cast<const void*>(x + 16 * c) : P.c.v.d_k, in);
          }
        }
        nq++;
        tc::mbar_arrive_copies(bar(sh.q_full));
        for (uint32_t step = g.s0; step < g.s1; step++, it++) {
          const uint32_t place = it % RING;
          if (it >= RING && !(ok = warp_wait(sh.empty[place], (it / RING - 1) & 1u))) break;
          load_keys<T, DP, KT>(P, g, step, cs, pw, lane, ring_s + place * C::TILE, bar(sh.full[place]));
        }
      }
    } while (ok && next_seg(P, g));
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (!ok) sh.failed = 1;
  } else if (any && warp == MMA_WARP) {
    constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t base = (1u << 4) | (fmt << 7) | (fmt << 10) | ((128u >> 4) << 24);
    const bool one = tc::elect_one();
    const uint32_t tm = tc::uniform(tmem), q_lo = (q_s >> 4) | (1u << 16), ring_lo = (ring_s >> 4) | (1u << 16);
    uint32_t it = 0, nq = 0, nt[2] = {0, 0};
    bool ok = true;
    do {
      const uint32_t n = tc::uniform(g.s1 - g.s0);
      for (uint32_t m = 0; m < blocks && ok; m++) {
        const uint32_t idesc = base | ((((min(NB, P.R - m * NB) + 31u) & ~31u) >> 3) << 17);
        if (!(ok = warp_wait(sh.q_full, nq++ & 1u))) break;
        tc::fence_async_smem();
        for (uint32_t i = 0; i < n; i++, it++) {
          const uint32_t slot = i & 1u, place = it % RING;
          ok = warp_wait(sh.full[place], (it / RING) & 1u);
          if (ok && nt[slot]) ok = warp_wait(sh.s_empty[slot], (nt[slot] - 1) & 1u);
          if (!ok) break;
          nt[slot]++;
          tc::fence_async_smem();
          tc::tc_fence_after();
          const uint32_t a = ring_lo + place * (C::TILE >> 4), d = tm + slot * 256u;
          if (one) {
#pragma unroll
            for (uint32_t k = 0; k < DP / 16; k++)
              tc::umma_bf16(d, tc::umma_desc_at(a + (k / 4) * (KT * 8u) + (k % 4) * 2u, tc::kDescHiSw128),
                            tc::umma_desc_at(q_lo + (k / 4) * (NB * 8u) + (k % 4) * 2u, tc::kDescHiSw128), idesc, k > 0);
            tc::umma_commit(bar(sh.s_full[slot]));
            tc::umma_commit(bar(sh.empty[place]));
            if (i + 1 == n) tc::umma_commit(bar(sh.q_empty));
          }
        }
      }
    } while (ok && next_seg(P, g));
    if (one) tc::umma_commit(bar(sh.drained));
    if (!warp_wait(sh.drained, 0)) ok = false;
    if (!ok) sh.failed = 1;
  } else if (any && warp < LOAD_WARP) {
    const uint32_t w = warp >> 2, tr = tid & 127u, lanes = (warp & 3u) << 21;
    uint32_t ns = 0, nr = 0;
    bool ok = true;
    auto together = [&]() {  // the warpgroup's threads, with a bounded wait
      tc::mbar_arrive(bar(sh.ready[w]));
      return warp_wait(sh.ready[w], nr++ & 1u);
    };
    do {
      const uint32_t cs = cache_steps(P, g.len), n = g.s1 - g.s0;
      float* sums = P.a.d_weights + int64_t(g.b) * P.a.w_b + int64_t(g.h) * P.a.w_h;
      for (uint32_t m = 0; m < blocks && ok; m++) {
        const uint32_t row0 = m * NB, nrows = min(NB, P.R - row0), cols = (nrows + 31u) & ~31u;
        if (!(ok = together())) break;  // the last block's denominators are read
        for (uint32_t r = tr; r < cols; r += 128) {
          const uint32_t row = row0 + r, i = row / P.g;
          float2 x = make_float2(-INFINITY, 0.0f);  // a row that is none, or sees nothing, has no weight anywhere
          if (row < P.R && sees(P, g.b, i, i)) {
            x.x = -kLog2e * P.lse[(uint64_t(g.b) * P.a.n + i) * P.a.hq + g.h * P.g + row % P.g];
            x.y = P.a.d_token_weight ? P.a.d_token_weight[uint64_t(g.b) * P.a.n + i] : 1.0f;
          }
          sh.row[w][r] = x;
          sh.tok[w][r] = row < P.R ? i : P.a.n;
        }
        if (!(ok = together())) break;
        for (uint32_t t = w; t < n; t += 2) {
          const uint32_t step = g.s0 + t;
          if (!(ok = warp_wait(sh.s_full[w], ns++ & 1u))) break;
          tc::tc_fence_after();
          const bool fresh = step >= cs;
          const uint32_t j = (fresh ? step - cs : step) * KT + tr;
          float acc[2] = {0.0f, 0.0f};
          for (uint32_t c = 0; c < cols; c += 32) {
            uint32_t s[32];
            tc::tmem_ld32(tmem + lanes + w * 256u + c, s);
            tc::tmem_wait_ld();
            tc::tmem_hold(s);
            const float4* row = reinterpret_cast<const float4*>(&sh.row[w][c]);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float4 x = row[e / 2];
              float p = exp2_fast(fmaf(__uint_as_float(s[e]), P.scale2, x.x));
              float q = exp2_fast(fmaf(__uint_as_float(s[e + 1]), P.scale2, x.z));
              if (fresh) {
                const uint32_t i0 = sh.tok[w][c + e], i1 = sh.tok[w][c + e + 1];
                if (i0 >= P.a.n || j >= P.a.n || !sees(P, g.b, i0, j)) p = 0.0f;
                if (i1 >= P.a.n || j >= P.a.n || !sees(P, g.b, i1, j)) q = 0.0f;
              }
              // rows that are none have queries of 0, whose score at an infinite key is NaN: not even times 0
              if (x.y != 0.0f) acc[0] = fmaf(x.y, p, acc[0]);
              if (x.w != 0.0f) acc[1] = fmaf(x.w, q, acc[1]);
            }
          }
          tc::tc_fence_before();
          tc::mbar_arrive(bar(sh.s_empty[w]));
          const float got = acc[0] + acc[1];
          if (fresh ? j < P.a.n : j < g.len) sums[fresh ? g.len + j : j] += got;
        }
      }
    } while (ok && next_seg(P, g));
    if (!ok) sh.failed = 1;
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == MMA_WARP) tc::tmem_dealloc(tmem, 512);
  if (tid == 0 && sh.failed && P.a.d_status) atomicOr(P.a.d_status, 1u);
}

}  // namespace kv
}  // namespace voom
