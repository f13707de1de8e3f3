// Cache attention of up to eight rows per key head, scored: warp-level matrix
// instructions with the rows as their narrow side.
//
//   S^T = K Q^T,   O^T += V^T P^T      (16 keys, or 16 values of a head, by 8 rows)
//
// One token of up to eight query heads to a key head is the usual call; attn_rows
// gives it matrices of 16 rows, most of them empty.  Turned around, a tile takes
// half the products, a lane holds half the scores and output, and what a capped or
// biased score costs more is paid for real rows only.  As there, each warp is a
// stream of its own, with three tiles of keys and values under way, and the block
// joins when a unit ends.  Whole tiles come by TMA where it can read the cache: a
// gather of 16 positions takes two hundred instructions, as many as all the rest.
// A row's maximum is raised only when it grows by more than 2^8, so that usually
// one vote stands for the lanes' exchange; until then probabilities are at most 2^8.
//
// Bound by the cache's bytes where requests are long.  Measured: 32 requests of up to
// 16000 positions in pages of 16, 4 rows of 128, capped: 180 us a call, 177 of it here,
// 5.8 TB/s (88 % of what a copy reaches); the same in attn_rows
// 223.  One token over a window of 1000, heads of 64: 13 us, a block's chain of loads.
// 168, 200 and 255 registers a thread (heads of 64, 128, 256), none spilled.
#pragma once

#include "kv_rows.cuh"
#include "tcgen05.cuh"

namespace voom {
namespace kv {

template <int DP>
struct Few {
  static constexpr uint32_t W = row_warps(DP, true), TILE = row_tile(DP, true), KT = row_keys(DP, true);
  static constexpr uint32_t JOIN = 64, LDJ = JOIN + 4;  // values of a head that the warps join at a time, and their rows
  static constexpr uint32_t STAGES = W * kRowStages * TILE;
  static constexpr uint32_t SMEM = STAGES + W * kFewRows * LDJ * 4 + 2 * W * kFewRows * 4 + kFewRows * DP * 2 + W * kRowStages * 8;
  static_assert(SMEM <= 227 * 1024 && KT % 16 == 0, "shared memory of a block; whole matrix instructions");
};

__device__ __forceinline__ uint32_t transposed8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <typename T, int DP>
__global__ void __launch_bounds__(32 * Few<DP>::W, 1) attn_few(const __grid_constant__ Attn P) {
  using F = Few<DP>;
  constexpr uint32_t W = F::W, TILE = F::TILE, KT = F::KT, CH = DP / 8, KB = KT / 16, DT = DP / 16;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, quad = lane & 3u, oct = lane >> 2;
  const uint32_t stage0 = smem_addr(smem) + warp * kRowStages * TILE;
  float* s_join = reinterpret_cast<float*>(smem + F::STAGES);  // [warp][row][LDJ]
  float* s_m = s_join + W * kFewRows * F::LDJ;                 // [warp][row]
  float* s_l = s_m + W * kFewRows;
  uint8_t* s_q = reinterpret_cast<uint8_t*>(s_l + W * kFewRows);
  const uint32_t q_addr = smem_addr(s_q), bars = smem_addr(s_q + kFewRows * DP * 2) + warp * kRowStages * 8;

  Seg g;
  if (!first_seg<true>(P, blockIdx.x, g)) return;
  if (lane == 0)
    for (uint32_t i = 0; i < kRowStages; i++) tc::mbar_init(bars + 8 * i, 1);
  __syncwarp();
  const bool tma = P.box && (stage0 & 1023u) == 0;
  uint32_t came = 0, due = 0, phase = 0;  // slots that TMA filled last, is to be waited for in; their barriers' parities
  bool ok = true, more = true;
  Seg pg = g;  // where the loads are, and what they know of their segment
  uint32_t ps = pg.s0 + warp, p_cached = 0, p_first = 0, p_none = 0;
  auto look = [&]() {
    p_first = first_tile(P, pg.len);
    p_cached = (pg.len + KT - 1) / KT - p_first;
    p_none = window_none(P, pg.len);
  };
  look();
  auto produce = [&](uint32_t slot) {
    while (more && ps >= pg.s1) {
      more = next_seg<true>(P, pg);
      ps = pg.s0 + warp;
      if (more) look();
    }
    if (more) {
      const uint32_t dst = stage0 + slot * TILE, p0 = (p_first + ps) * KT;
      if (tma && ps < p_cached && p0 + KT <= pg.len && p0 >= p_none) {
        if (!(came >> slot & 1u)) {  // what was copied there otherwise comes first
          tc::fence_async_smem();
          __syncwarp();
        }
        came |= 1u << slot;
        due |= 1u << slot;
        if (lane == 0) tc::mbar_arrive_expect(bars + 8 * slot, TILE);
        __syncwarp();
        if (lane < KT / P.box) {
          const uint32_t s = p0 + lane * P.box, at = P.c.page_of(s);
          const int32_t w = P.c.page_box(pg.b, at);
          const uint32_t y = P.c.v.d_table ? s - at * P.c.v.page : s;
#pragma unroll
          for (uint32_t x = 0; x < DP; x += 64) {
            const uint32_t to = dst + (x / 64) * (KT * 128u) + lane * P.box * 128u;
            tc::tma_load4(to, &P.k_map, bars + 8 * slot, int32_t(x), int32_t(y), int32_t(pg.h), w);
            tc::tma_load4(to + TILE / 2, &P.v_map, bars + 8 * slot, int32_t(x), int32_t(y), int32_t(pg.h), w);
          }
        }
      } else {
        load_tile<T, DP, true, true>(P, pg, pg.h, ps, dst);
        came &= ~(1u << slot);
      }
      ps += W;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (uint32_t i = 0; i + 1 < kRowStages; i++) produce(i);

  uint32_t slot = 0;
  do {
    const uint32_t h = g.h, nrows = P.R;
    const uint32_t w0 = first_tile(P, g.len), cs = (g.len + KT - 1) / KT - w0;
    // a position from which on all rows see every key of the cache
    const uint32_t all_from = window_all(P, g.len);
    // the unit's queries
    for (uint32_t i = tid; i < kFewRows * CH; i += 32 * W) {
      const uint32_t r = i / CH, c = i % CH;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (r < nrows && c * 8 < P.c.v.D && sees(P, g.b, r / P.g, r / P.g))
        x = *reinterpret_cast<const uint4*>(static_cast<const T*>(P.a.d_q) + int64_t(g.b) * P.a.q_b + int64_t(r / P.g) * P.a.q_t +
                                            int64_t(h * P.g + r % P.g) * P.a.q_h + 8 * c);
      *reinterpret_cast<uint4*>(s_q + row_off<DP>(r, c)) = x;
    }
    // the lane's two rows
    uint32_t tok[2];
    int32_t behind[2];
    float slope2[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const uint32_t r = min(2 * quad + e, nrows - 1);
      tok[e] = r / P.g;
      behind[e] = depth_of(P, g.b, tok[e]);
      slope2[e] = slope2_of(P, h * P.g + r % P.g);
    }
    const F2 slopes = make2(slope2[0], slope2[1]), back = make2(-float(behind[0]), -float(behind[1]));
    __syncthreads();
    uint32_t qb[DT][2];
#pragma unroll
    for (uint32_t k = 0; k < DT; k += 2) {
      uint32_t x[4];
      ldsm4(x, q_addr + row_off<DP>(lane & 7u, 2 * k + (lane >> 3)));
      qb[k][0] = x[0];
      qb[k][1] = x[1];
      qb[k + 1][0] = x[2];
      qb[k + 1][1] = x[3];
    }
    float o[DT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, rest[2] = {0.0f, 0.0f};  // l + rest: the denominator
#pragma unroll
    for (uint32_t d = 0; d < DT; d++)
#pragma unroll
      for (int i = 0; i < 4; i++) o[d][i] = 0.0f;
    for (uint32_t step = g.s0 + warp; step < g.s1; step += W) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kRowStages - 2) : "memory");
      if (due >> slot & 1u) {
        ok = __all_sync(0xFFFFFFFFu, tc::mbar_wait(bars + 8 * slot, phase >> slot & 1u)) && ok;
        if (!ok) more = false;  // only what is under way is still waited for
        due &= ~(1u << slot);
        phase ^= 1u << slot;
      }
      __syncwarp();
      produce(slot == 0 ? kRowStages - 1 : slot - 1);
      const uint32_t ks = stage0 + slot * TILE, vs = ks + TILE / 2;
      // the products: s[kb][2 x + e] of key 16 kb + 8 x + oct and row 2 quad + e
      float s[KB][4];
#pragma unroll
      for (uint32_t kb = 0; kb < KB; kb++) {
#pragma unroll
        for (int i = 0; i < 4; i++) s[kb][i] = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < DT; k++) {
          uint32_t a[4];
          ldsm4(a, ks + sw128(16 * kb + (lane & 15u), 2 * k + (lane >> 4), KT));
          mma16816<T>(s[kb], a, qb[k][0], qb[k][1]);
        }
      }
      const bool fresh = step >= cs;
      const uint32_t p0 = (w0 + step) * KT;  // of a cached tile: its first position
      uint32_t odd = 0;                      // keys that some rows do not see and whose values are not all finite
      // the scores
      if (fresh && P.a.d_mask) {  // a tree's tokens stand at their depths
#pragma unroll
        for (uint32_t kb = 0; kb < KB; kb++)
#pragma unroll
          for (int x = 0; x < 2; x++) {
            const float at = float(depth_of(P, g.b, (step - cs) * KT + 16 * kb + 8 * x + oct));
            take2(scored2(P, make2(s[kb][2 * x], s[kb][2 * x + 1]), mul2(slopes, add2(make2(at, at), back))), s[kb][2 * x], s[kb][2 * x + 1]);
          }
      } else {
        // the key's place from the cache's end
        const float at = float((fresh ? int32_t((step - cs) * KT) : int32_t(p0) - int32_t(g.len)) + int32_t(oct));
        auto all = [&](auto kind) {
#pragma unroll
          for (uint32_t kb = 0; kb < KB; kb++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
              const float y = at + float(16 * kb + 8 * x);
              take2(scored2<decltype(kind)::value>(P, make2(s[kb][2 * x], s[kb][2 * x + 1]), mul2(slopes, add2(make2(y, y), back))), s[kb][2 * x],
                    s[kb][2 * x + 1]);
            }
        };
        if (P.cap_in != 0.0f) all(Kind<kAny>());
        else all(Kind<kPlain>());
      }
      // masks: positions past the length, what a window leaves out, and the new tokens that a row does not see
      if (fresh || p0 + KT > g.len || p0 < all_from) {
#pragma unroll
        for (uint32_t kb = 0; kb < KB; kb++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t k = 16 * kb + 8 * (i >> 1) + oct, e = i & 1;
            bool in;
            if (fresh) {
              const uint32_t j = (step - cs) * KT + k;
              in = j < P.a.n && sees(P, g.b, tok[e], j) && in_window(P, depth_of(P, g.b, j) - behind[e]);
            } else {
              in = p0 + k < g.len && in_window(P, int32_t(p0 + k) - int32_t(g.len) - behind[e]);
            }
            if (!in) s[kb][i] = -INFINITY;
          }
        if (P.a.n > 1 && (fresh || p0 < all_from)) {  // a probability of 0 must not meet an infinite or NaN value: those are taken out
          bool found = false;
          for (uint32_t id = lane; id < KT * CH; id += 32) {
            const uint32_t r = id / CH, at = vs - smem_addr(smem) + sw128(r, id % CH, KT);
            if (odd_values<T>(*reinterpret_cast<const uint4*>(smem + at))) {
              *reinterpret_cast<uint4*>(smem + at) = make_uint4(0, 0, 0, 0);
              odd |= 1u << r;
              found = true;
            }
          }
          if (__any_sync(0xFFFFFFFFu, found)) {
            odd = __reduce_or_sync(0xFFFFFFFFu, odd);
            tc::fence_async_smem();  // before TMA writes there again
          }
          __syncwarp();
        }
      }
      if (P.scores) {
        const uint32_t at = fresh ? P.score_new + (step - cs) * KT : p0;
#pragma unroll
        for (uint32_t kb = 0; kb < KB; kb++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t r = 2 * quad + (i & 1);
            if (r < nrows) P.scores[(uint64_t(g.b * P.c.v.hk + h) * P.R + r) * P.score_ld + at + 16 * kb + 8 * (i >> 1) + oct] = s[kb][i];
          }
      }
      // the probabilities
      float top[2] = {s[0][0], s[0][1]};
#pragma unroll
      for (uint32_t kb = 0; kb < KB; kb++)
#pragma unroll
        for (int i = kb ? 0 : 2; i < 4; i++) top[i & 1] = fmaxf(top[i & 1], s[kb][i]);
      if (__any_sync(0xFFFFFFFFu, top[0] > m[0] + 8.0f || top[1] > m[1] + 8.0f)) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float t = top[e];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, d));
          t = t > m[e] + 8.0f ? t : m[e];
          f[e] = t == m[e] ? 1.0f : exp2_fast(m[e] - t);
          m[e] = t;
          l[e] *= f[e];
          rest[e] *= f[e];
        }
#pragma unroll
        for (uint32_t d = 0; d < DT; d++)
#pragma unroll
          for (int i = 0; i < 4; i++) o[d][i] *= f[i & 1];
      }
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const float base = m[e] == -INFINITY ? 0.0f : m[e] - kLift<T, 8>;
        float sum = 0.0f;
#pragma unroll
        for (uint32_t kb = 0; kb < KB; kb++)
#pragma unroll
          for (int x = 0; x < 2; x++) sum += s[kb][2 * x + e] = exp2_fast(s[kb][2 * x + e] - base);
        add_kept(l[e], rest[e], sum);
      }
      // o += p v
#pragma unroll
      for (uint32_t kb = 0; kb < KB; kb++) {
        const uint32_t p0t = transposed8(pack2(s[kb][0], s[kb][1], T())), p1t = transposed8(pack2(s[kb][2], s[kb][3], T()));
#pragma unroll
        for (uint32_t d = 0; d < DT; d++) {
          uint32_t a[4];
          ldsm4_t(a, vs + sw128(16 * kb + (lane & 7u) + ((lane >> 4) << 3), 2 * d + (lane >> 3 & 1u), KT));
          mma16816<T>(o[d], a, p0t, p1t);
        }
      }
      if (odd) {  // rare: what was taken out, for the rows that see it
#pragma unroll
        for (uint32_t kb = 0; kb < KB; kb++)
#pragma unroll
          for (int x = 0; x < 2; x++)
            for (uint32_t q = 0; q < 8; q++) {
              const uint32_t k = 16 * kb + 8 * x + q;
              if (!(odd >> k & 1u)) continue;
              const uint32_t j = (step - cs) * KT + k;
              const T* v = static_cast<const T*>(P.a.d_vn) + int64_t(g.b) * P.a.vn_b + int64_t(j) * P.a.vn_t + int64_t(h) * P.a.vn_h;
              const int32_t key = fresh ? depth_of(P, g.b, j) : int32_t(p0 + k) - int32_t(g.len);
              int64_t ko, vo;
              if (!fresh) {
                if (!P.c.row_at(g.b, h, p0 + k, ko, vo)) continue;  // (was zeros)
                v = static_cast<const T*>(P.c.v.d_v) + vo;
              }
#pragma unroll
              for (int e = 0; e < 2; e++) {
                const float p = __shfl_sync(0xFFFFFFFFu, s[kb][2 * x + e], q << 2 | quad);
                if (2 * quad + e >= nrows || (fresh && !sees(P, g.b, tok[e], j)) || !in_window(P, key - behind[e])) continue;
#pragma unroll
                for (uint32_t d = 0; d < DT; d++)
#pragma unroll
                  for (int y = 0; y < 2; y++) {
                    const uint32_t at = 16 * d + 8 * y + oct;
                    // the whole chunk of eight was taken out
                    if (at < P.c.v.D && odd_values<T>(*reinterpret_cast<const uint4*>(v + (at & ~7u)))) o[d][2 * y + e] += p * elem<T>(v[at]);
                  }
              }
            }
      }
      slot = slot + 1 == kRowStages ? 0 : slot + 1;
    }
    // join the warps' sums, JOIN values at a time
#pragma unroll
    for (int e = 0; e < 2; e++) {
      l[e] += rest[e];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[e] += __shfl_xor_sync(0xFFFFFFFFu, l[e], d);
      if (oct == 0) {
        const uint32_t r = 2 * quad + e;
        const bool token = r < nrows && sees(P, g.b, tok[e], tok[e]);  // else it has seen nothing
        s_m[warp * kFewRows + r] = token ? m[e] - kLift<T, 8> : -INFINITY;  // what o and l are relative to
        s_l[warp * kFewRows + r] = token ? l[e] : 0.0f;
      }
    }
    const bool whole = g.s0 == 0 && g.s1 == g.steps;
    // a unit that starts in this block and goes on goes to the second slot
    float* part = whole ? nullptr : slot_of(P, 2 * blockIdx.x + (g.s0 == 0 ? 1u : 0u));
#pragma unroll
    for (uint32_t d0 = 0; d0 < DP; d0 += F::JOIN) {
#pragma unroll
      for (uint32_t d = 0; d < F::JOIN / 16; d++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          s_join[(warp * kFewRows + 2 * quad + (i & 1)) * F::LDJ + 16 * d + 8 * (i >> 1) + oct] = o[d0 / 16 + d][i];
      __syncthreads();
      for (uint32_t i = tid; i < nrows * (F::JOIN / 2); i += 32 * W) {
        const uint32_t r = i / (F::JOIN / 2), d = 2 * (i % (F::JOIN / 2));
        if (d0 + d >= P.c.v.D) continue;
        float mm[W], top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < W; w++) top = fmaxf(top, mm[w] = s_m[w * kFewRows + r]);
        const float base = top == -INFINITY ? 0.0f : top;
        float2 y = make_float2(0.0f, 0.0f);
#pragma unroll
        for (uint32_t w = 0; w < W; w++) {
          const float f = exp2_fast(mm[w] - base);
          const float2 v = *reinterpret_cast<const float2*>(s_join + (w * kFewRows + r) * F::LDJ + d);
          sum += f * s_l[w * kFewRows + r];
          y.x += f * v.x;
          y.y += f * v.y;
        }
        if (whole) {
          const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          T* out = static_cast<T*>(P.a.d_out) + int64_t(g.b) * P.a.o_b + int64_t(r / P.g) * P.a.o_t + int64_t(h * P.g + r % P.g) * P.a.o_h +
                   d0 + d;
          *reinterpret_cast<uint32_t*>(out) = sum == 0.0f ? 0u : pack2(y.x * inv, y.y * inv, T());
          if (P.lse && d0 + d == 0) P.lse[(uint64_t(g.b) * P.a.n + r / P.g) * P.a.hq + h * P.g + r % P.g] = kLn2 * (base + log2f(sum));
        } else {
          *reinterpret_cast<float2*>(part + r * P.ld_o + d0 + d) = y;
          if (d0 + d == 0) {
            part[P.rows * P.ld_o + 2 * r] = top;
            part[P.rows * P.ld_o + 2 * r + 1] = sum;
          }
        }
      }
      __syncthreads();
    }
  } while (next_seg<true>(P, g));
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (!ok && lane == 0 && P.a.d_status) atomicOr(P.a.d_status, 1u);
}

}  // namespace kv
}  // namespace voom
