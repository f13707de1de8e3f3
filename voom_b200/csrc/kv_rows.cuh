// Cache attention of few rows per key head: warp-level matrix instructions.
//
//   z = scale2 * q . k   (log2 units),   o = sum 2^(z - m) v,   l = sum 2^(z - m)
//
// Bound by the cache's bytes: 16 (32) rows make 16 (32) multiply-adds of every
// value read, far below what even the warp-level instructions take in.  What
// it needs is bytes in flight, so each of a block's four warps is a stream of
// its own: it walks every fourth tile of keys (16 KB of keys and values) with
// three tiles in flight through cp.async into its own shared memory, and keeps
// its own running maximum, sum and output in registers.  No warp waits for
// another until a unit ends and the four join.  192 KB in flight per SM.
// Measured: one token over 131072 positions, 8 key heads of 128, with weight sums:
// 119 us a call, 84 % of it here, 5.4 TB/s (82 % of what a copy reaches); 32 requests
// of up to 16000 positions in pages of 16: 197 us, 96 % of it here.  At 255
// registers a thread some values spill (32 rows, or heads of 256: 92-152 bytes).
#pragma once

#include "kv_attn.cuh"

namespace voom {
namespace kv {

constexpr uint32_t kRowWarps = 4;
constexpr uint32_t kRowStages = 3;
constexpr uint32_t kJoin = 64;  // values of a head that the warps join at a time

// Keys of a tile: 8 KB of keys and 8 KB of values.
__host__ __device__ constexpr uint32_t row_keys(uint32_t dp) { return 4096u / dp; }
// Shared memory: the warps' stages, the joining buffer, the rows' maxima and
// sums, and the queries.
__host__ __device__ constexpr uint32_t row_smem(uint32_t dp, uint32_t mt) {
  return kRowWarps * kRowStages * 16384u + kRowWarps * 16u * kJoin * 4u + 2u * kRowWarps * 16u * mt * 4u + 16u * mt * dp * 2u;
}
static_assert(row_smem(128, 2) <= 227 * 1024 && row_smem(256, 1) <= 227 * 1024, "shared memory of a block");

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// Byte offset of 16-byte chunk c of row r: rows of DP values, the chunk's low
// three bits turned by the row, so that eight rows' equal chunks (a matrix
// load) lie in different banks.
template <int DP>
__device__ __forceinline__ uint32_t row_off(uint32_t r, uint32_t c) {
  return r * (DP * 2u) + ((c ^ (r & 7u)) << 4);
}

// One tile's loads: K to dst, V to dst + 8 KB.  Rows past the valid ones, and
// new tokens that are none, become zeros.
template <typename T, int DP>
__device__ __forceinline__ void load_tile(const Attn& P, const Seg& g, uint32_t h, uint32_t step, uint32_t dst) {
  constexpr uint32_t KT = row_keys(DP), CH = DP / 8, per = (KT + 31) / 32;
  const uint32_t lane = threadIdx.x & 31u, cs = cache_steps(P, g.len);
  // a lane finds the rows lane, lane + 32; the loads take them by shuffles
  uint64_t ka[per], va[per];
#pragma unroll
  for (uint32_t i = 0; i < per; i++) {
    const uint32_t r = lane + 32 * i;
    ka[i] = va[i] = 0;
    if (r < KT) {
      if (step < cs) {
        const uint32_t s = step * KT + r;
        int64_t ko, vo;
        if (s < g.len && P.c.row_at(g.b, h, s, ko, vo)) {
          ka[i] = reinterpret_cast<uint64_t>(static_cast<const T*>(P.c.v.d_k) + ko);
          va[i] = reinterpret_cast<uint64_t>(static_cast<const T*>(P.c.v.d_v) + vo);
        }
      } else {
        const uint32_t j = (step - cs) * KT + r;
        if (j < P.a.n && sees(P, g.b, j, j)) {
          ka[i] = reinterpret_cast<uint64_t>(static_cast<const T*>(P.a.d_kn) + int64_t(g.b) * P.a.kn_b +
                                             int64_t(j) * P.a.kn_t + int64_t(h) * P.a.kn_h);
          va[i] = reinterpret_cast<uint64_t>(static_cast<const T*>(P.a.d_vn) + int64_t(g.b) * P.a.vn_b +
                                             int64_t(j) * P.a.vn_t + int64_t(h) * P.a.vn_h);
        }
      }
    }
  }
#pragma unroll
  for (uint32_t it = 0; it < KT * CH / 32; it++) {
    const uint32_t id = it * 32 + lane, r = id / CH, c = id % CH;
    const uint64_t k = __shfl_sync(0xFFFFFFFFu, ka[(it * 32 / CH) / 32], r & 31u);
    const uint64_t v = __shfl_sync(0xFFFFFFFFu, va[(it * 32 / CH) / 32], r & 31u);
    const bool in = c * 8 < P.c.v.D;
    const uint32_t off = row_off<DP>(r, c);
    const void* any = P.c.v.d_k;  // a readable address for the chunks that are zeros
    cp16(dst + off, in && k ? reinterpret_cast<const void*>(k + 16 * c) : any, in && k);
    cp16(dst + 8192u + off, in && v ? reinterpret_cast<const void*>(v + 16 * c) : any, in && v);
  }
}

// DP: head size rounded up to 64, 128 or 256.  MT: blocks of 16 rows.
template <typename T, int DP, int MT>
__global__ void __launch_bounds__(32 * kRowWarps, 1) attn_rows(const __grid_constant__ Attn P) {
  constexpr uint32_t KT = row_keys(DP), CH = DP / 8, NT = KT / 8, DT = DP / 8, LDJ = kJoin, ROWS = 16 * MT;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, quad = lane & 3u, oct = lane >> 2;
  const uint32_t stage0 = smem_addr(smem) + warp * kRowStages * 16384u;
  float* s_join = reinterpret_cast<float*>(smem + kRowWarps * kRowStages * 16384u);  // [warp][16][LDJ]
  float* s_m = s_join + kRowWarps * 16 * LDJ;                                        // [warp][ROWS]
  float* s_l = s_m + kRowWarps * ROWS;
  uint8_t* s_q = reinterpret_cast<uint8_t*>(s_l + kRowWarps * ROWS);
  const uint32_t q_addr = smem_addr(s_q);

  Seg g;
  if (!first_seg(P, blockIdx.x, g)) return;
  Seg pg = g;  // where the loads are
  bool more = true;
  uint32_t ps = pg.s0 + warp;
  auto produce = [&](uint32_t slot) {
    while (more && ps >= pg.s1) {
      more = next_seg(P, pg);
      ps = pg.s0 + warp;
    }
    if (more) {
      load_tile<T, DP>(P, pg, pg.h, ps, stage0 + slot * 16384u);
      ps += kRowWarps;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (uint32_t i = 0; i + 1 < kRowStages; i++) produce(i);

  uint32_t slot = 0;
  do {
    const uint32_t h = g.h, row0 = g.m * ROWS, nrows = min(ROWS, P.R - row0);
    const uint32_t cs = cache_steps(P, g.len);
    // the unit's queries
    for (uint32_t i = tid; i < ROWS * CH; i += 32 * kRowWarps) {
      const uint32_t r = i / CH, c = i % CH, row = row0 + r;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (r < nrows && c * 8 < P.c.v.D && sees(P, g.b, row / P.g, row / P.g))
        x = *reinterpret_cast<const uint4*>(static_cast<const T*>(P.a.d_q) + int64_t(g.b) * P.a.q_b +
                                            int64_t(row / P.g) * P.a.q_t + int64_t(h * P.g + row % P.g) * P.a.q_h + 8 * c);
      *reinterpret_cast<uint4*>(s_q + row_off<DP>(r, c)) = x;
    }
    __syncthreads();
    float o[MT][DT][4], m[MT][2], l[MT][2], rest[MT][2];  // l + rest: the denominator
#pragma unroll
    for (int t = 0; t < MT; t++) {
#pragma unroll
      for (uint32_t d = 0; d < DT; d++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[t][d][e] = 0.0f;
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = rest[t][0] = rest[t][1] = 0.0f;
    }
    for (uint32_t step = g.s0 + warp; step < g.s1; step += kRowWarps) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kRowStages - 2) : "memory");
      __syncwarp();
      produce(slot == 0 ? kRowStages - 1 : slot - 1);
      const uint32_t ks = stage0 + slot * 16384u, vs = ks + 8192u;
      // z = q . k
      float z[MT][NT][4];
#pragma unroll
      for (int t = 0; t < MT; t++)
#pragma unroll
        for (uint32_t j = 0; j < NT; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) z[t][j][e] = 0.0f;
#pragma unroll
      for (uint32_t c = 0; c < CH; c += 4) {  // 32 of the head's values
        uint32_t a[MT][2][4];
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
          for (int x = 0; x < 2; x++)
            ldsm4(a[t][x], q_addr + row_off<DP>(16 * t + (lane & 15u), c + 2 * x + (lane >> 4)));
#pragma unroll
        for (uint32_t j = 0; j < NT; j++) {
          uint32_t b[4];
          ldsm4(b, ks + row_off<DP>(8 * j + (lane & 7u), c + (lane >> 3)));
#pragma unroll
          for (int t = 0; t < MT; t++) {
            mma16816<T>(z[t][j], a[t][0], b[0], b[1]);
            mma16816<T>(z[t][j], a[t][1], b[2], b[3]);
          }
        }
      }
      // masks: positions past the length, and the new tokens that a row does not see
      const bool fresh = step >= cs;
      uint32_t odd = 0, odd_hi = 0;  // new tokens of the tile whose values are not all finite
      if (fresh || step * KT + KT > g.len) {
        const uint32_t j0 = fresh ? (step - cs) * KT : 0u, valid = fresh ? 0u : g.len - step * KT;
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
          for (int x = 0; x < 2; x++) {
            const uint32_t i = (row0 + 16 * t + oct + 8 * x) / P.g;
            const uint32_t lo = fresh ? sees32(P, g.b, i, j0) : valid >= 32 ? 0xFFFFFFFFu : (1u << valid) - 1u;
            const uint32_t hi = KT <= 32 ? 0u : fresh ? sees32(P, g.b, i, j0 + 32) : valid >= 64 ? 0xFFFFFFFFu : valid <= 32 ? 0u : (1u << (valid - 32)) - 1u;
#pragma unroll
            for (uint32_t j = 0; j < NT; j++)
#pragma unroll
              for (int e = 0; e < 2; e++) {
                const uint32_t k = 8 * j + 2 * quad + e;
                if (!((k < 32 ? lo : hi) >> (k & 31u) & 1u)) z[t][j][2 * x + e] = -INFINITY;
              }
          }
        if (fresh) {  // a probability of 0 must not meet an infinite or NaN value: take those out here
          bool found = false;
          for (uint32_t id = lane; id < KT * CH; id += 32) {
            const uint32_t r = id / CH, at = vs - smem_addr(smem) + row_off<DP>(r, id % CH);
            if (odd_values<T>(*reinterpret_cast<const uint4*>(smem + at))) {
              *reinterpret_cast<uint4*>(smem + at) = make_uint4(0, 0, 0, 0);
              if (r < 32) odd |= 1u << r;
              else odd_hi |= 1u << (r - 32);
              found = true;
            }
          }
          if (__any_sync(0xFFFFFFFFu, found)) {
            odd = __reduce_or_sync(0xFFFFFFFFu, odd);
            odd_hi = __reduce_or_sync(0xFFFFFFFFu, odd_hi);
          }
          __syncwarp();
        }
      }
#pragma unroll
      for (int t = 0; t < MT; t++) {
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (uint32_t j = 0; j < NT; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            z[t][j][e] *= P.scale2;
            top[e >> 1] = fmaxf(top[e >> 1], z[t][j][e]);
          }
        if (P.scores) {
          const uint32_t at = fresh ? P.score_new + (step - cs) * KT : step * KT;
#pragma unroll
          for (int x = 0; x < 2; x++) {
            const uint32_t r = 16 * t + oct + 8 * x;
            if (r < nrows) {
              float* to = P.scores + (uint64_t(g.b * P.c.v.hk + h) * P.R + row0 + r) * P.score_ld + at + 2 * quad;
#pragma unroll
              for (uint32_t j = 0; j < NT; j++)
                *reinterpret_cast<float2*>(to + 8 * j) = make_float2(z[t][j][2 * x], z[t][j][2 * x + 1]);
            }
          }
        }
        float f[2];
#pragma unroll
        for (int x = 0; x < 2; x++) {
          top[x] = fmaxf(top[x], __shfl_xor_sync(0xFFFFFFFFu, top[x], 1));
          top[x] = fmaxf(top[x], __shfl_xor_sync(0xFFFFFFFFu, top[x], 2));
          top[x] = fmaxf(top[x], m[t][x]);
          f[x] = top[x] == m[t][x] ? 1.0f : exp2_fast(m[t][x] - top[x]);  // (nothing seen yet: -inf both)
          m[t][x] = top[x];
          l[t][x] *= f[x];
          rest[t][x] *= f[x];
        }
        if (__any_sync(0xFFFFFFFFu, f[0] != 1.0f || f[1] != 1.0f)) {
#pragma unroll
          for (uint32_t d = 0; d < DT; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[t][d][e] *= f[e >> 1];
        }
#pragma unroll
        for (int x = 0; x < 2; x++) {
          const float base = m[t][x] == -INFINITY ? 0.0f : m[t][x];
          float sum = 0.0f;  // of the tile
#pragma unroll
          for (uint32_t j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const float p = exp2_fast((z[t][j][2 * x + e] - base) + kLift<T, 0>);
              z[t][j][2 * x + e] = p;
              sum += p;
            }
          add_kept(l[t][x], rest[t][x], sum);
        }
      }
      // o += p v
#pragma unroll
      for (uint32_t j = 0; j < NT; j += 2) {
        uint32_t a[MT][4];
#pragma unroll
        for (int t = 0; t < MT; t++) {
          a[t][0] = pack2(z[t][j][0], z[t][j][1], T());
          a[t][1] = pack2(z[t][j][2], z[t][j][3], T());
          a[t][2] = pack2(z[t][j + 1][0], z[t][j + 1][1], T());
          a[t][3] = pack2(z[t][j + 1][2], z[t][j + 1][3], T());
        }
#pragma unroll
        for (uint32_t d = 0; d < DT; d += 2) {
          uint32_t b[4];
          ldsm4_t(b, vs + row_off<DP>(8 * j + (lane & 15u), d + (lane >> 4)));
#pragma unroll
          for (int t = 0; t < MT; t++) {
            mma16816<T>(o[t][d], a[t], b[0], b[1]);
            mma16816<T>(o[t][d + 1], a[t], b[2], b[3]);
          }
        }
      }
      if (odd | odd_hi) {  // rare: what was taken out, for the rows that see it
#pragma unroll
        for (uint32_t j = 0; j < NT; j++)
#pragma unroll
          for (int e = 0; e < 2; e++)
            for (uint32_t s = 0; s < 4; s++) {
              const uint32_t k = 8 * j + 2 * s + e, tok = (step - cs) * KT + k;
              if (!((k < 32 ? odd : odd_hi) >> (k & 31u) & 1u)) continue;
              const T* v = static_cast<const T*>(P.a.d_vn) + int64_t(g.b) * P.a.vn_b + int64_t(tok) * P.a.vn_t +
                           int64_t(h) * P.a.vn_h;
#pragma unroll
              for (int t = 0; t < MT; t++)
#pragma unroll
                for (int x = 0; x < 2; x++) {
                  const float p = __shfl_sync(0xFFFFFFFFu, z[t][j][2 * x + e], (lane & ~3u) | s);
                  const uint32_t i = (row0 + 16 * t + oct + 8 * x) / P.g;
                  if (i >= P.a.n || !sees(P, g.b, i, tok)) continue;
#pragma unroll
                  for (uint32_t d = 0; d < DT; d++)
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                      const uint32_t at = 8 * d + 2 * quad + y;
                      // the whole chunk of eight was taken out
                      if (at < P.c.v.D && odd_values<T>(*reinterpret_cast<const uint4*>(v + (at & ~7u))))
                        o[t][d][2 * x + y] += p * elem<T>(v[at]);
                    }
                }
            }
      }
      slot = slot + 1 == kRowStages ? 0 : slot + 1;
    }
    // join the four warps' sums, 16 rows and 64 values at a time
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
      for (int x = 0; x < 2; x++) {
        l[t][x] += rest[t][x];
        l[t][x] += __shfl_xor_sync(0xFFFFFFFFu, l[t][x], 1);
        l[t][x] += __shfl_xor_sync(0xFFFFFFFFu, l[t][x], 2);
        if (quad == 0) {
          const uint32_t r = 16 * t + oct + 8 * x, i = (row0 + r) / P.g;
          const bool token = r < nrows && sees(P, g.b, i, i);  // else it has seen nothing
          s_m[warp * ROWS + r] = token ? m[t][x] - kLift<T, 0> : -INFINITY;  // what o and l are relative to
          s_l[warp * ROWS + r] = token ? l[t][x] : 0.0f;
        }
      }
    const bool whole = g.s0 == 0 && g.s1 == g.steps;
    // a unit that starts in this block and goes on goes to the second slot
    float* part = whole ? nullptr : slot_of(P, 2 * blockIdx.x + (g.s0 == 0 ? 1u : 0u));
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
      for (uint32_t d0 = 0; d0 < DP; d0 += LDJ) {
#pragma unroll
        for (uint32_t d = 0; d < LDJ / 8; d++)
#pragma unroll
          for (int x = 0; x < 2; x++)
            *reinterpret_cast<float2*>(s_join + (warp * 16 + oct + 8 * x) * LDJ + 8 * d + 2 * quad) =
                make_float2(o[t][d0 / 8 + d][2 * x], o[t][d0 / 8 + d][2 * x + 1]);
        __syncthreads();
        for (uint32_t i = tid; i < 16 * LDJ / 2; i += 32 * kRowWarps) {
          const uint32_t r = i / (LDJ / 2), d = 2 * (i % (LDJ / 2)), rr = 16 * t + r, row = row0 + rr;
          if (rr >= nrows || d0 + d >= P.c.v.D) continue;
          float mm[kRowWarps], top = -INFINITY, sum = 0.0f;
#pragma unroll
          for (uint32_t w = 0; w < kRowWarps; w++) top = fmaxf(top, mm[w] = s_m[w * ROWS + rr]);
          const float base = top == -INFINITY ? 0.0f : top;
          float2 y = make_float2(0.0f, 0.0f);
#pragma unroll
          for (uint32_t w = 0; w < kRowWarps; w++) {
            const float f = exp2_fast(mm[w] - base);
            const float2 v = *reinterpret_cast<const float2*>(s_join + (w * 16 + r) * LDJ + d);
            sum += f * s_l[w * ROWS + rr];
            y.x += f * v.x;
            y.y += f * v.y;
          }
          if (whole) {
            const float inv = 1.0f / sum;
            if (sum == 0.0f) y = make_float2(0.0f, 0.0f);
            else y = make_float2(y.x * inv, y.y * inv);
            T* out = static_cast<T*>(P.a.d_out) + int64_t(g.b) * P.a.o_b + int64_t(row / P.g) * P.a.o_t +
                     int64_t(h * P.g + row % P.g) * P.a.o_h + d0 + d;
            *reinterpret_cast<uint32_t*>(out) = pack2(y.x, y.y, T());
            if (P.lse && d0 + d == 0)
              P.lse[(uint64_t(g.b) * P.a.n + row / P.g) * P.a.hq + h * P.g + row % P.g] = kLn2 * (base + log2f(sum));
          } else {
            *reinterpret_cast<float2*>(part + rr * P.ld_o + d0 + d) = y;
            if (d0 + d == 0) {
              part[P.rows * P.ld_o + 2 * rr] = top;
              part[P.rows * P.ld_o + 2 * rr + 1] = sum;
            }
          }
        }
        __syncthreads();
      }
  } while (next_seg(P, g));
  asm volatile("cp.async.wait_all;" ::: "memory");
}

}  // namespace kv
}  // namespace voom
