// Cache attention of many rows per key head: tcgen05.
//
// Tiles of 128 rows times `KT` keys.  S = Q K^T goes to TMEM; a warpgroup of
// softmax threads, one row each, turns it into probabilities, which go back
// to TMEM over S as the A operand of O += P V.  Roles in a block: one or two
// softmax warpgroups, four warps that load tiles, one thread that issues the
// matrix instructions.  Two S/P/O sets ("slots") keep the tensor cores busy
// with one while the softmax works on the other:
//   kPair       the slots are two tiles of rows that share every tile of keys;
//   kAlternate  one tile of rows, the slots take every other tile of keys and
//               are joined at the end;
//   kSingle     (heads of 256: O fills half of TMEM) one tile of rows, one O,
//               the slots are two S buffers.
// A row's maximum is raised only when it grows by more than 2^8: O is rescaled
// then, which is rare; until then probabilities are at most 2^8, which 16-bit
// types hold as precisely as 1 (kLift: what that leaves of FP16's range).
//
// Bound by the softmax beside the products (kPair: both take about 2000 cycles
// of the 4200 that a tile of keys takes), kSingle by the tiles' way from L2 and
// the operands' from shared memory.  Measured: 64 tokens x 32 heads of 128
// over up to 16384 positions, 8 requests: 109 us a call, 83 % of it here, 710
// TFLOP/s; 1023 tokens x 16 heads of 256 over 6145: 171 us, 87 % of it here, 750
// TFLOP/s (46 % of a large matrix product's rate); the tensor pipe is busy for a
// third of the time in both.  kPair and kAlternate
// compile to the 128 registers a thread that the split below starts from, and spill
// about 290 bytes; a softmax thread holds a row of S, 128 registers of its 192.
//
// Scored, the steps go from the newest keys to the oldest, so that a row whose bias falls
// with distance meets its largest scores first.  Measured: 1000 tokens x 32 heads of
// 128 over 8192 positions, capped, biased, window of 6000: 226 us a call, 203 of it
// here (485 TFLOP/s), the tensor pipe busy 24 % of the time.  A tile takes about 7400
// cycles: 2000 for the cap's polynomial, the bias and the maximum, 1600 for the
// exponentials, 600 for S out of TMEM, the rest waits for products and barriers.  Spilled: 384-440 bytes.  Slower
// here: two threads to a row (256 us, S read twice), probabilities kept in registers
// against a guessed maximum (300-346), other register splits (no change).
#pragma once

#include "kv_attn.cuh"
#include "kv_modes.cuh"
#include "tcgen05.cuh"

namespace voom {
namespace kv {

template <int DP, int MODE>
struct Tc {
  static constexpr uint32_t KT = MODE == kSingle ? 64 : 128;       // keys of a tile
  static constexpr uint32_t ROWS = MODE == kPair ? 256 : 128;      // rows of a unit
  static constexpr uint32_t WGS = MODE == kSingle ? 1 : 2;         // softmax warpgroups
  // two softmax warpgroups: a full fourth one with the issuing warp, so that
  // registers can be moved to the softmax, whose threads hold a row of S
  static constexpr uint32_t THREADS = WGS * 128 + 128 + (WGS == 2 ? 128 : 32);
  static constexpr uint32_t MORE = 192, LESS = 64;                 // 2 x 128 x 192 + 2 x 128 x 64 = 512 x 128
  static constexpr uint32_t TILE = KT * DP * 2;                    // bytes of a tile of keys or values
  static constexpr uint32_t QTILE = 128 * DP * 2;
  static constexpr uint32_t Q = (ROWS / 128) * QTILE;
  static constexpr uint32_t RING = (224 * 1024 - Q) / TILE;        // tiles in flight or in use
  static constexpr uint32_t O_COL = 256;                           // TMEM columns: S at 0 and S_COL, then O
  static constexpr uint32_t S_COL = 128;
};

struct TcShared {
  uint64_t full[16], empty[16];  // ring of tiles
  uint64_t q_full, q_empty, s_full[2], p_ready[2], o_full[2], pv_done, drained, joined;
  uint32_t tmem, failed;
  uint32_t odd;         // a new token's value was not finite and taken out of its tile
  uint32_t pad;
  float2 ml[2][128];    // kAlternate: the slots' maxima and sums
};

template <int DP, int MODE>
constexpr uint32_t tc_smem() {
  constexpr uint32_t n = Tc<DP, MODE>::Q + Tc<DP, MODE>::RING * Tc<DP, MODE>::TILE + uint32_t(sizeof(TcShared));
  static_assert(n <= 227 * 1024 && Tc<DP, MODE>::RING <= 16 && Tc<DP, MODE>::RING >= 3, "shared memory of a block");
  return n;
}

// Values of new tokens that are not finite were taken out of their tiles (a
// probability of 0 must not meet them); this adds them back for a row that
// sees them, one at a time: y[0..32) are the row's sums of values col ..
template <typename T, bool SCORED>
__device__ __forceinline__ void odd_fix(const Attn& P, const Seg& g, uint32_t row, float m2, uint32_t col, float* y) {
  const uint32_t cs = cache_steps<SCORED>(P, g.len), i = row / P.g;
  const T* q = static_cast<const T*>(P.a.d_q) + int64_t(g.b) * P.a.q_b + int64_t(i) * P.a.q_t +
               int64_t(g.h * P.g + row % P.g) * P.a.q_h;
  // one key's part; `ahead`: from the row to it
  auto add = [&](const T* k, const T* v, int32_t ahead) {
    float p = -1.0f;
    for (uint32_t c = 0; c < 32 && col + c < P.c.v.D; c += 8) {
      if (!odd_values<T>(*reinterpret_cast<const uint4*>(v + col + c))) continue;
      if (p < 0.0f) {
        float z = 0.0f;
        #pragma unroll 1
        for (uint32_t d = 0; d < P.c.v.D; d++) z += elem<T>(q[d]) * elem<T>(k[d]);
        if constexpr (SCORED) p = exp2_fast(scored(P, z, slope2_of(P, g.h * P.g + row % P.g), float(ahead)) - m2);
        else p = exp2_fast(z * P.scale2 - m2);
      }
      for (uint32_t e = 0; e < 8; e++) y[c + e] += p * elem<T>(v[col + c + e]);
    }
  };
  const int32_t behind = SCORED ? depth_of(P, g.b, i) : 0;
  if constexpr (SCORED) {  // cached positions that the window's edge passes
    const uint32_t w0 = first_tile<SCORED>(P, g.len);
    const uint32_t edge = ceil_div(window_all(P, g.len), P.keys) * P.keys;  // (whole tiles are looked through)
    const uint32_t s0 = max(window_none<SCORED>(P, g.len), (w0 + g.s0) * P.keys), s1 = min(min(edge, g.len), (w0 + g.s1) * P.keys);
    if (P.a.n > 1)
      for (uint32_t s = s0; s < s1; s++) {
        const int32_t ahead = int32_t(s) - int32_t(g.len) - behind;
        int64_t ko, vo;
        if (in_window(P, ahead) && P.c.row_at(g.b, g.h, s, ko, vo))
          add(static_cast<const T*>(P.c.v.d_k) + ko, static_cast<const T*>(P.c.v.d_v) + vo, ahead);
      }
  }
  const uint32_t j0 = (max(g.s0, cs) - cs) * P.keys, j1 = g.s1 > cs ? min(P.a.n, (g.s1 - cs) * P.keys) : 0u;
  for (uint32_t j = j0; j < j1; j++) {
    if (!sees(P, g.b, i, j)) continue;
    const int32_t ahead = SCORED ? depth_of(P, g.b, j) - behind : 0;
    if (SCORED && !in_window(P, ahead)) continue;
    add(static_cast<const T*>(P.a.d_kn) + int64_t(g.b) * P.a.kn_b + int64_t(j) * P.a.kn_t + int64_t(g.h) * P.a.kn_h,
        static_cast<const T*>(P.a.d_vn) + int64_t(g.b) * P.a.vn_b + int64_t(j) * P.a.vn_t + int64_t(g.h) * P.a.vn_h, ahead);
  }
}

// One of four warps' part (128 threads) of bringing a tile of keys or values to
// shared memory; its barrier gets 128 arrivals.  A tile of cached positions
// that are all valid and seen comes by TMA, one box for each run of positions in a page:
// the lanes of the first warp find the pages.  Others (the end of a cache, new
// tokens, caches that TMA cannot read) are gathered through cp.async; their
// barrier hears of the copies as they land, and the issuing thread fences them
// for the tensor cores.  With `hold` nothing is announced: the caller waits
// for the copies, and arrives; true then.
template <typename T, int DP, int KT, bool SCORED>
__device__ __forceinline__ bool load_tile_sw128(const Attn& P, const Seg& g, uint32_t step, uint32_t cs, bool is_v, uint32_t pw,
                                                uint32_t lane, uint32_t dst, uint32_t full, bool hold) {
  constexpr uint32_t CH = DP / 8, RW = KT / 4;
  const bool fresh = step >= cs;
  const uint32_t p0 = (first_tile<SCORED>(P, g.len) + step) * KT;  // of a cached tile: its first position
  const uint32_t none = window_none<SCORED>(P, g.len);  // what no row sees comes as zeros
  if (P.box && !fresh && p0 + KT <= g.len && p0 >= none && !hold) {
    if (pw == 0) {
      if (lane == 0) tc::mbar_arrive_expect(full, KT * DP * 2);
      else tc::mbar_arrive(full);
      __syncwarp();
      if (lane < KT / P.box) {
        const uint32_t s = p0 + lane * P.box, pg = P.c.page_of(s);
        const int32_t w = P.c.page_box(g.b, pg);
        const uint32_t y = P.c.v.d_table ? s - pg * P.c.v.page : s;
        const void* map = is_v ? &P.v_map : &P.k_map;
#pragma unroll
        for (uint32_t x = 0; x < DP; x += 64)
          tc::tma_load4(dst + (x / 64) * (KT * 128u) + lane * P.box * 128u, map, full, int32_t(x), int32_t(y), int32_t(g.h), w);
      }
    } else {
      tc::mbar_arrive(full);
    }
    return false;
  }
  uint64_t a = 0;
  if (lane < RW) {
    const uint32_t r = pw * RW + lane;
    if (!fresh) {
      const uint32_t s = p0 + r;
      int64_t ko, vo;
      if (s >= none && s < g.len && P.c.row_at(g.b, g.h, s, ko, vo))
        a = is_v ? reinterpret_cast<uint64_t>(static_cast<const T*>(P.c.v.d_v) + vo)
                 : reinterpret_cast<uint64_t>(static_cast<const T*>(P.c.v.d_k) + ko);
    } else {
      const uint32_t s = (step - cs) * KT + r;
      if (s < P.a.n && sees(P, g.b, s, s))
        a = is_v ? reinterpret_cast<uint64_t>(static_cast<const T*>(P.a.d_vn) + int64_t(g.b) * P.a.vn_b + int64_t(s) * P.a.vn_t +
                                              int64_t(g.h) * P.a.vn_h)
                 : reinterpret_cast<uint64_t>(static_cast<const T*>(P.a.d_kn) + int64_t(g.b) * P.a.kn_b + int64_t(s) * P.a.kn_t +
                                              int64_t(g.h) * P.a.kn_h);
    }
  }
#pragma unroll
  for (uint32_t k = 0; k < RW * CH / 32; k++) {
    const uint32_t id = k * 32 + lane, r = id / CH, c = id % CH;
    const uint64_t y = __shfl_sync(0xFFFFFFFFu, a, r);
    const bool in = y && c * 8 < P.c.v.D;
    cp16(dst + sw128(pw * RW + r, c, KT), in ? reinterpret_cast<const void*>(y + 16 * c) : P.c.v.d_k, in);
  }
  if (!hold) tc::mbar_arrive_copies(full);
  return hold;
}

template <typename T, int DP, int KT, bool SCORED>
__device__ __forceinline__ void load_keys(const Attn& P, const Seg& g, uint32_t step, uint32_t cs, uint32_t pw, uint32_t lane,
                                          uint32_t dst, uint32_t full) {
  load_tile_sw128<T, DP, KT, SCORED>(P, g, step, cs, false, pw, lane, dst, full, false);
}

template <typename T, int DP, int MODE, bool SCORED>
__global__ void __launch_bounds__(Tc<DP, MODE>::THREADS, 1) attn_tc(const __grid_constant__ Attn P) {
  using C = Tc<DP, MODE>;
  constexpr uint32_t KT = C::KT, ROWS = C::ROWS, CH = DP / 8, RING = C::RING;
  extern __shared__ __align__(1024) uint8_t smem[];
  TcShared& sh = *reinterpret_cast<TcShared*>(smem + C::Q + RING * C::TILE);
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  const uint32_t q_s = smem_addr(smem), ring_s = q_s + C::Q;
  constexpr uint32_t LOAD_WARP = C::WGS * 4, MMA_WARP = LOAD_WARP + 4;
  auto bar = [](const uint64_t& b) { return smem_addr(&b); };
  // a whole warp's bounded wait: all lanes go on, or none
  auto warp_wait = [&](const uint64_t& b, uint32_t parity) {
    return __all_sync(0xFFFFFFFFu, tc::mbar_wait(smem_addr(&b), parity)) != 0;
  };

  Seg g;
  const bool any = first_seg<SCORED>(P, blockIdx.x, g) && (q_s & 1023u) == 0;
  if (tid == 0) {
    for (uint32_t i = 0; i < RING; i++) {
      tc::mbar_init(bar(sh.full[i]), 128);
      tc::mbar_init(bar(sh.empty[i]), 1);
    }
    tc::mbar_init(bar(sh.q_full), 128);
    tc::mbar_init(bar(sh.q_empty), 1);
    for (int i = 0; i < 2; i++) {
      tc::mbar_init(bar(sh.s_full[i]), 1);
      tc::mbar_init(bar(sh.p_ready[i]), 128);
      tc::mbar_init(bar(sh.o_full[i]), 1);
    }
    tc::mbar_init(bar(sh.pv_done), 1);
    tc::mbar_init(bar(sh.drained), 1);
    tc::mbar_init(bar(sh.joined), 256);
    sh.failed = (q_s & 1023u) != 0;
    sh.odd = 0;
  }
  if (warp == MMA_WARP) tc::tmem_alloc(bar(*reinterpret_cast<uint64_t*>(&sh.tmem)), 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = sh.tmem;
  if (any && warp >= LOAD_WARP && warp < MMA_WARP) {
    // ------------------------------------------------------------- loaders
    if (C::WGS == 2) tc::regs_less<C::LESS>();
    constexpr uint32_t RW = KT / 4;  // rows of a tile to a warp
    const uint32_t pw = warp - LOAD_WARP;
    uint32_t it = 0, nq = 0;  // tiles and query tiles asked for
    bool ok = true;
    // New tokens' values are looked through first: those that are not finite
    // are taken out, whatever probability they meet.
    auto look_through = [&](uint32_t place) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      bool found = false;
      for (uint32_t k = 0; k < RW * CH / 32; k++) {
        const uint32_t id = k * 32 + lane, r = pw * RW + id / CH;
        uint4* at = reinterpret_cast<uint4*>(smem + C::Q + place * C::TILE + sw128(r, id % CH, KT));
        if (odd_values<T>(*at)) {
          *at = make_uint4(0, 0, 0, 0);
          found = true;
        }
      }
      if (found) sh.odd = 1;
    };
    do {
      const uint32_t row0 = g.m * ROWS, cs = cache_steps<SCORED>(P, g.len), n = g.s1 - g.s0;
      // tiles of values below it are looked through, as those of the new tokens are
      const uint32_t edge = SCORED && P.a.n > 1 ? window_all(P, g.len) : 0u, w0 = first_tile<SCORED>(P, g.len);
      if (nq) {  // the last segment's products of the queries must be done
        if (!(ok = warp_wait(sh.q_empty, (nq - 1) & 1u))) break;
      }
#pragma unroll 1
      for (uint32_t t = 0; t < ROWS / 128; t++) {
        const uint32_t row = row0 + t * 128 + pw * 32 + lane, i = row / P.g;
        uint64_t a = 0;
        if (row < P.R && sees(P, g.b, i, i))
          a = reinterpret_cast<uint64_t>(static_cast<const T*>(P.a.d_q) + int64_t(g.b) * P.a.q_b + int64_t(i) * P.a.q_t +
                                         int64_t(g.h * P.g + row % P.g) * P.a.q_h);
#pragma unroll 4
        for (uint32_t k = 0; k < CH; k++) {
          const uint32_t id = k * 32 + lane, r = id / CH, c = id % CH;
          const uint64_t x = __shfl_sync(0xFFFFFFFFu, a, r);
          const bool in = x && c * 8 < P.c.v.D;
          cp16(q_s + t * C::QTILE + sw128(pw * 32 + r, c, 128), in ? reinterpret_cast<const void*>(x + 16 * c) : P.c.v.d_k, in);
        }
      }
      nq++;
      tc::mbar_arrive_copies(bar(sh.q_full));
      for (uint32_t x = 0; x < 2 * n; x++) {
        // order of use: K0 V0 K1 V1 .. for kPair, K0 K1 V0 K2 V1 .. else
        bool is_v;
        uint32_t j;
        if (MODE == kPair) {
          is_v = x & 1u;
          j = x >> 1;
        } else {
          is_v = x == 2 * n - 1 || (x >= 2 && !(x & 1u));
          j = is_v ? (x == 2 * n - 1 ? n - 1 : (x - 2) >> 1) : (x + 1) >> 1;
        }
        const uint32_t step = SCORED ? g.s1 - 1 - j : g.s0 + j, place = it % RING;
        if (it >= RING && !(ok = warp_wait(sh.empty[place], (it / RING - 1) & 1u))) break;
        it++;
        if (load_tile_sw128<T, DP, KT, SCORED>(P, g, step, cs, is_v, pw, lane, ring_s + place * C::TILE, bar(sh.full[place]),
                                           is_v && (step >= cs || (SCORED && (w0 + step) * KT < edge)))) {
          look_through(place);
          tc::mbar_arrive(bar(sh.full[place]));
        }
      }
    } while (ok && next_seg<SCORED>(P, g));
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (!ok) sh.failed = 1;
  } else if (any && warp >= MMA_WARP) {
    // ------------------------------------------------ the tensor cores' orders
    if (C::WGS == 2) tc::regs_less<C::LESS>();
    if (warp == MMA_WARP) {
    constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t base = (1u << 4) | (fmt << 7) | (fmt << 10) | ((128u >> 4) << 24);
    constexpr uint32_t id_qk = base | ((KT >> 3) << 17), id_pv = base | ((uint32_t(DP) >> 3) << 17) | (1u << 16);
    uint32_t it = 0, nq = 0, np[2] = {0, 0};  // tiles, query tiles and probabilities used so far
    bool ok = true;
    const bool one = tc::elect_one();  // the whole warp goes along; one lane issues
    const uint32_t tm = tc::uniform(tmem), q_lo = (q_s >> 4) | (1u << 16), ring_lo = (ring_s >> 4);
    auto wait = [&](const uint64_t& b, uint32_t parity) {
      if (ok) ok = warp_wait(b, parity);
      tc::tc_fence_after();
    };
    auto wait_tile = [&](uint32_t i) {
      wait(sh.full[i % RING], (i / RING) & 1u);
      tc::fence_async_smem();  // what the loaders copied, for the tensor cores
    };
    auto commit = [&](const uint64_t& b) {
      if (one) tc::umma_commit(bar(b));
    };
    auto tile_at = [&](uint32_t i) { return ring_lo + (i % RING) * (C::TILE >> 4); };  // in 16-byte units
    auto qk = [&](uint32_t slot, uint32_t qt, uint32_t k_at) {
      const uint32_t a = q_lo + qt * (C::QTILE >> 4), b = k_at | (1u << 16), d = tm + slot * C::S_COL;
      if (one) {
#pragma unroll
        for (uint32_t k = 0; k < DP / 16; k++)
          tc::umma_bf16(d, tc::umma_desc_at(a + (k / 4) * 1024u + (k % 4) * 2u, tc::kDescHiSw128),
                        tc::umma_desc_at(b + (k / 4) * (KT * 8u) + (k % 4) * 2u, tc::kDescHiSw128), id_qk, k > 0);
        tc::umma_commit(bar(sh.s_full[slot]));
      }
    };
    auto pv = [&](uint32_t slot, uint32_t o_col, uint32_t v_at, bool first) {
      wait(sh.p_ready[slot], np[slot]++ & 1u);
      if (!ok) return;
      const uint32_t b = v_at | (KT * 8u) << 16, d = tm + o_col, a = tm + slot * C::S_COL;
      if (one) {
#pragma unroll
        for (uint32_t k = 0; k < KT / 16; k++)
          tc::umma_f16_ts(d, a + k * 8u, tc::umma_desc_at(b + k * 128u, tc::kDescHiSw128), id_pv, !first || k > 0);
      }
    };
    do {
      const uint32_t n = tc::uniform(g.s1 - g.s0), i0 = it;
      wait(sh.q_full, nq++ & 1u);
      tc::fence_async_smem();
      if (MODE == kPair) {
        wait_tile(i0);
        if (!ok) break;
        qk(0, 0, tile_at(i0));
        qk(1, 1, tile_at(i0));
        commit(sh.empty[i0 % RING]);
        if (n == 1) commit(sh.q_empty);
        for (uint32_t j = 0; j < n && ok; j++) {
          const uint32_t v = i0 + 2 * j + 1, k = v + 1;
          for (uint32_t t = 0; t < 2; t++) {
            if (t == 0) wait_tile(v);
            pv(t, C::O_COL + t * DP, tile_at(v), j == 0);
            if (!ok) break;
            if (t == 1) commit(sh.empty[v % RING]);
            if (j + 1 < n) {
              if (t == 0) wait_tile(k);
              if (!ok) break;
              qk(t, t, tile_at(k));
              if (t == 1) {
                commit(sh.empty[k % RING]);
                if (j + 2 == n) commit(sh.q_empty);
              }
            } else {
              commit(sh.o_full[t]);
            }
          }
        }
      } else {
        // tile i of keys is item 2 i - 1 (the first: 0), of values 2 i + 2 (the last: 2 n - 1)
        for (uint32_t i = 0; i < 2 && i < n; i++) {
          const uint32_t k = i0 + i;
          wait_tile(k);
          if (!ok) break;
          qk(i, 0, tile_at(k));
          commit(sh.empty[k % RING]);
          if (i + 1 == n) commit(sh.q_empty);
        }
        for (uint32_t i = 0; i < n && ok; i++) {
          const uint32_t t = i & 1u, v = i0 + (i + 1 == n ? 2 * n - 1 : 2 * i + 2);
          wait_tile(v);
          pv(t, C::O_COL + (MODE == kAlternate ? t * DP : 0u), tile_at(v), MODE == kAlternate ? i < 2 : i == 0);
          if (!ok) break;
          commit(sh.empty[v % RING]);
          if (MODE == kSingle) commit(sh.pv_done);
          if (i + 2 < n) {
            const uint32_t k = i0 + 2 * (i + 2) - 1;
            wait_tile(k);
            if (!ok) break;
            qk(t, 0, tile_at(k));
            commit(sh.empty[k % RING]);
            if (i + 3 == n) commit(sh.q_empty);
          }
          if (MODE == kAlternate ? i + 2 >= n : i + 1 == n) commit(sh.o_full[MODE == kAlternate ? t : 0]);
        }
      }
      it += 2 * n;
    } while (ok && next_seg<SCORED>(P, g));
    commit(sh.drained);  // nothing may be under way when TMEM is given back
    if (!warp_wait(sh.drained, 0)) ok = false;
    if (!ok) sh.failed = 1;
    }
  } else if (any && warp < LOAD_WARP) {
    // ------------------------------------------------------------- softmax
    if (C::WGS == 2) tc::regs_more<C::MORE>();
    const uint32_t w = warp >> 2, tr = tid & 127u, lanes = (warp & 3u) << 21;  // TMEM lane 32 * (warp % 4)
    uint32_t ns[2] = {0, 0}, no[2] = {0, 0}, done = 0, nj = 0;  // S tiles, finished outputs, steps, joins so far
    bool ok = true;
    do {
      const uint32_t row = g.m * ROWS + (MODE == kPair ? w * 128 : 0) + tr, tok = row / P.g, cs = cache_steps<SCORED>(P, g.len);
      const uint32_t n = g.s1 - g.s0, w0 = first_tile<SCORED>(P, g.len);
      float m = -INFINITY, l = 0.0f, rest = 0.0f;  // l + rest: the denominator
      const float to_log2 = SCORED ? 1.0f : P.scale2;
      const float slope2 = SCORED ? slope2_of(P, g.h * P.g + row % P.g) : 0.0f;
      const int32_t behind = SCORED ? depth_of(P, g.b, tok) : 0;  // how far behind the cache the row stands
      for (uint32_t i = MODE == kAlternate ? w : 0; i < n; i += MODE == kAlternate ? 2 : 1) {
        // scored: the newest keys first, whose biases are the largest, so that the maximum is not raised tile by tile
        const uint32_t slot = MODE == kSingle ? i & 1u : w, step = SCORED ? g.s1 - 1 - i : g.s0 + i;
        const uint32_t o_col = C::O_COL + (MODE == kSingle ? 0u : w * DP);
        if (!(ok = warp_wait(sh.s_full[slot], ns[slot]++ & 1u))) break;
        tc::tc_fence_after();
        const uint32_t s_at = tmem + lanes + slot * C::S_COL;
        const uint32_t p0 = (w0 + step) * KT;  // of a cached tile: its first position
        const bool fresh = step >= cs;
        // of the tile's first key, in a cached tile or a chain
        const int32_t ahead = (fresh ? int32_t((step - cs) * KT) : int32_t(p0) - int32_t(g.len)) - behind;
        const bool masked = fresh || p0 + KT > g.len || (SCORED && P.a.window && -int64_t(ahead) >= int64_t(P.a.window));
        uint32_t see[KT / 32];
        if (masked) {
#pragma unroll
          for (uint32_t c = 0; c < KT / 32; c++) {
            if (fresh) {
              see[c] = sees32(P, g.b, tok, (step - cs) * KT + 32 * c);
            } else {
              const uint32_t valid = g.len - p0;
              see[c] = valid >= 32 * c + 32 ? 0xFFFFFFFFu : valid <= 32 * c ? 0u : (1u << (valid - 32 * c)) - 1u;
            }
            if constexpr (SCORED) {
              if (!fresh || !P.a.d_mask) {
                see[c] &= window32(P, ahead + int32_t(32 * c));
              } else if (P.a.window) {  // a tree's tokens stand at their depths
                for (uint32_t left = see[c]; left; left &= left - 1) {
                  const uint32_t e = __ffs(left) - 1;
                  if (int64_t(behind) - depth_of(P, g.b, (step - cs) * KT + 32 * c + e) >= int64_t(P.a.window)) see[c] &= ~(1u << e);
                }
              }
            }
          }
        }
        uint32_t s[KT / 32][32];
#pragma unroll
        for (uint32_t c = 0; c < KT / 32; c++) tc::tmem_ld32(s_at + 32 * c, s[c]);
        tc::tmem_wait_ld();
#pragma unroll
        for (uint32_t c = 0; c < KT / 32; c++) tc::tmem_hold(s[c]);
        if constexpr (SCORED) {
          auto pair = [&](uint32_t c, int e) { return make2(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1])); };
          auto put = [&](uint32_t c, int e, F2 v) {
            float x, y;
            take2(v, x, y);
            s[c][e] = __float_as_uint(x);
            s[c][e + 1] = __float_as_uint(y);
          };
          auto all = [&](auto kind, auto biased) {
            const F2 by = make2(2.0f * slope2, 2.0f * slope2);
            const float from = slope2 * float(ahead);
#pragma unroll
            for (uint32_t c = 0; c < KT / 32; c++)
#pragma unroll
              for (int q = 0; q < 32; q += 8) {  // a bias by steps: four of them from one that is made anew
                const float first = fmaf(slope2, float(32 * c + q), from);
                F2 bias = decltype(biased)::value ? make2(first, first + slope2) : make2(0.0f, 0.0f);
#pragma unroll
                for (int e = q; e < q + 8; e += 2) {
                  put(c, e, scored2<decltype(kind)::value>(P, pair(c, e), bias));
                  if (decltype(biased)::value) bias = add2(bias, by);
                }
              }
          };
          auto with_bias = [&](auto kind) {
            if (P.a.d_slopes) all(kind, std::true_type());
            else all(kind, std::false_type());
          };
          if (fresh && P.a.d_mask && P.a.d_slopes) {  // a tree's tokens stand at their depths
#pragma unroll
            for (uint32_t c = 0; c < KT / 32; c++)
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const uint32_t j = (step - cs) * KT + 32 * c + e;
                put(c, e, scored2(P, pair(c, e), make2(slope2 * float(depth_of(P, g.b, j) - behind),
                                                       slope2 * float(depth_of(P, g.b, j + 1) - behind))));
              }
          } else if (P.cap_in == 0.0f) {
            with_bias(Kind<kPlain>());
          } else {
            float most[2] = {0.0f, 0.0f};
#pragma unroll
            for (uint32_t c = 0; c < KT / 32; c++)
#pragma unroll
              for (int e = 0; e < 32; e += 2)
                most[e >> 1 & 1] = max3(most[e >> 1 & 1], fabsf(__uint_as_float(s[c][e])), fabsf(__uint_as_float(s[c][e + 1])));
            const float m1 = fmaxf(most[0], most[1]);
            if (__any_sync(0xFFFFFFFFu, m1 > P.cap_small)) with_bias(Kind<kAny>());
            else with_bias(Kind<kSmall>());
          }
        }
        if (masked) {
#pragma unroll
          for (uint32_t c = 0; c < KT / 32; c++)
#pragma unroll
            for (int e = 0; e < 32; e++) s[c][e] = see[c] >> e & 1u ? s[c][e] : 0xFF800000u;
        }
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (uint32_t c = 0; c < KT / 32; c++)
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            tops[(e >> 1) & 3] = max3(tops[(e >> 1) & 3], __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const bool grow = m != -INFINITY && (top - m) * to_log2 > 8.0f;
        if (__any_sync(0xFFFFFFFFu, grow)) {
          const float f = grow ? exp2_fast((m - top) * to_log2) : 1.0f;
          if (MODE == kSingle && done) {
            if (!(ok = warp_wait(sh.pv_done, (done - 1) & 1u))) break;
            tc::tc_fence_after();
          }
#pragma unroll 1
          for (uint32_t c = 0; c < DP; c += 32) {
            uint32_t o[32];
            tc::tmem_ld32(tmem + lanes + o_col + c, o);
            tc::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tc::tmem_st32(tmem + lanes + o_col + c, o);
          }
          l *= f;
          rest *= f;
          if (grow) m = top;
        }
        if (m == -INFINITY) m = top;
        const float base = m == -INFINITY ? 0.0f : m * to_log2 - kLift<T, 8>;
        const F2 sc = make2(to_log2, to_log2), nb = make2(-base, -base);
        F2 sum[2] = {make2(0.0f, 0.0f), make2(0.0f, 0.0f)};
#pragma unroll
        for (uint32_t c = 0; c < KT / 32; c++) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 16; e++) {
            float x, y;
            take2(fma2(make2(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1])), sc, nb), x, y);
            x = exp2_fast(x);
            y = exp2_fast(y);
            sum[e & 1] = add2(sum[e & 1], make2(x, y));
            p[e] = pack2(x, y, T());
          }
          tc::tmem_st16(s_at + 16 * c, p);
        }
        float s0, s1, s2, s3;
        take2(sum[0], s0, s1);
        take2(sum[1], s2, s3);
        add_kept(l, rest, (s0 + s1) + (s2 + s3));
        tc::tmem_wait_st();
        tc::tc_fence_before();
        tc::mbar_arrive(bar(sh.p_ready[slot]));
        done++;
      }
      if (!ok) break;
      // the segment's sums
      l += rest;
      float m2 = m == -INFINITY ? -INFINITY : m * to_log2 - kLift<T, 8>, f0 = 1.0f, f1 = 0.0f;  // what O and l are relative to
      uint32_t c0 = 0, c1 = DP;
      if (MODE == kAlternate) {
        sh.ml[w][tr] = make_float2(m2, l);
        tc::mbar_arrive(bar(sh.joined));
        if (!(ok = warp_wait(sh.joined, nj++ & 1u))) break;
        const float2 a = sh.ml[0][tr], b = sh.ml[1][tr];
        m2 = fmaxf(a.x, b.x);
        const float base = m2 == -INFINITY ? 0.0f : m2;
        f0 = exp2_fast(a.x - base);
        f1 = exp2_fast(b.x - base);
        l = f0 * a.y + f1 * b.y;
        c0 = w * (DP / 2);
        c1 = c0 + DP / 2;
        ok = warp_wait(sh.o_full[0], no[0]++ & 1u);
        if (n > 1) ok = warp_wait(sh.o_full[1], no[1]++ & 1u) && ok;
      } else {
        const uint32_t x = MODE == kPair ? w : 0;
        ok = warp_wait(sh.o_full[x], no[x]++ & 1u);
      }
      if (!ok) break;
      tc::tc_fence_after();
      const bool whole = g.s0 == 0 && g.s1 == g.steps, in = row < P.R;
      const bool alive = in && sees(P, g.b, tok, tok);
      if (!alive) {  // it has seen nothing
        m2 = -INFINITY;
        l = 0.0f;
      }
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const uint32_t pr = (MODE == kPair ? w * 128 : 0) + tr, head = g.h * P.g + row % P.g;
      float* part = whole ? nullptr : slot_of(P, 2 * blockIdx.x + (g.s0 == 0 ? 1u : 0u));
      T* out = static_cast<T*>(P.a.d_out) + int64_t(g.b) * P.a.o_b + int64_t(tok) * P.a.o_t + int64_t(head) * P.a.o_h;
      const bool odd = *reinterpret_cast<volatile uint32_t*>(&sh.odd) != 0;
#pragma unroll 1
      for (uint32_t c = c0; c < c1; c += 32) {
        uint32_t o[32];
        float y[32];
        tc::tmem_ld32(tmem + lanes + C::O_COL + (MODE == kPair ? w * DP : 0u) + c, o);
        tc::tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e++) y[e] = __uint_as_float(o[e]);
        if (MODE == kAlternate && n > 1) {
          tc::tmem_ld32(tmem + lanes + C::O_COL + DP + c, o);
          tc::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e++) y[e] = f0 * y[e] + f1 * __uint_as_float(o[e]);
        }
        if (odd && alive) {
          float z[32];
#pragma unroll
          for (int e = 0; e < 32; e++) z[e] = y[e];
          odd_fix<T, SCORED>(P, g, row, m2, c, z);
#pragma unroll
          for (int e = 0; e < 32; e++) y[e] = z[e];
        }
        if (!in) continue;
        if (whole) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (l != 0.0f)
              x = make_uint4(pack2(y[e] * inv, y[e + 1] * inv, T()), pack2(y[e + 2] * inv, y[e + 3] * inv, T()),
                             pack2(y[e + 4] * inv, y[e + 5] * inv, T()), pack2(y[e + 6] * inv, y[e + 7] * inv, T()));
            if (c + e < P.c.v.D) *reinterpret_cast<uint4*>(out + c + e) = x;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<float4*>(part + pr * P.ld_o + c + e) = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
        }
      }
      if (in && c0 == 0) {
        if (!whole) *reinterpret_cast<float2*>(part + ROWS * P.ld_o + 2 * pr) = make_float2(m2, l);
        else if (P.lse) P.lse[(uint64_t(g.b) * P.a.n + tok) * P.a.hq + head] = kLn2 * ((m2 == -INFINITY ? 0.0f : m2) + log2f(l));
      }
      tc::tc_fence_before();
      if (MODE == kAlternate) {  // both halves of both slots are read
        tc::mbar_arrive(bar(sh.joined));
        if (!(ok = warp_wait(sh.joined, nj++ & 1u))) break;
      }
    } while (next_seg<SCORED>(P, g));
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
