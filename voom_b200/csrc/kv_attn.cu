// Attention of drafted tokens over a KV cache, its weight sums, and the tree masks.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstddef>
#include <cstring>
#include <initializer_list>
#include <type_traits>

#include "kv_attn.cuh"
#include "kv_modes.cuh"
#include "rows.h"

namespace {

using std::max;
using std::min;
using voom::kv::Attn;

constexpr uint32_t kMaxTree = 1024;

// --------------------------------------------------------------- tree masks
// One CTA per tree, a warp per row, which walks from its token to the root.
__global__ void __launch_bounds__(256) tree_mask(const int32_t* __restrict__ parents, uint32_t n, uint32_t* mask,
                                                 int32_t* depth) {
  __shared__ int32_t s_up[kMaxTree];
  const uint32_t b = blockIdx.x, words = (n + 31) / 32;
  parents += uint64_t(b) * n;
  uint32_t* m = mask + uint64_t(b) * n * words;
  for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
    const int32_t p = parents[i];
    s_up[i] = p >= 0 && p < int32_t(i) && parents[p] != -2 ? p : -1;
  }
  __syncthreads();
  const uint32_t lane = threadIdx.x & 31u;
  for (uint32_t i = threadIdx.x >> 5; i < n; i += blockDim.x >> 5) {
    const bool none = parents[i] == -2;
    uint32_t w = 0;
    int32_t d = -1;
    if (!none)
      for (int32_t j = int32_t(i); j >= 0; j = s_up[j]) {
        if (uint32_t(j >> 5) == lane) w |= 1u << (j & 31);  // a lane keeps its own word
        d++;
      }
    if (lane < words) m[uint64_t(i) * words + lane] = w;
    if (lane == 0) depth[uint64_t(b) * n + i] = d;
  }
}

// ------------------------------------------------------------------- finish
// Joins the partial sums of units that several blocks shared (blocks below
// n_merge: one per unit and merge_rows of its rows), and adds the rows' weights at each
// position to the running sums (the others: one per key head and kWeightSpan
// positions), from the scores the attention kept and the rows' denominators.
// The partial sums are joined in block order, the rows added in row order, so
// that nothing depends on scheduling.
constexpr uint32_t kWeightSpan = 1024;
constexpr uint32_t kMergeRows = 16;  // at most

// (more blocks than the GPU holds at a time: the latency of one counts for 16 rows, 1000
// tokens x 32 heads 188 us a call against 194; fewer: more of them at work, 26 drafts
// x 32 heads 30 us against 34)
__host__ __device__ __forceinline__ uint32_t merge_rows(const Attn& P) {
  return uint64_t(P.c.v.B) * P.c.v.hk * P.mblocks * P.rows >= 16384u ? kMergeRows : 8u;
}

struct Split {
  uint32_t first, last;  // blocks that hold the unit's partial sums; first > last: none, it is whole
};

__device__ __forceinline__ Split split_of(const Attn& P, uint32_t b, uint32_t h, uint32_t m, uint64_t total, uint64_t before) {
  Split s{1, 0};
  if (!P.ctas) return s;
  const uint32_t len = P.c.length(b), cs = voom::kv::cache_steps(P, len);
  const uint64_t at = before + h * voom::kv::head_steps(P, len) + uint64_t(m) * cs + voom::kv::tails_before(P, m);
  voom::kv::owners(P, total, at, cs + voom::kv::tail_of(P, m), s.first, s.last);
  if (s.first == s.last) s = Split{1, 0};
  return s;
}

__device__ __forceinline__ const float* part_of(const Attn& P, const Split& s, uint32_t c) {
  return voom::kv::slot_of(P, 2 * c + (c == s.first ? 1u : 0u));
}

// Maximum and sum of one row over the partial sums (warp-collective).
__device__ __forceinline__ float2 joined(const Attn& P, const Split& s, uint32_t r) {
  const uint32_t lane = threadIdx.x & 31u;
  float top = -INFINITY, sum = 0.0f;
  for (uint32_t c = s.first + lane; c <= s.last; c += 32) {
    const float2 ml = *reinterpret_cast<const float2*>(part_of(P, s, c) + P.rows * P.ld_o + 2 * r);
    const float t = fmaxf(top, ml.x), base = t == -INFINITY ? 0.0f : t;
    sum = sum * voom::kv::exp2_fast(top - base) + ml.y * voom::kv::exp2_fast(ml.x - base);
    top = t;
  }
  for (int o = 16; o; o >>= 1) {
    const float ot = __shfl_xor_sync(0xFFFFFFFFu, top, o), os = __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    const float t = fmaxf(top, ot), base = t == -INFINITY ? 0.0f : t;
    // both lanes of a pair add the same two terms in the same order
    const bool low = (lane & uint32_t(o)) == 0;
    const float a = (low ? sum : os) * voom::kv::exp2_fast((low ? top : ot) - base);
    const float c = (low ? os : sum) * voom::kv::exp2_fast((low ? ot : top) - base);
    sum = a + c;
    top = t;
  }
  return make_float2(top, sum);
}

template <typename T>
__global__ void __launch_bounds__(256) attn_finish(const __grid_constant__ Attn P, uint32_t n_merge) {
  extern __shared__ float s_row[];  // lse (log2 units) of the key head's rows, then their weights
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  __shared__ Split s_split;
  if (blockIdx.x < n_merge) {
    const uint32_t some = merge_rows(P), groups = (P.rows + some - 1) / some, unit = blockIdx.x / groups, r0 = (blockIdx.x - unit * groups) * some;
    const uint32_t m = unit % P.mblocks, head = unit / P.mblocks, b = head / P.c.v.hk, h = head - b * P.c.v.hk, row0 = m * P.rows;
    if (row0 + r0 >= P.R) return;
    if (warp == 0) {
      const uint64_t total = voom::kv::steps_before(P, P.c.v.B), before = voom::kv::steps_before(P, b);
      if (lane == 0) s_split = split_of(P, b, h, m, total, before);
    }
    __syncthreads();
    const Split s = s_split;
    if (s.first > s.last) return;
    const uint32_t rows = min(min(some, P.rows - r0), P.R - row0 - r0);
    for (uint32_t k = warp; k < rows; k += 8) {
      const float2 ml = joined(P, s, r0 + k);
      if (lane == 0) {
        const uint32_t row = row0 + r0 + k;
        s_row[2 * k] = ml.x == -INFINITY ? 0.0f : ml.x;
        s_row[2 * k + 1] = ml.y == 0.0f ? 0.0f : 1.0f / ml.y;
        if (P.lse)
          P.lse[(uint64_t(b) * P.a.n + row / P.g) * P.a.hq + h * P.g + row % P.g] = voom::kv::kLn2 * (s_row[2 * k] + log2f(ml.y));
      }
    }
    __syncthreads();
    const uint32_t quads = P.ld_o / 4;
    for (uint32_t i = tid; i < rows * quads; i += 256) {
      const uint32_t k = i / quads, d = 4 * (i - k * quads), r = r0 + k, row = row0 + r;
      if (d >= P.c.v.D) continue;
      const float base = s_row[2 * k], inv = s_row[2 * k + 1];
      float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
      for (uint32_t c = s.first; c <= s.last; c++) {
        const float* part = part_of(P, s, c);
        const float f = voom::kv::exp2_fast(part[P.rows * P.ld_o + 2 * r] - base);
        const float4 v = *reinterpret_cast<const float4*>(part + r * P.ld_o + d);
        y.x += f * v.x;
        y.y += f * v.y;
        y.z += f * v.z;
        y.w += f * v.w;
      }
      T* out = static_cast<T*>(P.a.d_out) + int64_t(b) * P.a.o_b + int64_t(row / P.g) * P.a.o_t +
               int64_t(h * P.g + row % P.g) * P.a.o_h + d;
      uint2 x = make_uint2(voom::kv::pack2(y.x * inv, y.y * inv, T()), voom::kv::pack2(y.z * inv, y.w * inv, T()));
      if (inv == 0.0f) x = make_uint2(0u, 0u);  // a row that sees nothing
      *reinterpret_cast<uint2*>(out) = x;
    }
    return;
  }
  const uint32_t spans = (P.score_ld + kWeightSpan - 1) / kWeightSpan, item = blockIdx.x - n_merge;
  const uint32_t head = item / spans, b = head / P.c.v.hk, h = head - b * P.c.v.hk, s0 = (item - head * spans) * kWeightSpan;
  const uint32_t len = P.c.length(b);
  if (s0 >= len && s0 + kWeightSpan <= P.score_new) return;
  float* s_w = s_row + P.R;
  // (the scores are kept for one block of rows only)
  if (P.ctas && warp == 0) {
    const uint64_t total = voom::kv::steps_before(P, P.c.v.B), before = voom::kv::steps_before(P, b);
    if (lane == 0) s_split = split_of(P, b, h, 0, total, before);
  } else if (!P.ctas && tid == 0) {
    s_split = Split{1, 0};
  }
  __syncthreads();
  const Split s = s_split;
  for (uint32_t r = warp; r < P.R; r += 8) {
    const uint32_t i = r / P.g, hh = h * P.g + r % P.g;
    float lse2;
    if (s.first <= s.last) {
      const float2 ml = joined(P, s, r);
      lse2 = (ml.x == -INFINITY ? 0.0f : ml.x) + log2f(ml.y);
    } else {
      lse2 = P.lse[(uint64_t(b) * P.a.n + i) * P.a.hq + hh] * voom::kv::kLog2e;
    }
    if (lane == 0) {
      // a row that sees nothing has no weight anywhere, whatever its factor and its scores are
      const bool none = lse2 == -INFINITY;
      s_row[r] = none ? INFINITY : lse2;
      s_w[r] = none ? 0.0f : P.a.d_token_weight ? P.a.d_token_weight[uint64_t(b) * P.a.n + i] : 1.0f;
    }
  }
  __syncthreads();
  const float* z = P.scores + uint64_t(head) * P.R * P.score_ld;
  const uint32_t begin = voom::kv::first_tile(P, len) * P.keys;  // no row sees what lies before: it has no scores
  float got[kWeightSpan / 256] = {};
  const uint32_t end = min(P.score_ld, s0 + kWeightSpan);
  // four rows' scores under way at a time (up to 16 loads a thread)
  for (uint32_t r0 = 0; r0 < P.R; r0 += 4) {
    float x[4][kWeightSpan / 256];
#pragma unroll
    for (uint32_t q = 0; q < 4; q++) {
      const uint32_t r = r0 + q;
      // in a chain, tiles past the row's own token have no scores
      const uint32_t lim = r >= P.R || s_row[r] == INFINITY ? 0u : P.a.d_mask ? end : min(end, P.score_new + r / P.g + 1);
#pragma unroll
      for (uint32_t k = 0; k < kWeightSpan / 256; k++) {
        const uint32_t s = s0 + k * 256 + tid;
        x[q][k] = s >= begin && s < lim ? z[uint64_t(r) * P.score_ld + s] : -INFINITY;
      }
    }
#pragma unroll
    for (uint32_t q = 0; q < 4; q++) {
      const uint32_t r = min(r0 + q, P.R - 1);
      const float lse2 = s_row[r], w = s_w[r];
#pragma unroll
      for (uint32_t k = 0; k < kWeightSpan / 256; k++) got[k] += w * voom::kv::exp2_fast(x[q][k] - lse2);
    }
  }
  float* sums = P.a.d_weights + int64_t(b) * P.a.w_b + int64_t(h) * P.a.w_h;
#pragma unroll
  for (uint32_t k = 0; k < kWeightSpan / 256; k++) {
    const uint32_t s = s0 + k * 256 + tid;
    if (s < len) sums[s] += got[k];
    else if (s >= P.score_new && s - P.score_new < P.a.n) sums[len + s - P.score_new] += got[k];
  }
}

bool rows16(const void* p, std::initializer_list<int64_t> strides) {
  if (reinterpret_cast<uintptr_t>(p) & 15u) return false;
  for (int64_t s : strides)
    if (s % 8) return false;
  return true;
}

int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      return EncodeTiled(nullptr);
    }
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// Tensor maps of the cache, where TMA can read it: in one piece, or pages of a
// pool whose size is a multiple of 8 positions (a swizzled tile's row groups).
void map_cache(Attn& P) {
  const voom_kv_view& c = P.c.v;
  P.box = 0;
  if (c.d_offsets) return;
  uint32_t box = P.keys;
  if (c.d_table)
    while (box >= 8 && c.page % box) box /= 2;
  if (box < 8 || !encode_tiled()) return;
  const cuuint64_t dims[4] = {c.D, c.page, c.hk, c.d_table ? c.n_pages : c.B};
  const cuuint32_t size[4] = {64, box, 1, 1}, ones[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type = c.type == VOOM_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  auto one = [&](CUtensorMap& map, const void* base, int64_t pos, int64_t head, int64_t page) {
    // a stride that is never used may be anything: TMA wants a positive one
    auto bytes = [](int64_t s, uint64_t n) { return n > 1 ? s * 2 : 16; };
    for (int64_t s : {bytes(pos, dims[1]), bytes(head, dims[2]), bytes(page, dims[3])})
      if (s <= 0 || s >= (int64_t(1) << 40)) return false;
    const cuuint64_t strides[3] = {cuuint64_t(bytes(pos, dims[1])), cuuint64_t(bytes(head, dims[2])), cuuint64_t(bytes(page, dims[3]))};
    return dims[3] > 0 &&
           encode_tiled()(&map, type, 4, const_cast<void*>(base), dims, strides, size, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  if (one(P.k_map, c.d_k, c.k_pos, c.k_head, c.k_page) && one(P.v_map, c.d_v, c.v_pos, c.v_head, c.v_page)) P.box = box;
}

// The scores are more than products.
bool scored(const Attn& P) { return P.a.cap > 0.0f || P.a.d_slopes || P.a.window; }

// Tiles, grid and scratch of a call.  Returns the scratch bytes; sets the
// pointers where `scratch` is given.
uint64_t plan(Attn& P, void* scratch) {
  const voom_kv_view& c = P.c.v;
  P.g = P.a.hq / c.hk;
  P.R = P.a.n * P.g;
  P.words = (P.a.n + 31) / 32;
  P.scale2 = P.a.scale * voom::kv::kLog2e;
  if (P.a.cap > 0.0f) {
    P.cap_in = 2.0f * P.scale2 / P.a.cap;
    P.cap_out = P.a.cap * voom::kv::kLog2e;
    // cap tanh(z / cap) log2(e) = x P(x^2) for z = scale x, |z| <= 3/4 cap
    const double r = double(P.a.scale) / P.a.cap;
    double f = P.scale2;
    bool fine = true;
    for (int i = 0; i < 5; i++, f *= r * r) {
      P.poly[i] = make_float2(float(voom::kv::kTanh[i] * f), float(voom::kv::kTanh[i] * f));
      fine = fine && std::isfinite(P.poly[i].x);
    }
    P.cap_small = fine ? float(0.75 / r) : -1.0f;
  }
  P.ld_o = c.D <= 64 ? 64 : c.D <= 128 ? 128 : 256;
  P.tc = scored(P) && P.R <= voom::kv::kFewRows ? voom::kv::kFew : voom::kv::kRows;
  // attn_rows up to the rows whose output its registers hold in one block; it
  // takes a block of 32 (16 at head size 256) rows over the cache again for
  // each further one: 65 us against 27 at 104 rows over 8191 positions, 630
  // against 88 at 256 rows (8 requests of up to 16384)
  if (P.R > voom::kv::row_most(P.ld_o, scored(P))) {
    P.tc = P.ld_o == 256 ? voom::kv::kSingle : P.R > 128 ? voom::kv::kPair : voom::kv::kAlternate;
    P.keys = P.tc == voom::kv::kSingle ? 64 : 128;
    P.rows = P.tc == voom::kv::kPair ? 256 : 128;
  } else {
    P.keys = voom::kv::row_keys(P.ld_o, scored(P));
    P.rows = P.R > 16 ? 32 : 16;
  }
  P.mblocks = (P.R + P.rows - 1) / P.rows;
  P.tails = uint32_t(voom::kv::tails_before(P, P.mblocks - 1)) + voom::kv::tail_of(P, P.mblocks - 1);
  const uint64_t units = uint64_t(c.B) * c.hk * P.mblocks;
  uint32_t cached = (c.max_len + P.keys - 1) / P.keys;
  if (P.a.window) cached = min(cached, P.a.window / P.keys + 2);  // (a window ends inside a tile at either side)
  const uint32_t steps = cached + (P.a.n + P.keys - 1) / P.keys;
  // a block takes at least two tiles for each of its warps (rows), or a few of
  // the larger ones (tensor cores), before the work is spread further
  const uint32_t least = P.tc >= 0 ? 3 : 2 * voom::kv::row_warps(P.ld_o, scored(P));
  // attn_few: a block alone up to six tiles for each of its warps (3 heads of 64 over
  // 1000 positions: 11.9 us alone, 16.5 split and joined; over 2000, 16.6 and 13.9)
  P.ctas = steps <= (P.tc >= 0 ? 4u : P.tc == voom::kv::kFew ? 3 * least : 2 * least) ? 0u : uint32_t(min(uint64_t(sm_count()), (units * steps + least - 1) / least));
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t o = at;
    at += (bytes + 255) & ~uint64_t(255);
    return scratch ? static_cast<uint8_t*>(scratch) + o : nullptr;
  };
  P.partial = reinterpret_cast<float*>(take(uint64_t(2) * P.ctas * P.rows * (P.ld_o + 2) * sizeof(float)));
  P.lse = P.a.d_lse;
  if (P.a.d_weights) {
    if (!P.lse) P.lse = reinterpret_cast<float*>(take(uint64_t(c.B) * P.a.n * P.a.hq * sizeof(float)));
    // beyond one block of 16 rows attn_sums goes over the keys again: 2 D bytes a
    // position against 8 a row kept here, which is fewer up to D / 4 rows (16 for
    // heads of 64; 32 and 64 rows of larger heads are not measured this way)
    if (P.R > 16) return at;
    P.score_new = (c.max_len + P.keys - 1) / P.keys * P.keys;
    P.score_ld = P.score_new + (P.a.n + P.keys - 1) / P.keys * P.keys;
    P.scores = reinterpret_cast<float*>(take(uint64_t(c.B) * c.hk * P.R * P.score_ld * sizeof(float)));
  }
  return at;
}

template <typename T>
int finish(const Attn& P, cudaStream_t s) {
  const uint64_t units = uint64_t(P.c.v.B) * P.c.v.hk * P.mblocks;
  const uint32_t n_merge = P.ctas ? uint32_t(units * ((P.rows + merge_rows(P) - 1) / merge_rows(P))) : 0u;
  const uint64_t spans = P.scores ? uint64_t(P.c.v.B) * P.c.v.hk * ((P.score_ld + kWeightSpan - 1) / kWeightSpan) : 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(uint32_t(n_merge + spans));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = max(2u * kMergeRows, 2u * (P.scores ? P.R : 0u)) * sizeof(float);
  cfg.stream = s;
  // the launch itself is over by the time the attention ends; its blocks start when
  // the last of the attention's has (none releases them earlier) and wait for its writes
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attn_finish<T>, P, n_merge) == cudaSuccess ? VOOM_OK : VOOM_E_CUDA;
}

template <typename T>
int run(Attn& P, cudaStream_t s) {
  // (attn_few with few tiles: the maps cost the host more than they save)
  if (P.tc >= 0 || (P.tc == voom::kv::kFew && P.ctas == uint32_t(sm_count()))) map_cache(P);
  int rc = scored(P) ? voom::kv::launch_attention<T, true>(P, s) : voom::kv::launch_attention<T, false>(P, s);
  if (rc != VOOM_OK) return rc;
  if (P.ctas || P.scores) rc = finish<T>(P, s);
  if (rc != VOOM_OK || !P.a.d_weights || P.scores) return rc;
  // the rows' weights from the keys again: all rows of a key head as one unit, tiles of 128 keys
  P.keys = 128;
  P.rows = P.R;
  P.mblocks = 1;
  P.tails = voom::kv::tail_of(P, 0);
  uint32_t cached = (P.c.v.max_len + 127) / 128;
  if (P.a.window) cached = min(cached, P.a.window / 128 + 2);
  const uint64_t steps = uint64_t(P.c.v.B) * P.c.v.hk * (cached + P.tails);
  P.ctas = uint32_t(min(uint64_t(sm_count()), steps));
  map_cache(P);
  return scored(P) ? voom::kv::launch_sums<T, true>(P, s) : voom::kv::launch_sums<T, false>(P, s);
}

}  // namespace

VOOM_API int voom_tree_mask(const int32_t* d_parents, uint32_t B, uint32_t n, uint32_t* d_mask, int32_t* d_depth,
                            void* stream) {
  if (!d_parents || !d_mask || !d_depth) return VOOM_E_INVALID_ARG;
  if (n > kMaxTree) return VOOM_E_CAPACITY;
  if (!B || !n) return VOOM_OK;
  tree_mask<<<B, 256, 0, static_cast<cudaStream_t>(stream)>>>(d_parents, n, d_mask, d_depth);
  return cudaGetLastError() == cudaSuccess ? VOOM_OK : VOOM_E_CUDA;
}

namespace {

int check(const voom_kv_view* c, const voom_tree_attention_args* args, Attn& P) {
  if (!args) return VOOM_E_INVALID_ARG;
  // (P is zeros: so is what a caller built before slopes, caps and windows does not have)
  if (args->size == sizeof *args) P.a = *args;
  else std::memcpy(&P.a, args, offsetof(voom_tree_attention_args, d_slopes));
  const voom_tree_attention_args* a = &P.a;
  if (!a->d_q || !a->d_kn || !a->d_vn || !a->d_out) return VOOM_E_INVALID_ARG;
  const int rc = voom::kv::make_view(c, P.c);
  if (rc != VOOM_OK) return rc;
  if (!a->hq || a->hq % c->hk || !(a->scale > 0.0f && a->scale <= 3.0e38f)) return VOOM_E_INVALID_ARG;
  if (!(a->cap >= 0.0f && a->cap <= 3.0e38f)) return VOOM_E_INVALID_ARG;
  if (a->cap > 0.0f && !std::isfinite(4.0f * a->scale / a->cap)) return VOOM_E_INVALID_ARG;
  if (a->d_mask && (a->d_slopes || a->window) && !a->d_depth) return VOOM_E_INVALID_ARG;
  if (a->d_mask && a->n > kMaxTree) return VOOM_E_CAPACITY;
  if (uint64_t(c->max_len) + a->n > 0x7FFFFFFFu || uint64_t(c->B) * a->n * a->hq > 0x7FFFFFFFu) return VOOM_E_UNSUPPORTED;
  if (!rows16(a->d_q, {a->q_b, a->q_t, a->q_h}) || !rows16(a->d_kn, {a->kn_b, a->kn_t, a->kn_h}) ||
      !rows16(a->d_vn, {a->vn_b, a->vn_t, a->vn_h}) || !rows16(a->d_out, {a->o_b, a->o_t, a->o_h}))
    return VOOM_E_INVALID_ARG;
  // blocks write out while others still read the new tokens, and add to the weights without atomics
  const int64_t B = c->B, n = a->n, hq = a->hq, hk = c->hk, D = c->D;
  const voom::Rows out{a->d_out, {B, n, hq}, {a->o_b, a->o_t, a->o_h}, D, 2};
  if (!voom::separate(out) || !voom::disjoint(out, {a->d_q, {B, n, hq}, {a->q_b, a->q_t, a->q_h}, D, 2}) ||
      !voom::disjoint(out, {a->d_kn, {B, n, hk}, {a->kn_b, a->kn_t, a->kn_h}, D, 2}) ||
      !voom::disjoint(out, {a->d_vn, {B, n, hk}, {a->vn_b, a->vn_t, a->vn_h}, D, 2}))
    return VOOM_E_OVERLAP;
  if (a->d_weights && !voom::separate({a->d_weights, {B, hk, 1}, {a->w_b, a->w_h, 0}, int64_t(c->max_len) + n, 4}))
    return VOOM_E_OVERLAP;
  return VOOM_OK;
}

}  // namespace

VOOM_API uint64_t voom_tree_attention_scratch_bytes(const voom_kv_view* c, const voom_tree_attention_args* a) {
  Attn P{};
  if (check(c, a, P) != VOOM_OK || !a->n) return 0;
  return plan(P, nullptr);
}

VOOM_API int voom_tree_attention(const voom_kv_view* c, const voom_tree_attention_args* a, void* d_scratch,
                                 uint64_t bytes, void* stream) {
  Attn P{};
  const int rc = check(c, a, P);
  if (rc != VOOM_OK) return rc;
  if (!a->n) return VOOM_OK;
  const uint64_t need = plan(P, d_scratch);
  if (bytes < need) return VOOM_E_CAPACITY;
  if (need && (!d_scratch || (reinterpret_cast<uintptr_t>(d_scratch) & 15u))) return VOOM_E_INVALID_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return c->type == VOOM_BF16 ? run<__nv_bfloat16>(P, s) : run<__half>(P, s);
}
