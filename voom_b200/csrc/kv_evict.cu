// Eviction from a KV cache by accumulated attention weight.
//
// For each request and head: of the positions between the first `sinks` and
// the newest `recent`, the budget - sinks - recent with the largest weights
// stay.
//
// evict_select finds the smallest weight that stays by a radix select over the
// weights' bits, ordered as unsigned numbers, 11 bits to a pass.  A cluster of
// up to eight blocks shares a head: each reads its slice of the weights once,
// into shared memory, and the passes exchange only their 2048 counts, through
// distributed shared memory.  Ties at the smallest weight go to the lower
// positions, so each block also counts what its predecessors keep; then it
// writes its kept positions in order.
//
// evict_gather copies the kept rows, bound by HBM: a warp finds 32 rows'
// addresses at once, its lanes then copy them 16 bytes at a time.
//
// Measured: 131071 -> 32768 positions, 8 heads of 128: 79 us, 45 % of it
// the selection (one block per head took 200 us), the rest the copy, 6.2 TB/s.
#include <atomic>

#include <cooperative_groups.h>

#include "kv_view.cuh"

namespace {

using voom::kv::View;

namespace cg = cooperative_groups;

constexpr uint32_t kSelThreads = 512;
constexpr uint32_t kSelWarps = kSelThreads / 32;
constexpr uint32_t kBins = 2048;
constexpr uint32_t kMaxKeys = 40960;  // keys of a block's slice that shared memory holds

struct Evict {
  View c;
  voom_kv_evict_args a;
  uint32_t held;  // keys of a slice are held in shared memory
};

// Unsigned order of the weights: larger weight, larger key; NaN above all, -0 = 0.
__device__ __forceinline__ uint32_t key_of(float w) {
  if (isnan(w)) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The weight of a key (a NaN comes back as the canonical one, -0 as 0).
__device__ __forceinline__ float weight_of(uint32_t k) {
  return __uint_as_float(k == 0xFFFFFFFFu ? 0x7FFFFFFFu : k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// Sum of x over the threads after this one (by index); every thread gets `total`.
__device__ __forceinline__ uint32_t sum_after(uint32_t x, uint32_t* s_warp, uint32_t& total) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  uint32_t y = x;
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t z = __shfl_down_sync(0xFFFFFFFFu, y, o);
    if (lane + o < 32) y += z;
  }
  __syncthreads();
  if (lane == 0) s_warp[warp] = y;
  __syncthreads();
  uint32_t after = 0;
  total = 0;
  for (uint32_t w = 0; w < kSelWarps; w++) {
    total += s_warp[w];
    if (w > warp) after += s_warp[w];
  }
  return y - x + after;
}

__global__ void __launch_bounds__(kSelThreads) evict_select(const __grid_constant__ Evict P) {
  extern __shared__ uint32_t s_keys[];
  __shared__ __align__(16) uint32_t s_hist[2][kBins];
  __shared__ uint32_t s_warp[kSelWarps], s_pick[2], s_gt[kSelWarps], s_tie[kSelWarps], s_all[2];
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t rank = cluster.block_rank(), ranks = cluster.num_blocks();
  const uint32_t h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t len = P.c.length(b), budget = P.a.budget, kept = min(len, budget);
  const uint64_t out = (uint64_t(b) * P.c.v.hk + h) * budget;
  const float* w = P.a.d_weights + int64_t(b) * P.a.w_b + int64_t(h) * P.a.w_h;
  int32_t* index = P.a.d_index + out;
  float* w_out = P.a.d_w_out + out;
  const uint32_t first = rank * kSelThreads + tid, stride = ranks * kSelThreads;
  if (h == 0 && first == 0) P.a.d_len_out[b] = int32_t(kept);
  for (uint32_t j = kept + first; j < budget; j += stride) {
    index[j] = -1;
    w_out[j] = 0.0f;
  }
  if (len <= budget) {  // the same for the whole cluster
    for (uint32_t j = first; j < kept; j += stride) {
      index[j] = int32_t(j);
      w_out[j] = w[j];
    }
    return;
  }
  // [0, lo) and [hi, len) stay; of the m positions between, `want`
  const uint32_t lo = P.a.sinks, hi = len - P.a.recent, m = hi - lo;
  uint32_t want = budget - P.a.sinks - P.a.recent;
  for (uint32_t s = first; s < lo; s += stride) {
    index[s] = int32_t(s);
    w_out[s] = w[s];
  }
  for (uint32_t s = hi + first; s < len; s += stride) {
    index[s - len + budget] = int32_t(s);
    w_out[s - len + budget] = w[s];
  }
  if (!want) return;  // the same for the whole cluster
  const uint32_t per = (m + ranks - 1) / ranks, begin = min(m, rank * per), n = min(m, begin + per) - begin;
  w += lo + begin;  // this block's slice
  const bool held = P.held;
  if (held) {
    constexpr uint32_t kDeep = 8;  // loads of a thread under way
    for (uint32_t i0 = tid; i0 < n; i0 += kDeep * kSelThreads) {
      float x[kDeep];
#pragma unroll
      for (uint32_t k = 0; k < kDeep; k++) x[k] = i0 + k * kSelThreads < n ? w[i0 + k * kSelThreads] : 0.0f;
#pragma unroll
      for (uint32_t k = 0; k < kDeep; k++)
        if (i0 + k * kSelThreads < n) s_keys[i0 + k * kSelThreads] = key_of(x[k]);
    }
  }
  auto key = [&](uint32_t i) { return held ? s_keys[i] : key_of(w[i]); };
  uint32_t prefix = 0, mask = 0;
#pragma unroll 1
  for (uint32_t pass = 0; pass < 3; pass++) {
    const uint32_t shift = pass == 0 ? 21u : pass == 1 ? 10u : 0u, bits = pass == 2 ? 10u : 11u;
    uint32_t* hist = s_hist[pass & 1u];
    for (uint32_t i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < n; i += kSelThreads) {
      const uint32_t k = key(i);
      if (((k ^ prefix) & mask) == 0) atomicAdd(&hist[k >> shift & ((1u << bits) - 1u)], 1u);
    }
    cluster.sync();
    // four bins to a thread, summed over the cluster
    uint4 c = make_uint4(0, 0, 0, 0);
    for (uint32_t r = 0; r < ranks; r++) {
      const uint4 x = reinterpret_cast<const uint4*>(cluster.map_shared_rank(hist, r))[tid];
      c.x += x.x;
      c.y += x.y;
      c.z += x.z;
      c.w += x.w;
    }
    uint32_t total;
    const uint32_t above = sum_after(c.x + c.y + c.z + c.w, s_warp, total);
    // the digit of the smallest key that stays: as many larger ones as are wanted, less one, at most
    uint32_t a = above;
    const uint32_t bins[4] = {c.w, c.z, c.y, c.x};
#pragma unroll
    for (uint32_t d = 0; d < 4; d++) {
      if (a < want && want <= a + bins[d]) {
        s_pick[0] = 4 * tid + 3 - d;
        s_pick[1] = want - a;
      }
      a += bins[d];
    }
    __syncthreads();
    prefix |= s_pick[0] << shift;
    mask |= ((1u << bits) - 1u) << shift;
    want = s_pick[1];
    // the counts of this pass are read until the next pass's sync; the pass after that writes them again
  }
  // `prefix` is the smallest key that stays, for the first `want` positions that have it
  const uint32_t chunk = ((n + kSelWarps - 1) / kSelWarps + 31u) & ~31u, c0 = min(n, warp * chunk), c1 = min(n, c0 + chunk);
  uint32_t gt = 0, tie = 0;
  for (uint32_t i = c0 + lane; i < c1; i += 32) {
    const uint32_t k = key(i);
    gt += k > prefix;
    tie += k == prefix;
  }
  gt = __reduce_add_sync(0xFFFFFFFFu, gt);
  tie = __reduce_add_sync(0xFFFFFFFFu, tie);
  if (lane == 0) {
    s_gt[warp] = gt;
    s_tie[warp] = tie;
  }
  __syncthreads();
  uint32_t gt0 = 0, tie0 = 0;
  for (uint32_t x = 0; x < kSelWarps; x++) {
    if (tid == 0 && x == 0) s_all[0] = s_all[1] = 0;
    if (tid == 0) {
      s_all[0] += s_gt[x];
      s_all[1] += s_tie[x];
    }
    if (x < warp) {
      gt0 += s_gt[x];
      tie0 += s_tie[x];
    }
  }
  cluster.sync();
  for (uint32_t r = 0; r < rank; r++) {
    const uint32_t* x = cluster.map_shared_rank(s_all, r);
    gt0 += x[0];
    tie0 += x[1];
  }
  uint32_t at = lo + gt0 + min(tie0, want);
  for (uint32_t i0 = c0; i0 < c1; i0 += 32) {
    const uint32_t i = i0 + lane, k = i < c1 ? key(i) : 0u, below = (1u << lane) - 1u;
    const uint32_t ties = __ballot_sync(0xFFFFFFFFu, i < c1 && k == prefix);
    const bool keep = i < c1 && (k > prefix || (k == prefix && tie0 + __popc(ties & below) < want));
    const uint32_t keeps = __ballot_sync(0xFFFFFFFFu, keep);
    if (keep) {
      index[at + __popc(keeps & below)] = int32_t(lo + begin + i);
      w_out[at + __popc(keeps & below)] = weight_of(k);
    }
    at += __popc(keeps);
    tie0 += __popc(ties);
  }
  cluster.sync();  // no block leaves while another reads its counts
}

constexpr uint32_t kGatherRows = 32;  // of a warp

// chunks: 16-byte pieces of a row, D / 8, of which a group of `lanes` lanes copies one row.
__global__ void __launch_bounds__(128) evict_gather(const __grid_constant__ Evict P, uint32_t lanes) {
  const uint32_t chunks = P.c.v.D / 8, h = blockIdx.y, b = blockIdx.z, budget = P.a.budget, lane = threadIdx.x & 31u;
  const uint32_t j0 = (blockIdx.x * 4 + (threadIdx.x >> 5)) * kGatherRows;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (j0 >= budget) return;
  const uint64_t row0 = (uint64_t(b) * P.c.v.hk + h) * budget + j0;
  uint64_t ka = 0, va = 0;
  if (j0 + lane < budget) {
    const int32_t s = P.a.d_index[row0 + lane];
    int64_t ko, vo;
    if (s >= 0 && P.c.row_at(b, h, uint32_t(s), ko, vo)) {
      ka = reinterpret_cast<uint64_t>(static_cast<const uint16_t*>(P.c.v.d_k) + ko);
      va = reinterpret_cast<uint64_t>(static_cast<const uint16_t*>(P.c.v.d_v) + vo);
    }
  }
  const uint32_t rows = min(kGatherRows, budget - j0), e = lane & (lanes - 1), step = 32 / lanes;
  uint4* k_out = static_cast<uint4*>(P.a.d_k_out) + row0 * chunks + e;
  uint4* v_out = static_cast<uint4*>(P.a.d_v_out) + row0 * chunks + e;
  constexpr uint32_t kDeep = 4;  // rows of a lane under way
  for (uint32_t r0 = 0; r0 < kGatherRows; r0 += step * kDeep) {
    uint4 k[kDeep], v[kDeep];
#pragma unroll
    for (uint32_t x = 0; x < kDeep; x++) {
      const uint32_t r = r0 + x * step + lane / lanes;
      const uint64_t kp = __shfl_sync(0xFFFFFFFFu, ka, r & 31u), vp = __shfl_sync(0xFFFFFFFFu, va, r & 31u);
      k[x] = v[x] = make_uint4(0, 0, 0, 0);
      if (r < rows && e < chunks && kp) {
        k[x] = __ldcs(reinterpret_cast<const uint4*>(kp) + e);
        v[x] = __ldcs(reinterpret_cast<const uint4*>(vp) + e);
      }
    }
#pragma unroll
    for (uint32_t x = 0; x < kDeep; x++) {
      const uint32_t r = r0 + x * step + lane / lanes;
      if (r < rows && e < chunks) {
        k_out[uint64_t(r) * chunks] = k[x];
        v_out[uint64_t(r) * chunks] = v[x];
      }
    }
  }
}

}  // namespace

VOOM_API int voom_kv_evict(const voom_kv_view* c, const voom_kv_evict_args* a, void* stream) {
  if (!a || !a->d_weights || !a->d_k_out || !a->d_v_out || !a->d_w_out || !a->d_index || !a->d_len_out)
    return VOOM_E_INVALID_ARG;
  Evict P{};
  const int rc = voom::kv::make_view(c, P.c);
  if (rc != VOOM_OK) return rc;
  if (!a->budget || uint64_t(a->sinks) + a->recent > a->budget) return VOOM_E_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(a->d_k_out) | reinterpret_cast<uintptr_t>(a->d_v_out)) & 15u) return VOOM_E_INVALID_ARG;
  if (a->budget > 0x7FFFFFFFu / 32u) return VOOM_E_UNSUPPORTED;
  P.a = *a;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // blocks to a head: enough that a slice is short, as long as SMs are free
  const uint64_t heads = uint64_t(c->B) * c->hk;
  uint32_t ranks = 1;
  while (ranks < 8 && c->max_len > ranks * 4096u && heads * ranks < 148) ranks *= 2;
  while (ranks < 8 && c->max_len > ranks * kMaxKeys) ranks *= 2;
  const uint32_t slice = (c->max_len + ranks - 1) / ranks;
  P.held = slice <= kMaxKeys;
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return VOOM_E_CUDA;
  if (!(allowed.load(std::memory_order_relaxed) >> (dev & 63) & 1u)) {
    if (cudaFuncSetAttribute(evict_select, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxKeys * 4) != cudaSuccess) {
      cudaGetLastError();
      return VOOM_E_CUDA;
    }
    allowed.fetch_or(uint64_t(1) << (dev & 63), std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at{};
  cfg.gridDim = dim3(ranks, c->hk, c->B);
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = P.held ? slice * 4u : 0u;
  cfg.stream = s;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = ranks;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, evict_select, P) != cudaSuccess) {
    cudaGetLastError();
    return VOOM_E_CUDA;
  }
  uint32_t lanes = 1;
  while (lanes < c->D / 8) lanes *= 2;
  const uint32_t per = 4 * kGatherRows;
  cudaLaunchConfig_t gcfg{};
  // the launch itself is over by the time the selection ends; its blocks start when
  // the last of the selection's has (none releases them earlier) and wait for its writes
  cudaLaunchAttribute early{};
  gcfg.gridDim = dim3((a->budget + per - 1) / per, c->hk, c->B);
  gcfg.blockDim = dim3(128);
  gcfg.stream = s;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  gcfg.attrs = &early;
  gcfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&gcfg, evict_gather, P, lanes) != cudaSuccess) {
    cudaGetLastError();
    return VOOM_E_CUDA;
  }
  return VOOM_OK;
}
