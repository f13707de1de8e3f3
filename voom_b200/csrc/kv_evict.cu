// Eviction from a KV cache by accumulated attention weight.
//
// For each request and head: of the positions between the first `sinks` and
// the newest `recent`, the budget - sinks - recent with the largest weights
// stay.  evict_select finds the smallest weight that stays by a radix select
// over the weights' bits (ordered as unsigned numbers), 8 bits to a pass, and
// writes the kept positions in order; evict_gather copies their rows.
#include "kv_view.cuh"

namespace {

using voom::kv::View;

constexpr uint32_t kSelThreads = 1024;

struct Evict {
  View c;
  voom_kv_evict_args a;
};

// Unsigned order of the weights: larger weight, larger key; NaN above all, -0 = 0.
__device__ __forceinline__ uint32_t key_of(float w) {
  if (isnan(w)) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive prefix of `flag` over the block's threads; `total` gets the sum.
__device__ __forceinline__ uint32_t block_rank(bool flag, uint32_t* s_warp, uint32_t& total) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, m = __ballot_sync(0xFFFFFFFFu, flag);
  if (lane == 0) s_warp[warp] = __popc(m);
  __syncthreads();
  if (warp == 0) {
    const uint32_t v = s_warp[lane];
    uint32_t x = v;
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, x, o);
      if (int(lane) >= o) x += y;
    }
    s_warp[lane] = x - v;
    if (lane == 31) s_warp[32] = x;
  }
  __syncthreads();
  const uint32_t r = s_warp[warp] + __popc(m & ((1u << lane) - 1u));
  total = s_warp[32];
  __syncthreads();
  return r;
}

__global__ void __launch_bounds__(kSelThreads) evict_select(const Evict P) {
  __shared__ uint32_t s_hist[256], s_warp[33], s_pick[2];
  const uint32_t h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const uint32_t len = P.c.length(b), budget = P.a.budget;
  const uint32_t kept = min(len, budget);
  const uint64_t out = (uint64_t(b) * P.c.v.hk + h) * budget;
  const float* w = P.a.d_weights + int64_t(b) * P.a.w_b + int64_t(h) * P.a.w_h;
  int32_t* index = P.a.d_index + out;
  if (h == 0 && tid == 0) P.a.d_len_out[b] = int32_t(kept);
  for (uint32_t j = kept + tid; j < budget; j += kSelThreads) {
    index[j] = -1;
    P.a.d_w_out[out + j] = 0.0f;
  }
  if (len <= budget) {
    for (uint32_t j = tid; j < kept; j += kSelThreads) {
      index[j] = int32_t(j);
      P.a.d_w_out[out + j] = w[j];
    }
    return;
  }
  const uint32_t lo = P.a.sinks, hi = len - P.a.recent;
  uint32_t want = budget - P.a.sinks - P.a.recent;  // of [lo, hi): fewer than hi - lo
  uint32_t prefix = 0, mask = 0;
  for (int shift = 24; shift >= 0 && want; shift -= 8) {
    if (tid < 256) s_hist[tid] = 0;
    __syncthreads();
    for (uint32_t s = lo + tid; s < hi; s += kSelThreads) {
      const uint32_t k = key_of(w[s]);
      if ((k & mask) == prefix) atomicAdd(&s_hist[k >> shift & 255u], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t left = want;
      int d = 255;
      while (s_hist[d] < left) left -= s_hist[d--];
      s_pick[0] = uint32_t(d);
      s_pick[1] = left;
    }
    __syncthreads();
    prefix |= s_pick[0] << shift;
    mask |= 255u << shift;
    want = s_pick[1];
    __syncthreads();
  }
  // prefix: the smallest key that stays; `want` of the positions that have it do
  const bool none = budget == P.a.sinks + P.a.recent;
  uint32_t done = 0, ties = 0;
  for (uint32_t s0 = 0; s0 < len; s0 += kSelThreads) {
    const uint32_t s = s0 + tid;
    const bool in = s < len, middle = in && s >= lo && s < hi && !none;
    const uint32_t k = middle ? key_of(w[s]) : 0u;
    uint32_t total;
    const uint32_t tie = block_rank(middle && k == prefix, s_warp, total) + ties;
    ties += total;
    const bool keep = in && (s < lo || s >= hi || (middle && (k > prefix || (k == prefix && tie < want))));
    const uint32_t at = block_rank(keep, s_warp, total) + done;
    done += total;
    if (keep) {
      index[at] = int32_t(s);
      P.a.d_w_out[out + at] = w[s];
    }
  }
}

// A group of D / 8 threads per kept row: 16 bytes of its key and of its value each.
__global__ void __launch_bounds__(256) evict_gather(const Evict P) {
  const uint32_t chunks = P.c.v.D / 8, h = blockIdx.y, b = blockIdx.z, budget = P.a.budget;
  const uint64_t item = uint64_t(blockIdx.x) * 256 + threadIdx.x;
  const uint32_t j = uint32_t(item / chunks), e = uint32_t(item % chunks);
  if (j >= budget) return;
  const uint64_t row = (uint64_t(b) * P.c.v.hk + h) * budget + j;
  const int32_t s = P.a.d_index[row];
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  int64_t ko, vo;
  if (s >= 0 && P.c.row_at(b, h, uint32_t(s), ko, vo)) {
    k = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(P.c.v.d_k) + ko + 8 * e);
    v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(P.c.v.d_v) + vo + 8 * e);
  }
  reinterpret_cast<uint4*>(P.a.d_k_out)[row * chunks + e] = k;
  reinterpret_cast<uint4*>(P.a.d_v_out)[row * chunks + e] = v;
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
  evict_select<<<dim3(c->hk, c->B), kSelThreads, 0, s>>>(P);
  const uint64_t items = uint64_t(a->budget) * (c->D / 8);
  evict_gather<<<dim3(uint32_t((items + 255) / 256), c->hk, c->B), 256, 0, s>>>(P);
  return cudaGetLastError() == cudaSuccess ? VOOM_OK : VOOM_E_CUDA;
}
