// Attention of drafted tokens over a KV cache, its weight sums, and the tree masks.
#include <initializer_list>

#include "kv_view.cuh"

namespace {

using voom::kv::elem;
using voom::kv::rounded;
using voom::kv::View;

constexpr uint32_t kMaxTree = 1024;

struct Attn {
  View c;
  voom_tree_attention_args a;
  float* lse;  // a.d_lse, or scratch
  uint32_t g, words;
};

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

// ------------------------------------------------------------------- rows
__device__ __forceinline__ bool sees(const Attn& P, uint32_t b, uint32_t i, uint32_t j) {
  if (!P.a.d_mask) return j <= i;
  return P.a.d_mask[(uint64_t(b) * P.a.n + i) * P.words + (j >> 5)] >> (j & 31u) & 1u;
}

// Key and value row of position s (cached, then new); false: a page that is none.
template <typename T>
__device__ __forceinline__ bool rows_of(const Attn& P, uint32_t b, uint32_t h, uint32_t len, uint32_t s, const T*& k,
                                        const T*& v) {
  if (s < len) {
    int64_t ko, vo;
    if (!P.c.row_at(b, h, s, ko, vo)) return false;
    k = static_cast<const T*>(P.c.v.d_k) + ko;
    v = static_cast<const T*>(P.c.v.d_v) + vo;
  } else {
    const int64_t j = s - len;
    k = static_cast<const T*>(P.a.d_kn) + int64_t(b) * P.a.kn_b + j * P.a.kn_t + int64_t(h) * P.a.kn_h;
    v = static_cast<const T*>(P.a.d_vn) + int64_t(b) * P.a.vn_b + j * P.a.vn_t + int64_t(h) * P.a.vn_h;
  }
  return true;
}

__device__ __forceinline__ float warp_sum(float x) {
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
  return x;
}

constexpr uint32_t kPer = voom::kv::kMaxD / 32;  // head values of a lane

// One warp per row (request, new token, query head): running maximum and sum
// of the softmax over the keys, one at a time.
template <typename T>
__global__ void __launch_bounds__(256) attn_rows(const Attn P) {
  const uint32_t lane = threadIdx.x & 31u, n = P.a.n, hq = P.a.hq, D = P.c.v.D;
  const uint64_t row = uint64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= uint64_t(P.c.v.B) * n * hq) return;
  const uint32_t hh = uint32_t(row % hq), i = uint32_t(row / hq % n), b = uint32_t(row / hq / n), h = hh / P.g;
  const uint32_t len = P.c.length(b);
  const T* q = static_cast<const T*>(P.a.d_q) + int64_t(b) * P.a.q_b + int64_t(i) * P.a.q_t + int64_t(hh) * P.a.q_h;
  float x[kPer], o[kPer];
  for (uint32_t e = 0; e < kPer; e++) {
    x[e] = lane + 32 * e < D ? elem<T>(q[lane + 32 * e]) * P.a.scale : 0.0f;
    o[e] = 0.0f;
  }
  float top = -INFINITY, sum = 0.0f;
  if (sees(P, b, i, i))
    for (uint32_t s = 0; s < len + n; s++) {
      if (s >= len && !sees(P, b, i, s - len)) continue;
      const T *k, *v;
      const bool is = rows_of<T>(P, b, h, len, s, k, v);
      float z = 0.0f;
      for (uint32_t e = 0; e < kPer; e++)
        if (is && lane + 32 * e < D) z += x[e] * elem<T>(k[lane + 32 * e]);
      z = warp_sum(z);
      const float t = fmaxf(top, z), f = expf(top - t), p = expf(z - t);
      sum = sum * f + p;
      for (uint32_t e = 0; e < kPer; e++)
        o[e] = o[e] * f + (is && lane + 32 * e < D ? p * elem<T>(v[lane + 32 * e]) : 0.0f);
      top = t;
    }
  T* out = static_cast<T*>(P.a.d_out) + int64_t(b) * P.a.o_b + int64_t(i) * P.a.o_t + int64_t(hh) * P.a.o_h;
  for (uint32_t e = 0; e < kPer; e++)
    if (lane + 32 * e < D) out[lane + 32 * e] = rounded<T>(sum == 0.0f ? 0.0f : o[e] / sum);
  if (P.lse && lane == 0) P.lse[row] = top + logf(sum);
}

// One warp per (request, key head, position): the rows' weights at it, from
// the scores and the rows' softmax denominators.
template <typename T>
__global__ void __launch_bounds__(256) attn_weights(const Attn P) {
  const uint32_t lane = threadIdx.x & 31u, n = P.a.n, D = P.c.v.D, b = blockIdx.z, h = blockIdx.y;
  const uint32_t len = P.c.length(b), s = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (s >= len + n) return;
  const T *k, *v;
  const bool is = rows_of<T>(P, b, h, len, s, k, v);
  float x[kPer];
  for (uint32_t e = 0; e < kPer; e++) x[e] = is && lane + 32 * e < D ? elem<T>(k[lane + 32 * e]) * P.a.scale : 0.0f;
  float got = 0.0f;
  for (uint32_t i = 0; i < n; i++) {
    if (!sees(P, b, i, i) || (s >= len && !sees(P, b, i, s - len))) continue;
    const float tw = P.a.d_token_weight ? P.a.d_token_weight[uint64_t(b) * n + i] : 1.0f;
    for (uint32_t hh = h * P.g; hh < (h + 1) * P.g; hh++) {
      const T* q = static_cast<const T*>(P.a.d_q) + int64_t(b) * P.a.q_b + int64_t(i) * P.a.q_t + int64_t(hh) * P.a.q_h;
      float z = 0.0f;
      for (uint32_t e = 0; e < kPer; e++)
        if (lane + 32 * e < D) z += x[e] * elem<T>(q[lane + 32 * e]);
      z = warp_sum(z);
      got += tw * expf(z - P.lse[(uint64_t(b) * n + i) * P.a.hq + hh]);
    }
  }
  if (lane == 0) P.a.d_weights[int64_t(b) * P.a.w_b + int64_t(h) * P.a.w_h + s] += got;
}

bool rows16(const void* p, std::initializer_list<int64_t> strides) {
  if (reinterpret_cast<uintptr_t>(p) & 15u) return false;
  for (int64_t s : strides)
    if (s % 8) return false;
  return true;
}

uint64_t plan(Attn& P, void* scratch) {
  P.g = P.a.hq / P.c.v.hk;
  P.words = (P.a.n + 31) / 32;
  P.lse = P.a.d_lse;
  if (!P.a.d_weights || P.lse) return 0;
  P.lse = static_cast<float*>(scratch);
  return uint64_t(P.c.v.B) * P.a.n * P.a.hq * sizeof(float);
}

template <typename T>
int run(const Attn& P, cudaStream_t s) {
  const uint64_t rows = uint64_t(P.c.v.B) * P.a.n * P.a.hq;
  attn_rows<T><<<uint32_t((rows + 7) / 8), 256, 0, s>>>(P);
  if (P.a.d_weights)
    attn_weights<T><<<dim3((P.c.v.max_len + P.a.n + 7) / 8, P.c.v.hk, P.c.v.B), 256, 0, s>>>(P);
  return cudaGetLastError() == cudaSuccess ? VOOM_OK : VOOM_E_CUDA;
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

int check(const voom_kv_view* c, const voom_tree_attention_args* a, Attn& P) {
  if (!a || !a->d_q || !a->d_kn || !a->d_vn || !a->d_out) return VOOM_E_INVALID_ARG;
  const int rc = voom::kv::make_view(c, P.c);
  if (rc != VOOM_OK) return rc;
  if (!a->hq || a->hq % c->hk) return VOOM_E_INVALID_ARG;
  if (a->d_mask && a->n > kMaxTree) return VOOM_E_CAPACITY;
  if (uint64_t(c->max_len) + a->n > 0x7FFFFFFFu || uint64_t(c->B) * a->n * a->hq > 0x7FFFFFFFu) return VOOM_E_UNSUPPORTED;
  if (!rows16(a->d_q, {a->q_b, a->q_t, a->q_h}) || !rows16(a->d_kn, {a->kn_b, a->kn_t, a->kn_h}) ||
      !rows16(a->d_vn, {a->vn_b, a->vn_t, a->vn_h}) || !rows16(a->d_out, {a->o_b, a->o_t, a->o_h}))
    return VOOM_E_INVALID_ARG;
  P.a = *a;
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
  if (need && (!d_scratch || (reinterpret_cast<uintptr_t>(d_scratch) & 15u))) return VOOM_E_INVALID_ARG;
  if (bytes < need) return VOOM_E_CAPACITY;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return c->type == VOOM_BF16 ? run<__nv_bfloat16>(P, s) : run<__half>(P, s);
}
