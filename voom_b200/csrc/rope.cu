// Per-head RMS norm of queries and keys and the position rotation, one pass.
//
//   y = x * rsqrt(mean(x^2) + eps) * w,   then for each pair of the first `rot`
//   values  (a, b) -> factor * (a cos t - b sin t, a sin t + b cos t)
//
// The angle: `turns` holds the pair's turns per position as a 64-bit fraction,
// so position * turns modulo 2^64 is the fraction of a turn whatever the
// position (fp32 position * frequency is off by 0.01 rad at 10^5 already).
// Its top 32 bits, as a signed half-turn count in [-1, 1), go to sincospif.
//
// Bound by HBM: every value is read and written once (2 bytes each way in
// BF16), about ten instructions per value.  A CTA takes a few tokens: its
// threads first make the tokens' cosines and sines, one pair each, into
// shared memory, then groups of lanes take one head each, two chunks of VEC
// values per lane: the two halves that a pair's members lie in ("half"
// layout), so that a pair never crosses lanes and the norm's sum is the only
// exchange.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxD = 512;

struct Rope {
  voom_qk_norm_rope_args a;
  uint32_t tokens;    // tokens per CTA
  uint32_t lanes;     // lanes per head: a power of two
  uint32_t rot_tasks; // tasks in the rotated part (two chunks each)
  uint32_t tasks;     // tasks of a head
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Chunk {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ void load_chunk(const T* p, float (&x)[VEC]) {
  const Chunk<T, VEC> c = *reinterpret_cast<const Chunk<T, VEC>*>(p);
#pragma unroll
  for (int i = 0; i < VEC; i++) x[i] = to_f<T>(c.v[i]);
}

template <typename T, int VEC>
__device__ __forceinline__ void store_chunk(T* p, const float (&x)[VEC]) {
  Chunk<T, VEC> c;
#pragma unroll
  for (int i = 0; i < VEC; i++) c.v[i] = from_f<T>(x[i]);
  *reinterpret_cast<Chunk<T, VEC>*>(p) = c;
}

__device__ __forceinline__ float weight(const void* w, uint32_t type, uint32_t i) {
  if (type == VOOM_FP32) return static_cast<const float*>(w)[i];
  if (type == VOOM_FP16) return __half2float(static_cast<const __half*>(w)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// What a lane's task covers: chunks at i0 and (two) i1.
struct Span {
  uint32_t i0, i1;
  bool has, two, rotated;
};

template <int VEC>
__device__ __forceinline__ Span span_of(const Rope& P, uint32_t task) {
  Span c;
  c.has = task < P.tasks;
  c.rotated = task < P.rot_tasks;
  c.two = true;
  if (!c.rotated) {
    c.i0 = P.a.rot + (task - P.rot_tasks) * 2 * VEC;
    c.i1 = c.i0 + VEC;
    c.two = c.i1 < P.a.D;
  } else if (P.a.interleaved) {
    c.i0 = task * 2 * VEC;
    c.i1 = c.i0 + VEC;
  } else {
    c.i0 = task * VEC;
    c.i1 = c.i0 + P.a.rot / 2;
  }
  return c;
}

__device__ __forceinline__ void turn(float& a, float& b, float2 cs) {
  const float p = a, q = b;
  a = p * cs.x - q * cs.y;
  b = p * cs.y + q * cs.x;
}

// KT tasks of two chunks to a lane: task k of lane l is l + k * lanes.
template <typename T, int VEC, int KT>
__global__ void __launch_bounds__(kThreads) qk_norm_rope(const Rope P) {
  const voom_qk_norm_rope_args& a = P.a;
  extern __shared__ float2 s_cs[];  // [token][pair]
  const uint32_t t0 = blockIdx.x * P.tokens, nt = min(P.tokens, a.T - t0), half = a.rot / 2;
  float* s_w = reinterpret_cast<float*>(s_cs + P.tokens * half);  // q weights, then k weights
  for (uint32_t i = threadIdx.x; i < nt * half; i += kThreads) {
    const uint32_t t = i / half, p = i - t * half;
    const int64_t pos =
        a.pos64 ? static_cast<const int64_t*>(a.d_pos)[t0 + t] : int64_t(static_cast<const int32_t*>(a.d_pos)[t0 + t]);
    const uint64_t frac = uint64_t(pos) * a.d_turns[p];
    const float x = float(int32_t(frac >> 32)) * (1.0f / 2147483648.0f);
    float s, c;
    sincospif(x, &s, &c);
    s_cs[i] = make_float2(c * a.factor, s * a.factor);
  }
  const float one = a.zero_centered ? 1.0f : 0.0f;
  for (uint32_t i = threadIdx.x; i < a.D; i += kThreads) {
    if (a.d_q_w) s_w[i] = weight(a.d_q_w, a.w_type, i) + one;
    if (a.d_k_w) s_w[a.D + i] = weight(a.d_k_w, a.w_type, i) + one;
  }
  __syncthreads();
  const uint32_t lane = threadIdx.x & (P.lanes - 1), per = kThreads / P.lanes, heads = a.hq + a.hk;
  const uint32_t items = nt * heads;
  // every thread makes the same number of rounds, so that the shuffles of the
  // norm always have all their lanes
  for (uint32_t first = 0; first < items; first += per) {
    const uint32_t it = first + threadIdx.x / P.lanes;
    const bool on = it < items;
    const uint32_t t = on ? it / heads : 0u, h = on ? it - t * heads : 0u;
    const bool isq = h < a.hq;
    const uint32_t hh = isq ? h : h - a.hq;
    const T* src = isq ? static_cast<const T*>(a.d_q) + int64_t(t0 + t) * a.q_token + int64_t(hh) * a.q_head
                       : static_cast<const T*>(a.d_k) + int64_t(t0 + t) * a.k_token + int64_t(hh) * a.k_head;
    T* dst = isq ? static_cast<T*>(a.d_q_out) + int64_t(t0 + t) * a.qo_token + int64_t(hh) * a.qo_head
                 : static_cast<T*>(a.d_k_out) + int64_t(t0 + t) * a.ko_token + int64_t(hh) * a.ko_head;
    const bool norm = isq ? a.d_q_w != nullptr : a.d_k_w != nullptr;
    const float* w = s_w + (isq ? 0u : a.D);
    const float2* cs = s_cs + t * half;
    float x[KT][VEC] = {}, y[KT][VEC] = {};
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < KT; k++) {
      const Span c = span_of<VEC>(P, lane + k * P.lanes);
      if (on && c.has) {
        load_chunk<T, VEC>(src + c.i0, x[k]);
        if (c.two) load_chunk<T, VEC>(src + c.i1, y[k]);
      }
#pragma unroll
      for (int i = 0; i < VEC; i++) sum += x[k][i] * x[k][i] + y[k][i] * y[k][i];
    }
    float r = 1.0f;
    if (a.d_q_w || a.d_k_w) {
      for (uint32_t o = P.lanes / 2; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
      r = rsqrtf(sum / float(a.D) + a.eps);
    }
#pragma unroll
    for (int k = 0; k < KT; k++) {
      const Span c = span_of<VEC>(P, lane + k * P.lanes);
      if (!on || !c.has) continue;
      if (norm) {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          x[k][i] *= r * w[c.i0 + i];
          if (c.two) y[k][i] *= r * w[c.i1 + i];
        }
      }
      if (c.rotated) {
        if (!a.interleaved || VEC == 1) {  // the pairs are (x[i], y[i])
#pragma unroll
          for (int i = 0; i < VEC; i++) turn(x[k][i], y[k][i], cs[(a.interleaved ? c.i0 / 2 : c.i0) + i]);
        } else {
#pragma unroll
          for (int i = 0; i + 1 < VEC; i += 2) {
            turn(x[k][i], x[k][i + 1], cs[(c.i0 + i) / 2]);
            turn(y[k][i], y[k][i + 1], cs[(c.i1 + i) / 2]);
          }
        }
      }
      store_chunk<T, VEC>(dst + c.i0, x[k]);
      if (c.two) store_chunk<T, VEC>(dst + c.i1, y[k]);
    }
  }
}

bool aligned(const voom_qk_norm_rope_args& a, uint32_t e, uint32_t vec) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.d_q) | reinterpret_cast<uintptr_t>(a.d_k) |
                       reinterpret_cast<uintptr_t>(a.d_q_out) | reinterpret_cast<uintptr_t>(a.d_k_out);
  if (at % (vec * e)) return false;
  for (int64_t s : {a.q_token, a.q_head, a.k_token, a.k_head, a.qo_token, a.qo_head, a.ko_token, a.ko_head})
    if (s % int64_t(vec)) return false;
  // two chunks to a task inside the rotated part; the rest in whole chunks
  return a.rot % (2 * vec) == 0 && a.D % vec == 0;
}

template <typename T, int VEC, int KT>
int launch(const voom_qk_norm_rope_args& a, cudaStream_t s) {
  Rope P{};
  P.a = a;
  P.rot_tasks = a.rot / (2 * VEC);
  P.tasks = P.rot_tasks + ((a.D - a.rot) / VEC + 1) / 2;
  P.lanes = 1;
  while (P.lanes < 32 && P.lanes * KT < P.tasks) P.lanes *= 2;
  // as many CTAs as fill the GPU first; then more tokens to a CTA, so that
  // its threads all have an angle to make
  uint32_t tokens = 1;
  while (tokens < 8 && a.T >= tokens * 2 * 148 * 8 && tokens * (a.rot / 2) < kThreads) tokens *= 2;
  P.tokens = tokens;
  const uint32_t smem = tokens * (a.rot / 2) * uint32_t(sizeof(float2)) + 2 * a.D * uint32_t(sizeof(float));
  qk_norm_rope<T, VEC, KT><<<(a.T + tokens - 1) / tokens, kThreads, smem, s>>>(P);
  return cudaGetLastError() == cudaSuccess ? VOOM_OK : VOOM_E_CUDA;
}

// The widest chunk that every pointer, stride and boundary allows: 16 bytes
// for the usual layouts; 4 bytes or one value for odd strides and splits.
template <typename T>
int dispatch(const voom_qk_norm_rope_args& a, cudaStream_t s) {
  constexpr uint32_t e = uint32_t(sizeof(T));
  if constexpr (e == 2) {
    if (aligned(a, e, 8)) return launch<T, 8, 1>(a, s);
    if (aligned(a, e, 2)) return launch<T, 2, 4>(a, s);
  } else {
    if (aligned(a, e, 4)) return launch<T, 4, 2>(a, s);
  }
  return launch<T, 1, 8>(a, s);
}

}  // namespace

VOOM_API int voom_qk_norm_rope(const voom_qk_norm_rope_args* a, void* stream) {
  if (!a || !a->d_q || !a->d_k || !a->d_q_out || !a->d_k_out || !a->d_pos) return VOOM_E_INVALID_ARG;
  if (!a->D || a->rot > a->D || a->rot % 2 || (a->rot && !a->d_turns)) return VOOM_E_INVALID_ARG;
  if (a->D > kMaxD) return VOOM_E_UNSUPPORTED;
  if (a->type > VOOM_FP32 || a->w_type > VOOM_FP32) return VOOM_E_INVALID_ARG;
  if (uint64_t(a->hq) + a->hk > 65536u) return VOOM_E_UNSUPPORTED;
  if (!a->T || a->hq + a->hk == 0) return VOOM_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->type == VOOM_BF16) return dispatch<__nv_bfloat16>(*a, s);
  if (a->type == VOOM_FP16) return dispatch<__half>(*a, s);
  return dispatch<float>(*a, s);
}
