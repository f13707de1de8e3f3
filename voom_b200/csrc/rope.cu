// Per-head RMS norm of queries and keys and the position rotation, one pass.
//
//   y = x * rsqrt(mean(x^2) + eps) * w,   then for each pair of the first `rot`
//   values  (a, b) -> factor * (a cos t - b sin t, a sin t + b cos t)
//
// The angle: `turns` holds the pair's turns per position as a 64-bit fraction,
// so position * turns modulo 2^64 is the fraction of a turn whatever the
// position (fp32 position * frequency is off by 0.01 rad at 10^5 already).
// Its top 32 bits are a signed half-turn count in [-1, 1): FP32 values take
// sincospif of it, 16-bit ones __sincosf of pi times it (exact to 2^-21, far
// below their rounding).
//
// Bound by HBM: every value is read and written once (2 bytes each way in
// BF16), about ten instructions per value.  A group of lanes takes a few heads
// of one token, two chunks of VEC values per lane: the two halves that a
// pair's members lie in ("half" layout), so that a pair never crosses lanes and
// the norm's sum is the only exchange.  A lane's place in the head is the same
// for all its heads, so cosines, sines and weights are made once and stay in
// registers.  What keeps HBM busy is the next three heads' values on their way
// into shared memory, where each lane reads back what it asked for itself.
// Measured: 16384 tokens x 40 heads of 128 in BF16, 57 us, 5.8 TB/s (89 % of
// what a copy reaches); without the read-ahead 94 us, with cosines, sines and
// weights in shared memory 84 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"
#include "rows.h"

namespace {

constexpr uint32_t kThreads = 128;
constexpr uint32_t kMaxD = 512;
constexpr uint32_t kDepth = 4;  // heads of a group under way, the one at work included

struct Rope {
  voom_qk_norm_rope_args a;
  uint32_t lanes;      // lanes per head: a power of two
  uint32_t rot_tasks;  // tasks in the rotated part (two chunks each)
  uint32_t tasks;      // tasks of a head
  uint32_t per, gq, g; // heads of a group; groups of a token's queries, and of all its heads
  uint32_t wide_w;     // weights of the values' type, chunk by chunk
  float one, inv_d;    // 1 for zero-centred weights; 1 / D
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

// Two adjacent values of a chunk as fp32, and back.
template <typename T>
__device__ __forceinline__ void unpack2(const T* p, float& a, float& b);
template <>
__device__ __forceinline__ void unpack2<__nv_bfloat16>(const __nv_bfloat16* p, float& a, float& b) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xFFFF0000u);
}
template <>
__device__ __forceinline__ void unpack2<__half>(const __half* p, float& a, float& b) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(p));
  a = f.x;
  b = f.y;
}
template <>
__device__ __forceinline__ void unpack2<float>(const float* p, float& a, float& b) {
  a = p[0];
  b = p[1];
}
__device__ __forceinline__ void repack2(__nv_bfloat16* p, float a, float b) {
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b);
}
__device__ __forceinline__ void repack2(__half* p, float a, float b) { *reinterpret_cast<__half2*>(p) = __floats2half2_rn(a, b); }
__device__ __forceinline__ void repack2(float* p, float a, float b) {
  p[0] = a;
  p[1] = b;
}

template <typename T, int VEC>
__device__ __forceinline__ Chunk<T, VEC> load_chunk(const T* p) {
  return *reinterpret_cast<const Chunk<T, VEC>*>(p);
}

template <typename T, int VEC>
__device__ __forceinline__ void store_chunk(T* p, const float (&x)[VEC]) {
  Chunk<T, VEC> c;
  if constexpr (VEC > 1) {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) repack2(&c.v[i], x[i], x[i + 1]);
  } else {
    c.v[0] = from_f<T>(x[0]);
  }
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
    const uint32_t rest = P.tasks - P.rot_tasks;
    c.i0 = P.a.rot + (task - P.rot_tasks) * VEC;
    c.i1 = c.i0 + rest * VEC;
    c.two = c.i1 < P.a.D;
  } else if (VEC == 1 && P.a.interleaved) {
    c.i0 = 2 * task;
    c.i1 = c.i0 + 1;
  } else {  // neighbouring lanes' chunks are neighbours
    c.i0 = task * VEC;
    c.i1 = c.i0 + P.a.rot / 2;
  }
  return c;
}

__device__ __forceinline__ void copy16(void* smem, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(uint32_t(__cvta_generic_to_shared(smem))), "l"(from) : "memory");
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
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 swap2(F2 x) {
  float a, b;
  take2(x, a, b);
  return make2(b, a);
}

template <int N>
__device__ __forceinline__ void load_turns(const uint64_t* p, uint64_t* x) {
  if constexpr (N > 1) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const ulonglong2 u = __ldg(reinterpret_cast<const ulonglong2*>(p + i));
      x[i] = u.x;
      x[i + 1] = u.y;
    }
  } else {
    x[0] = __ldg(p);
  }
}

// Weights of values i .. i + VEC (plus one, zero-centred).
template <typename T, int VEC>
__device__ __forceinline__ void load_weights(const Rope& P, const void* w, uint32_t i, float (&x)[VEC]) {
  if (P.wide_w) {
    const Chunk<T, VEC> c = load_chunk<T, VEC>(static_cast<const T*>(w) + i);
#pragma unroll
    for (int e = 0; e < VEC; e++) x[e] = to_f<T>(c.v[e]) + P.one;
  } else {
#pragma unroll
    for (int e = 0; e < VEC; e++) x[e] = weight(w, P.a.w_type, i + e) + P.one;
  }
}

// KT tasks of two chunks to a lane: task k of lane l is l + k * lanes.  With
// w the weights and c, s the pair's cosine and sine, a task's two chunks x, y
// become  r (x A + y B),  r (x C + y D)  in the half layout (A = w_x c, B =
// -w_y s, C = w_x s, D = w_y c), and each of them  r (x P + swapped x Q)  in the
// interleaved one.  Values that are not rotated take their own weight alone: a
// neighbour that is not finite must not reach them, not even times 0.
template <typename T, int VEC, int KT, bool INTER>
__global__ void __launch_bounds__(kThreads, KT * VEC == 8 ? 6 : 4) qk_norm_rope(const __grid_constant__ Rope P) {
  constexpr int N = VEC > 1 ? VEC / 2 : 1;        // register pairs of a chunk
  constexpr bool SWAP = INTER && VEC > 1;         // pairs lie within a chunk
  const voom_qk_norm_rope_args& a = P.a;
  const uint64_t group = (uint64_t(blockIdx.x) * kThreads + threadIdx.x) / P.lanes;
  const uint32_t lane = threadIdx.x & (P.lanes - 1);
  const uint32_t t = uint32_t(group / P.g), part = uint32_t(group - uint64_t(t) * P.g);
  const bool on = t < a.T, isq = part < P.gq;
  const uint32_t h0 = (isq ? part : part - P.gq) * P.per, heads = isq ? a.hq : a.hk;
  // lanes that have nothing to do go through the exchanges all the same
  const uint32_t count = on ? min(P.per, heads - h0) : 0u;
  const int64_t in_head = isq ? a.q_head : a.k_head, out_head = isq ? a.qo_head : a.ko_head;
  const T* src = nullptr;
  T* dst = nullptr;
  if (on) {
    src = (isq ? static_cast<const T*>(a.d_q) + int64_t(t) * a.q_token : static_cast<const T*>(a.d_k) + int64_t(t) * a.k_token) +
          int64_t(h0) * in_head;
    dst = (isq ? static_cast<T*>(a.d_q_out) + int64_t(t) * a.qo_token : static_cast<T*>(a.d_k_out) + int64_t(t) * a.ko_token) +
          int64_t(h0) * out_head;
  }
  Span c[KT];
#pragma unroll
  for (int k = 0; k < KT; k++) c[k] = span_of<VEC>(P, lane + k * P.lanes);
  constexpr bool WIDE = sizeof(T) * VEC == 16;  // else: values go straight to registers, one head at a time
  __shared__ Chunk<T, VEC> s_in[WIDE ? kDepth : 1][KT][2][kThreads];
  Chunk<T, VEC> nx[KT], ny[KT];
#pragma unroll
  for (int k = 0; k < KT; k++)
#pragma unroll
    for (int i = 0; i < VEC; i++) nx[k].v[i] = ny[k].v[i] = from_f<T>(0.0f);
  auto fetch = [&](uint32_t h) {  // head h of the group, if there is one
    if constexpr (WIDE) {
      if (h < count) {
#pragma unroll
        for (int k = 0; k < KT; k++) {
          if (c[k].has) copy16(&s_in[h % kDepth][k][0][threadIdx.x], src + c[k].i0);
          if (c[k].has && c[k].two) copy16(&s_in[h % kDepth][k][1][threadIdx.x], src + c[k].i1);
        }
        src += in_head;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  auto take = [&](uint32_t h) {
    if constexpr (WIDE) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
#pragma unroll
      for (int k = 0; k < KT; k++) {
        if (c[k].has) nx[k] = s_in[h % kDepth][k][0][threadIdx.x];
        if (c[k].has && c[k].two) ny[k] = s_in[h % kDepth][k][1][threadIdx.x];
      }
    } else if (h < count) {
#pragma unroll
      for (int k = 0; k < KT; k++) {
        if (c[k].has) nx[k] = load_chunk<T, VEC>(src + c[k].i0);
        if (c[k].has && c[k].two) ny[k] = load_chunk<T, VEC>(src + c[k].i1);
      }
      src += in_head;
    }
  };
#pragma unroll
  for (uint32_t h = 0; h + 1 < kDepth; h++) fetch(h);
  // the lane's coefficients
  const void* w = isq ? a.d_q_w : a.d_k_w;
  F2 ca[KT][N], cb[KT][N], cc[KT][N], cd[KT][N];
  if (on) {
    const int64_t pos = a.pos64 ? static_cast<const int64_t*>(a.d_pos)[t] : int64_t(static_cast<const int32_t*>(a.d_pos)[t]);
#pragma unroll
    for (int k = 0; k < KT; k++) {
      float wx[VEC], wy[VEC], co[VEC], si[VEC];
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        wx[i] = wy[i] = co[i] = 1.0f;
        si[i] = 0.0f;
      }
      if (w && c[k].has) {
        load_weights<T, VEC>(P, w, c[k].i0, wx);
        if (c[k].two) load_weights<T, VEC>(P, w, c[k].i1, wy);
      }
      if (c[k].has && c[k].rotated) {
        uint64_t turns[VEC];
        if constexpr (VEC == 1) {
          turns[0] = __ldg(a.d_turns + (INTER ? c[k].i0 / 2 : c[k].i0));
        } else if constexpr (SWAP) {  // N pairs of x, N of y
          load_turns<N>(a.d_turns + c[k].i0 / 2, turns);
          load_turns<N>(a.d_turns + c[k].i1 / 2, turns + N);
        } else {
          load_turns<VEC>(a.d_turns + c[k].i0, turns);
        }
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          const float x = float(int32_t((uint64_t(pos) * turns[i]) >> 32)) * (1.0f / 2147483648.0f);
          if (sizeof(T) == 4) sincospif(x, &si[i], &co[i]);
          else __sincosf(x * 3.14159265358979f, &si[i], &co[i]);
          co[i] *= a.factor;
          si[i] *= a.factor;
        }
      }
      if constexpr (SWAP) {  // pair i of a chunk is its values 2 i, 2 i + 1
#pragma unroll
        for (int i = 0; i < N; i++) {
          ca[k][i] = make2(wx[2 * i] * co[i], wx[2 * i + 1] * co[i]);
          cb[k][i] = make2(-wx[2 * i + 1] * si[i], wx[2 * i] * si[i]);
          cc[k][i] = make2(wy[2 * i] * co[N + i], wy[2 * i + 1] * co[N + i]);
          cd[k][i] = make2(-wy[2 * i + 1] * si[N + i], wy[2 * i] * si[N + i]);
        }
      } else if constexpr (VEC == 1) {
        ca[k][0] = make2(wx[0] * co[0], wx[0] * si[0]);
        cb[k][0] = make2(-wy[0] * si[0], wy[0] * co[0]);
      } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
          ca[k][i] = make2(wx[2 * i] * co[2 * i], wx[2 * i + 1] * co[2 * i + 1]);
          cb[k][i] = make2(-wy[2 * i] * si[2 * i], -wy[2 * i + 1] * si[2 * i + 1]);
          cc[k][i] = make2(wx[2 * i] * si[2 * i], wx[2 * i + 1] * si[2 * i + 1]);
          cd[k][i] = make2(wy[2 * i] * co[2 * i], wy[2 * i + 1] * co[2 * i + 1]);
        }
      }
    }
  }
  const bool norm = a.d_q_w || a.d_k_w;
  for (uint32_t h = 0; h < P.per; h++) {
    if (__all_sync(0xFFFFFFFFu, h >= count)) break;
    fetch(h + kDepth - 1);
    take(h);
    float x[KT][VEC], y[KT][VEC];
#pragma unroll
    for (int k = 0; k < KT; k++) {
      if constexpr (VEC > 1) {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
          unpack2<T>(&nx[k].v[i], x[k][i], x[k][i + 1]);
          unpack2<T>(&ny[k].v[i], y[k][i], y[k][i + 1]);
        }
      } else {
        x[k][0] = to_f<T>(nx[k].v[0]);
        y[k][0] = to_f<T>(ny[k].v[0]);
      }
    }
    float r = 1.0f;
    if (norm) {
      F2 acc = make2(0.0f, 0.0f), bcc = acc;
#pragma unroll
      for (int k = 0; k < KT; k++) {
        if constexpr (VEC > 1) {
#pragma unroll
          for (int i = 0; i < VEC; i += 2) {
            const F2 u = make2(x[k][i], x[k][i + 1]), v = make2(y[k][i], y[k][i + 1]);
            acc = fma2(u, u, acc);
            bcc = fma2(v, v, bcc);
          }
        } else {
          const F2 u = make2(x[k][0], y[k][0]);
          acc = fma2(u, u, acc);
        }
      }
      float s0, s1, s2, s3;
      take2(acc, s0, s1);
      take2(bcc, s2, s3);
      float sum = (s0 + s1) + (s2 + s3);
#pragma unroll
      for (uint32_t o = 16; o; o >>= 1)
        if (o < P.lanes) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
      if (w) r = rsqrtf(fmaf(sum, P.inv_d, a.eps));
    }
    if (h >= count) continue;
    const F2 rr = make2(r, r);
#pragma unroll
    for (int k = 0; k < KT; k++) {
      if (!c[k].has) continue;
      if constexpr (VEC == 1) {  // (x C + y D, x A + y B) at once
        F2 o;
        if (c[k].rotated) {
          o = fma2(make2(y[k][0], y[k][0]), cb[k][0], mul2(make2(x[k][0], x[k][0]), ca[k][0]));
        } else {
          float a0, a1, b0, b1;
          take2(ca[k][0], a0, a1);
          take2(cb[k][0], b0, b1);
          o = mul2(make2(x[k][0], y[k][0]), make2(a0, b1));
        }
        take2(mul2(o, rr), x[k][0], y[k][0]);
      } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
          const F2 u = mul2(make2(x[k][2 * i], x[k][2 * i + 1]), rr), v = mul2(make2(y[k][2 * i], y[k][2 * i + 1]), rr);
          F2 p = mul2(u, ca[k][i]), q = mul2(v, SWAP ? cc[k][i] : cd[k][i]);
          if (c[k].rotated) {
            if constexpr (SWAP) {
              p = fma2(swap2(u), cb[k][i], p);
              q = fma2(swap2(v), cd[k][i], q);
            } else {
              p = fma2(v, cb[k][i], p);
              q = fma2(v, cd[k][i], mul2(u, cc[k][i]));
            }
          }
          take2(p, x[k][2 * i], x[k][2 * i + 1]);
          take2(q, y[k][2 * i], y[k][2 * i + 1]);
        }
      }
      store_chunk<T, VEC>(dst + c[k].i0, x[k]);
      if (c[k].two) store_chunk<T, VEC>(dst + c[k].i1, y[k]);
    }
    dst += out_head;
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
  // a lane's coefficients cost about three heads' work: many heads to a group,
  // as long as the groups fill the GPU
  const uint64_t threads = uint64_t(a.T) * (a.hq + a.hk) * P.lanes;
  const uint32_t most = std::max(std::max(a.hq, a.hk), 1u);
  const uint32_t want = uint32_t(std::min<uint64_t>(8, std::max<uint64_t>(1, threads / (148 * 1024))));
  const uint32_t parts = (most + want - 1) / want;
  P.per = (most + parts - 1) / parts;
  P.gq = (a.hq + P.per - 1) / P.per;
  P.g = P.gq + (a.hk + P.per - 1) / P.per;
  P.one = a.zero_centered ? 1.0f : 0.0f;
  P.inv_d = 1.0f / float(a.D);
  P.wide_w = a.w_type == a.type && ((reinterpret_cast<uintptr_t>(a.d_q_w) | reinterpret_cast<uintptr_t>(a.d_k_w)) % (VEC * sizeof(T))) == 0;
  const uint64_t all = uint64_t(a.T) * P.g * P.lanes;
  const uint32_t grid = uint32_t((all + kThreads - 1) / kThreads);
  if (a.interleaved) qk_norm_rope<T, VEC, KT, true><<<grid, kThreads, 0, s>>>(P);
  else qk_norm_rope<T, VEC, KT, false><<<grid, kThreads, 0, s>>>(P);
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
  if (!a || (a->hq && (!a->d_q || !a->d_q_out)) || (a->hk && (!a->d_k || !a->d_k_out)) || (a->T && !a->d_pos)) return VOOM_E_INVALID_ARG;
  if (!a->D || a->rot > a->D || a->rot % 2 || (a->rot && !a->d_turns)) return VOOM_E_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(a->d_turns) & 15u) return VOOM_E_INVALID_ARG;
  if (a->D > kMaxD) return VOOM_E_UNSUPPORTED;
  if (a->type > VOOM_FP32 || a->w_type > VOOM_FP32) return VOOM_E_INVALID_ARG;
  if (uint64_t(a->hq) + a->hk > 65536u) return VOOM_E_UNSUPPORTED;
  if (!a->T || a->hq + a->hk == 0) return VOOM_OK;
  const int64_t T = a->T, D = a->D, e = a->type == VOOM_FP32 ? 4 : 2;
  const voom::Rows q{a->d_q, {T, a->hq, 1}, {a->q_token, a->q_head, 0}, D, e}, k{a->d_k, {T, a->hk, 1}, {a->k_token, a->k_head, 0}, D, e};
  const voom::Rows qo{a->d_q_out, {T, a->hq, 1}, {a->qo_token, a->qo_head, 0}, D, e}, ko{a->d_k_out, {T, a->hk, 1}, {a->ko_token, a->ko_head, 0}, D, e};
  if (!voom::separate(qo) || !voom::separate(ko) || !voom::disjoint(qo, ko) || !voom::disjoint(qo, k) || !voom::disjoint(ko, q) ||
      !(voom::same_place(qo, q) || voom::disjoint(qo, q)) || !(voom::same_place(ko, k) || voom::disjoint(ko, k)))
    return VOOM_E_OVERLAP;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->type == VOOM_BF16) return dispatch<__nv_bfloat16>(*a, s);
  if (a->type == VOOM_FP16) return dispatch<__half>(*a, s);
  return dispatch<float>(*a, s);
}
