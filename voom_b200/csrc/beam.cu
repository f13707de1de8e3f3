// The best continuations of each request over its beams and the vocabulary.
//
//   score(i, t) = s_i + x_t - log sum exp x,   the `width` largest of a request
//
// Within a beam the order is the logits' own, so one pass over a row gives both
// what the denominator needs and the row's best `width`: beam_rows.  Each lane
// keeps a running maximum and sum; a warp keeps the best values it has met in a
// short list in shared memory and compares with the worst of them.  After the
// first values hardly any gets past that comparison, one vote for 32 values a
// lane, so the pass is bound by reading.  beam_join, a block per request, makes
// the beams' denominators and sorts what their rows kept.
//
// A list entry is one number: the value's bits in unsigned order, then the token
// counted from the end, so that no two are equal and the larger one is the better.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace {

constexpr uint32_t kThreads = 256, kWarps = kThreads / 32;
constexpr uint32_t kMaxWidth = 64, kMaxBeams = 64;
constexpr uint32_t kList = 128;      // entries of a warp's list, 32 of them for what one step may add
constexpr uint32_t kChunks = 4;      // 16-byte chunks of a lane under way
constexpr uint32_t kMaxSort = 8192;  // entries that beam_join sorts
constexpr float kLog2e = 1.4426950408889634f;

struct Beam {
  voom_beam_select_args a;
  uint64_t* best;  // rows x parts x width entries, 0: none
  double* sums;    // rows x parts: sum of exp(x - top)
  float* tops;     // rows x parts
  uint32_t parts;  // blocks of a row
  uint32_t sorted; // entries that beam_join sorts: a power of two
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x == 0.0f ? 0.0f : x);  // (-0 = 0)
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
__device__ __forceinline__ uint64_t entry_of(float x, uint32_t t) { return uint64_t(ordered(x)) << 32 | ~t; }

// The VEC values of 16 bytes.
template <typename T>
__device__ __forceinline__ void unpack(uint4 c, float* x);
template <>
__device__ __forceinline__ void unpack<float>(uint4 c, float* x) {
  x[0] = __uint_as_float(c.x);
  x[1] = __uint_as_float(c.y);
  x[2] = __uint_as_float(c.z);
  x[3] = __uint_as_float(c.w);
}
template <>
__device__ __forceinline__ void unpack<__nv_bfloat16>(uint4 c, float* x) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
template <>
__device__ __forceinline__ void unpack<__half>(uint4 c, float* x) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ float value(float x) { return x; }
__device__ __forceinline__ float value(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float value(__half x) { return __half2float(x); }

// sum += x with what the addition lost kept in `rest`; both are at least 0.
__device__ __forceinline__ void add_kept(float& sum, float& rest, float x) {
  const float t = sum + x;
  rest += fminf(sum, x) - (t - fmaxf(sum, x));
  sum = t;
}

// The n entries of a warp's list put in order, the first `width` kept.
__device__ __forceinline__ uint32_t prune(uint64_t* list, uint32_t n, uint32_t width) {
  const uint32_t lane = threadIdx.x & 31u;
  uint64_t mine[kList / 32];
  uint32_t rank[kList / 32] = {};
  __syncwarp();
#pragma unroll
  for (uint32_t i = 0; i < kList / 32; i++) mine[i] = lane + 32 * i < n ? list[lane + 32 * i] : 0;
  for (uint32_t j = 0; j < n; j++) {
    const uint64_t x = list[j];
#pragma unroll
    for (uint32_t i = 0; i < kList / 32; i++) rank[i] += x > mine[i];
  }
  __syncwarp();
#pragma unroll
  for (uint32_t i = 0; i < kList / 32; i++)
    if (lane + 32 * i < n && rank[i] < width) list[rank[i]] = mine[i];
  __syncwarp();
  return min(n, width);
}

// Block: part `part` of a row.  The row's 16-byte chunks are counted from the
// aligned address at or before its start; those at its ends are read value by value.
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) beam_rows(const __grid_constant__ Beam P) {
  constexpr uint32_t VEC = 16 / sizeof(T);
  __shared__ uint64_t s_list[kWarps][kList];
  __shared__ unsigned long long s_least;  // an entry that `width` of the block's are at least as good as
  __shared__ double s_sum[kWarps];
  __shared__ float s_top[kWarps];
  __shared__ uint32_t s_count[kWarps];
  const uint32_t row = blockIdx.x / P.parts, part = blockIdx.x - row * P.parts;
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, width = P.a.width, V = P.a.V;
  const uint32_t b = row / P.a.beams, i = row - b * P.a.beams;
  // a logit of -inf is never chosen
  constexpr uint64_t kNothing = uint64_t(0x007FFFFFu) << 32 | 0xFFFFFFFFu;
  if (tid == 0) s_least = kNothing;
  const bool alive = P.a.d_scores[row] > -INFINITY;  // (nor is anything of a beam that has no score)
  const T* x0 = static_cast<const T*>(P.a.d_logits) + int64_t(b) * P.a.l_b + int64_t(i) * P.a.l_i;
  const uint32_t skew = uint32_t(reinterpret_cast<uintptr_t>(x0) & 15u) / uint32_t(sizeof(T));
  const uint32_t chunks = alive ? (V + skew + VEC - 1) / VEC : 0u;
  const uint32_t steps = (chunks + 32 * kChunks - 1) / (32 * kChunks);  // of a warp
  const uint32_t first = uint32_t(uint64_t(steps) * part / P.parts), last = uint32_t(uint64_t(steps) * (part + 1) / P.parts);
  uint64_t* list = s_list[warp];
  uint32_t n = 0;
  uint64_t least = kNothing;
  float top = -INFINITY, sum = 0.0f, rest = 0.0f;  // sum + rest: of exp(x - top)
  bool begun = false;
  __syncthreads();
  for (uint32_t step = first + warp; step < last; step += kWarps) {
    float x[kChunks][VEC];
    uint4 raw[kChunks];
    const uint32_t c0 = step * 32 * kChunks + lane;
#pragma unroll
    for (uint32_t u = 0; u < kChunks; u++) {
      const uint32_t c = c0 + 32 * u, at = c * VEC;  // value `at - skew` is the chunk's first
      if (at >= skew && at + VEC <= V + skew) raw[u] = __ldcs(reinterpret_cast<const uint4*>(x0 - skew + at));
    }
    float best = -INFINITY;
#pragma unroll
    for (uint32_t u = 0; u < kChunks; u++) {
      const uint32_t c = c0 + 32 * u, at = c * VEC;
      if (at >= skew && at + VEC <= V + skew) {
        unpack<T>(raw[u], x[u]);
      } else {
#pragma unroll
        for (uint32_t e = 0; e < VEC; e++) {
          const uint32_t t = at + e - skew;  // (before the row: wraps to a large number)
          x[u][e] = t < V ? value(x0[t]) : -INFINITY;
        }
      }
#pragma unroll
      for (uint32_t e = 0; e < VEC; e++) best = fmaxf(best, x[u][e]);
    }
    if (best > top) {
      const float f = exp2_fast((top - best) * kLog2e);
      sum *= f;
      rest *= f;
      top = best;
    }
    const float base = top == -INFINITY ? 0.0f : top;
    float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t u = 0; u < kChunks; u++)
#pragma unroll
      for (uint32_t e = 0; e < VEC; e++) s4[e & 3u] += exp2_fast((x[u][e] - base) * kLog2e);
    add_kept(sum, rest, (s4[0] + s4[1]) + (s4[2] + s4[3]));
    // the list
    if (!begun) {
      begun = true;
      if (width <= 32) {  // as many lanes have a value at least as large as the width-th of their largest ones
        float y = best;
#pragma unroll
        for (uint32_t k = 2; k <= 32; k <<= 1)
#pragma unroll
          for (uint32_t d = k >> 1; d; d >>= 1) {
            const float o = __shfl_xor_sync(0xFFFFFFFFu, y, d);
            const bool up = (lane & k) != 0, low = (lane & d) == 0;  // descending where not up
            y = (low != up) ? fmaxf(y, o) : fminf(y, o);
          }
        const float w = __shfl_sync(0xFFFFFFFFu, y, width - 1);
        if (w > -INFINITY) {
          least = max(least, uint64_t(ordered(w)) << 32);
          if (lane == 0) atomicMax(&s_least, static_cast<unsigned long long>(least));
        }
      }
    }
    least = max(least, uint64_t(*const_cast<volatile unsigned long long*>(&s_least)));
    const float bar = fmaxf(unordered(uint32_t(least >> 32)), -FLT_MAX);
    if (__any_sync(0xFFFFFFFFu, best >= bar)) {
      uint32_t hits = 0;
#pragma unroll
      for (uint32_t u = 0; u < kChunks; u++)
#pragma unroll
        for (uint32_t e = 0; e < VEC; e++) hits |= uint32_t(x[u][e] >= bar) << (u * VEC + e);
      while (__any_sync(0xFFFFFFFFu, hits != 0)) {
        uint64_t mine = 0;
        if (hits) {
          const uint32_t k = __ffs(hits) - 1, t = (c0 + 32 * (k / VEC)) * VEC + k % VEC - skew;
          hits &= hits - 1;
          if (t < V) mine = entry_of(value(x0[t]), t);
        }
        const uint32_t takes = __ballot_sync(0xFFFFFFFFu, mine > least);
        if (mine > least) list[n + __popc(takes & ((1u << lane) - 1u))] = mine;
        n += __popc(takes);
        if (n > kList - 32) {
          n = prune(list, n, width);
          if (n == width) {
            least = max(least, list[width - 1]);
            if (lane == 0) atomicMax(&s_least, static_cast<unsigned long long>(least));
          }
        }
      }
    }
  }
  n = prune(list, n, width);
  // the warp's and the block's sums
  float all = top;
  for (int o = 16; o; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xFFFFFFFFu, all, o));
  // (a NaN value is not a maximum, but it is in the sum)
  double s = top == -INFINITY ? double(sum) : (double(sum) + double(rest)) * exp(double(top) - double(all));
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  if (lane == 0) {
    s_top[warp] = all;
    s_sum[warp] = s;
    s_count[warp] = n;
  }
  __syncthreads();
  const uint64_t out = uint64_t(row) * P.parts + part;
  if (tid == 0) {
    float m = -INFINITY;
    for (uint32_t w = 0; w < kWarps; w++) m = fmaxf(m, s_top[w]);
    double t = 0.0;
    for (uint32_t w = 0; w < kWarps; w++) t += s_top[w] == -INFINITY ? s_sum[w] : s_sum[w] * exp(double(s_top[w]) - double(m));
    P.tops[out] = m;
    P.sums[out] = t;
  }
  // the best of the warps' lists: an entry's rank is the number of better ones
  uint32_t total = 0;
  for (uint32_t w = 0; w < kWarps; w++) total += s_count[w];
  for (uint32_t k = tid; k < kWarps * width; k += kThreads) {
    const uint32_t w = k / width, j = k - w * width;
    if (j >= s_count[w]) continue;
    const uint64_t mine = s_list[w][j];
    uint32_t rank = 0;
    for (uint32_t v = 0; v < kWarps; v++)
      for (uint32_t q = 0; q < s_count[v] && s_list[v][q] > mine; q++) rank++;
    if (rank < width) P.best[out * width + rank] = mine;
  }
  for (uint32_t k = total + tid; k < width; k += kThreads) P.best[out * width + k] = 0;
}

__device__ __forceinline__ uint64_t ordered(double x) {
  const uint64_t u = uint64_t(__double_as_longlong(x == 0.0 ? 0.0 : x));
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double unordered(uint64_t k) {
  return __longlong_as_double(static_cast<long long>(k >> 63 ? k & 0x7FFFFFFFFFFFFFFFull : ~k));
}

__global__ void __launch_bounds__(kThreads) beam_join(const __grid_constant__ Beam P) {
  extern __shared__ uint64_t s_key[];  // the scores in unsigned order, 0: none; then the candidates' indexes
  __shared__ double s_lse[kMaxBeams];
  uint32_t* s_at = reinterpret_cast<uint32_t*>(s_key + P.sorted);
  const uint32_t b = blockIdx.x, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t beams = P.a.beams, width = P.a.width, parts = P.parts;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (uint32_t i = warp; i < beams; i += kWarps) {
    const uint64_t at = (uint64_t(b) * beams + i) * parts;
    float m = -INFINITY;
    for (uint32_t p = lane; p < parts; p += 32) m = fmaxf(m, P.tops[at + p]);
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    double s = 0.0;
    for (uint32_t p = lane; p < parts; p += 32) {
      const float t = P.tops[at + p];
      s += t == -INFINITY ? P.sums[at + p] : P.sums[at + p] * exp(double(t) - double(m));
    }
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    if (lane == 0) s_lse[i] = double(m) + log(s);
  }
  __syncthreads();
  const uint32_t per = parts * width;
  for (uint32_t k = tid; k < P.sorted; k += kThreads) {
    uint64_t key = 0;
    uint32_t at = 0xFFFFFFFFu;
    if (k < beams * per) {
      const uint32_t i = k / per;
      const uint64_t x = P.best[uint64_t(b) * beams * per + k];
      if (x) {
        const double z = double(P.a.d_scores[b * beams + i]) + (double(unordered(uint32_t(x >> 32))) - s_lse[i]);
        if (z > -INFINITY) {  // (not NaN)
          key = ordered(z);
          at = i * P.a.V + ~uint32_t(x);
        }
      }
    }
    s_key[k] = key;
    s_at[k] = at;
  }
  __syncthreads();
  for (uint32_t k = 2; k <= P.sorted; k <<= 1)
    for (uint32_t d = k >> 1; d; d >>= 1) {
      for (uint32_t q = tid; q < P.sorted / 2; q += kThreads) {
        const uint32_t lo = 2 * q - (q & (d - 1)), hi = lo + d;
        const uint64_t x = s_key[lo], y = s_key[hi];
        const uint32_t xa = s_at[lo], ya = s_at[hi];
        const bool behind = x < y || (x == y && xa > ya);  // `lo` belongs behind `hi`
        if (behind == ((lo & k) == 0) && (x != y || xa != ya)) {
          s_key[lo] = y;
          s_key[hi] = x;
          s_at[lo] = ya;
          s_at[hi] = xa;
        }
      }
      __syncthreads();
    }
  for (uint32_t k = tid; k < width; k += kThreads) {
    const uint64_t out = uint64_t(b) * width + k;
    const bool any = k < P.sorted && s_key[k] != 0;
    const uint32_t at = any ? s_at[k] : 0u, i = at / P.a.V;
    P.a.d_scores_out[out] = any ? float(unordered(s_key[k])) : -INFINITY;
    P.a.d_parents[out] = any ? int32_t(b * beams + i) : -1;
    P.a.d_tokens[out] = any ? int32_t(at - i * P.a.V) : -1;
  }
}

int check(const voom_beam_select_args* a) {
  if (!a || !a->d_logits || !a->d_scores || !a->d_scores_out || !a->d_parents || !a->d_tokens) return VOOM_E_INVALID_ARG;
  if (!a->beams || !a->V || !a->width || a->type > VOOM_FP32) return VOOM_E_INVALID_ARG;
  if (a->width > kMaxWidth || a->beams > kMaxBeams || uint64_t(a->beams) * a->V > 0x7FFFFFFFu || uint64_t(a->B) * a->beams > 0x7FFFFFFu)
    return VOOM_E_UNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(a->d_logits) % (a->type == VOOM_FP32 ? 4 : 2)) return VOOM_E_INVALID_ARG;
  return VOOM_OK;
}

uint64_t plan(Beam& P, void* scratch) {
  const voom_beam_select_args& a = P.a;
  const uint32_t step = 32 * kChunks * (a.type == VOOM_FP32 ? 4 : 8);
  const uint64_t rows = uint64_t(a.B) * a.beams, steps = (a.V + step - 1) / step + 1;
  // enough blocks for four to an SM, a step to each of a block's warps at least
  uint64_t parts = (592 + rows - 1) / std::max<uint64_t>(rows, 1);
  parts = std::min(parts, (steps + kWarps - 1) / kWarps);
  parts = std::min<uint64_t>(parts, std::max(1u, kMaxSort / (a.beams * a.width)));
  P.parts = uint32_t(std::max<uint64_t>(parts, 1));
  P.sorted = 2;
  while (P.sorted < a.beams * P.parts * a.width) P.sorted *= 2;
  uint8_t* base = static_cast<uint8_t*>(scratch);
  const uint64_t n = rows * P.parts;
  P.best = reinterpret_cast<uint64_t*>(base);
  P.sums = reinterpret_cast<double*>(base + 8 * n * a.width);
  P.tops = reinterpret_cast<float*>(base + 8 * n * (a.width + 1));
  return 8 * n * (a.width + 1) + 4 * n;
}

}  // namespace

VOOM_API uint64_t voom_beam_select_scratch_bytes(const voom_beam_select_args* a) {
  if (check(a) != VOOM_OK) return 0;
  Beam P{};
  P.a = *a;
  return plan(P, nullptr);
}

VOOM_API int voom_beam_select(const voom_beam_select_args* a, void* d_scratch, uint64_t bytes, void* stream) {
  const int rc = check(a);
  if (rc != VOOM_OK || !a->B) return rc;
  if (!d_scratch || (reinterpret_cast<uintptr_t>(d_scratch) & 15u)) return VOOM_E_INVALID_ARG;
  Beam P{};
  P.a = *a;
  if (plan(P, d_scratch) > bytes) return VOOM_E_CAPACITY;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint32_t grid = a->B * a->beams * P.parts;
  if (a->type == VOOM_BF16) beam_rows<__nv_bfloat16><<<grid, kThreads, 0, s>>>(P);
  else if (a->type == VOOM_FP16) beam_rows<__half><<<grid, kThreads, 0, s>>>(P);
  else beam_rows<float><<<grid, kThreads, 0, s>>>(P);
  if (cudaGetLastError() != cudaSuccess) return VOOM_E_CUDA;
  const uint32_t smem = P.sorted * 12;
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return VOOM_E_CUDA;
  if (!(allowed.load(std::memory_order_relaxed) >> (dev & 63) & 1u)) {
    if (cudaFuncSetAttribute(beam_join, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSort * 12) != cudaSuccess) {
      cudaGetLastError();
      return VOOM_E_CUDA;
    }
    allowed.fetch_or(uint64_t(1) << (dev & 63), std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute early{};
  cfg.gridDim = dim3(a->B);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, beam_join, P) == cudaSuccess) return VOOM_OK;
  cudaGetLastError();
  return VOOM_E_CUDA;
}
