// The best continuations of each request over its beams and the vocabulary.
//
//   score(i, t) = s_i + x_t - log sum exp x,   the `width` largest of a request
//
// Within a beam the order is the logits' own, so one pass over a row gives both
// what the denominator needs and where the row's best are: beam_rows.  A thread
// keeps a running maximum and sum and notes the largest of every 32 (FP32: 16)
// values.  The width-th largest of the block's 256 running maxima is a bar that
// `width` values reach at least, and hardly more do; only the groups whose largest
// reaches it are read again, and what reaches it there is put in order by
// counting.  beam_join makes the beams' denominators and finds the best of what their
// rows kept in the same way; where two beams come too close for fp32 sums, it makes
// theirs again in fp64.
//
// The logits are read once: HBM would be the bound.  Measured: 32 requests of 8 beams
// over 200019 FP16 tokens, 16 wanted: 36 us a call, 28 of it beam_rows (3.6 TB/s, 56 %
// of what a copy reaches).  A block of one row over 100010 values is bound by its own
// instructions, exponentials and maxima, with 512 of 592 places taken, then by the
// last look at its groups (4.5 us).  More blocks to a row make the joining cost more
// (39 to 54 us a call), lists kept by warps as they read cost the reading (75 us).  One
// request of 4 beams over 49152: 11.4 us, two launches' latency; FP32, 8 requests'
// first step over 131072 and 5 beams: 15.7 us.
//
// An entry is one number: the value's bits in unsigned order, then the token
// counted from the end, so that no two are equal and the larger one is the better.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"

namespace {

constexpr uint32_t kThreads = 256, kWarps = kThreads / 32;
constexpr uint32_t kMaxWidth = 64, kMaxBeams = 64;
constexpr uint32_t kChunks = 4;      // 16-byte chunks of a thread under way
constexpr uint32_t kSteps = 16;      // steps of a thread between two looks at the groups' maxima
constexpr uint32_t kStages = 2;      // steps of a thread under way, the one at work included
constexpr uint32_t kPerSm = 4;       // blocks to an SM: 57 KB of shared memory each
constexpr uint32_t kSlots = 148 * kPerSm;
constexpr uint32_t kFound = 512;     // groups, and entries, that a block holds
constexpr uint32_t kMaxSort = 8192;  // entries that beam_join sorts
constexpr uint32_t kMaxCount = 512;  // entries that it puts in order by counting instead
constexpr uint32_t kCandidate = 20;  // bytes of one there
constexpr float kNear = 2e-6f;       // scores of two beams that are this close are made again
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFarRef = 1048576.0f, kFar = kFarRef / 2;  // rows whose largest value is further from 0 are summed in fp64

struct Beam {
  voom_beam_select_args a;
  uint64_t* best;  // rows x parts x width entries, 0: none
  double* sums;    // rows x parts: sum of exp(x - top)
  float* tops;     // rows x parts
  double* exact;   // rows x slices: beam_join's sums over a slice
  uint32_t* came;  // B: blocks that have made theirs
  uint32_t parts;  // blocks of a row
  uint32_t slices; // blocks of a request in beam_join
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
// The largest of 16 bytes' values (not a NaN, if there is another).
template <typename T>
__device__ __forceinline__ float largest(const uint4 (&c)[kChunks]) {
  if constexpr (sizeof(T) == 4) {
    float m = -INFINITY;
#pragma unroll
    for (uint32_t u = 0; u < kChunks; u++)
      m = fmaxf(fmaxf(m, fmaxf(__uint_as_float(c[u].x), __uint_as_float(c[u].y))), fmaxf(__uint_as_float(c[u].z), __uint_as_float(c[u].w)));
    return m;
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    auto two = [](uint32_t w) { return *reinterpret_cast<const T2*>(&w); };
    T2 m = two(c[0].x);
#pragma unroll
    for (uint32_t u = 0; u < kChunks; u++) {
      if (u) m = __hmax2(m, two(c[u].x));
      m = __hmax2(__hmax2(m, two(c[u].y)), __hmax2(two(c[u].z), two(c[u].w)));
    }
    return fmaxf(__low2float(m), __high2float(m));
  }
}

__device__ __forceinline__ void copy16(void* smem, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(uint32_t(__cvta_generic_to_shared(smem))), "l"(from) : "memory");
}

// Two bits patterns of -infinity, or one.
template <typename T>
constexpr uint32_t kNone = std::is_same<T, float>::value ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;

__device__ __forceinline__ float value(float x) { return x; }
__device__ __forceinline__ float value(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float value(__half x) { return __half2float(x); }

// sum += x with what the addition lost kept in `rest`; both are at least 0.
__device__ __forceinline__ void add_kept(float& sum, float& rest, float x) {
  const float t = sum + x;
  rest += fminf(sum, x) - (t - fmaxf(sum, x));
  sum = t;
}

// Two fp32 values in a register pair: one instruction works on both.
__device__ __forceinline__ uint64_t make2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void take2(uint64_t x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// 2^-n of a whole number n of at least 1.
__device__ __forceinline__ float down2(float n) { return n < 126.0f ? __int_as_float((127 - int(n)) << 23) : 0.0f; }

template <typename X>
struct Bar {
  X tops[kWarps][32];  // the warps' values, falling
  X at;
};

struct RowShared {
  uint4 raw[kStages][kChunks][kThreads];  // a thread's values on their way; it reads its own alone
  float best[kSteps][kThreads];  // the groups' largest values
  Bar<float> bar;
  uint64_t found[kFound];        // entries that reached the bar
  uint32_t groups[kFound];       // step, thread
  uint64_t most[kWarps];
  double sum[kWarps];
  float top[kWarps];
  uint32_t n_groups, n;
};

__device__ __forceinline__ float lane_xor(float x, uint32_t d) { return __shfl_xor_sync(0xFFFFFFFFu, x, d); }
__device__ __forceinline__ uint64_t lane_xor(uint64_t x, uint32_t d) {
  return uint64_t(__shfl_xor_sync(0xFFFFFFFFu, static_cast<unsigned long long>(x), d));
}

// The largest of the block's x; all threads call it.
__device__ __forceinline__ uint64_t block_max(RowShared& sh, uint64_t x) {
  for (uint32_t o = 16; o; o >>= 1) x = max(x, lane_xor(x, o));
  __syncthreads();
  if ((threadIdx.x & 31u) == 0) sh.most[threadIdx.x >> 5] = x;
  __syncthreads();
  for (uint32_t w = 0; w < kWarps; w++) x = max(x, sh.most[w]);
  return x;
}

// The width-th largest of the threads' values (of equal ones, each counts).  Every warp sorts its own; a value's rank among the others' is
// found by halving.
template <typename X>
__device__ __forceinline__ X find_bar(Bar<X>& sh, X y, uint32_t width) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
#pragma unroll
  for (uint32_t k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (uint32_t d = k >> 1; d; d >>= 1) {
      const X o = lane_xor(y, d);
      const bool up = (lane & k) != 0, low = (lane & d) == 0;  // falling where not up
      y = (low != up) == (y < o) ? o : y;
    }
  sh.tops[warp][lane] = y;
  __syncthreads();
  uint32_t rank = lane;
#pragma unroll
  for (uint32_t v = 0; v < kWarps; v++) {
    if (v == warp) continue;
    uint32_t at = 0;  // values of warp v that come before y
#pragma unroll
    for (uint32_t d = 16; d; d >>= 1) {
      const X o = sh.tops[v][at + d - 1];
      if (o > y || (o == y && v < warp)) at += d;
    }
    if (at == 31) {
      const X o = sh.tops[v][31];
      at += o > y || (o == y && v < warp);
    }
    rank += at;
  }
  if (rank == width - 1) sh.at = y;
  __syncthreads();
  return sh.at;
}

// A part's values once more, for what is rare: out of the way of beam_rows' registers.
template <typename T>
struct Part {
  const T* x0;
  uint64_t t0, t1;  // of the row's chunks
  uint32_t skew, V;

  template <typename F>
  __device__ __forceinline__ void each(F f) const {  // (-inf for what is not the row's)
    constexpr uint32_t kDeep = 8;
    for (uint64_t at = t0 + threadIdx.x; at < t1; at += kDeep * kThreads) {
      float x[kDeep];
#pragma unroll
      for (uint32_t u = 0; u < kDeep; u++) {
        const uint32_t t = uint32_t(at) + u * kThreads - skew;
        x[u] = at + u * kThreads < t1 && t < V ? value(x0[t]) : -INFINITY;
      }
#pragma unroll
      for (uint32_t u = 0; u < kDeep; u++) f(uint32_t(at) + u * kThreads - skew, x[u]);
    }
  }
};

// A thread's part of the sum of e^(x - top).
template <typename T>
__device__ __noinline__ double sum_far(const Part<T>& p, float top) {
  double s = 0.0;
  p.each([&](uint32_t, float x) { s += exp(double(x) - double(top)); });
  return s;
}

// The part's best entries where more reached the bar than a block holds: values that
// tie, as a mask of the type's lowest value does wherever fewer than `width` tokens are
// left, or that lie under few threads.  The threads' best entries, every 256th token to
// one, give a bar that ties cannot crowd: 32 requests of 8 such beams over 200019 values,
// 16 wanted, 248 us a call (2390 one after another; without the mask 48, L2 flushed).
template <typename T>
__device__ __noinline__ void best_again(RowShared& sh, const Part<T>& p, uint32_t width) {
  const uint32_t tid = threadIdx.x;
  Bar<uint64_t>& bar = *reinterpret_cast<Bar<uint64_t>*>(sh.raw);
  static_assert(sizeof(Bar<uint64_t>) <= sizeof(sh.raw), "nothing is on its way there any more");
  auto entry = [&](uint32_t t, float x) { return x > -INFINITY ? entry_of(x, t) : 0; };
  uint64_t most = 0;
  p.each([&](uint32_t t, float x) { most = max(most, entry(t, x)); });
  __syncthreads();  // sh.n and sh.raw are read
  if (tid == 0) sh.n = 0;
  const uint64_t reach = max(find_bar(bar, most, width), uint64_t(1));
  p.each([&](uint32_t t, float x) {
    const uint64_t y = entry(t, x);
    if (y < reach) return;
    const uint32_t at = atomicAdd(&sh.n, 1u);
    if (at < kFound) sh.found[at] = y;
  });
  __syncthreads();
  if (sh.n <= kFound) return;
  // under few threads again: one after another, each the best after the last
  uint64_t last_one = ~0ull;
  uint32_t k = 0;
  for (; k < width; k++) {
    uint64_t mine = 0;
    p.each([&](uint32_t t, float x) {
      const uint64_t y = entry(t, x);
      if (y < last_one) mine = max(mine, y);
    });
    last_one = block_max(sh, mine);
    if (!last_one) break;
    if (tid == 0) sh.found[k] = last_one;
  }
  if (tid == 0) sh.n = k;
  __syncthreads();
}

// Block: part `part` of a row.  The row's 16-byte chunks are counted from the
// aligned address at or before its start; those at its ends are read value by value.
template <typename T>
__global__ void __launch_bounds__(kThreads, kPerSm) beam_rows(const __grid_constant__ Beam P) {
  constexpr uint32_t VEC = 16 / sizeof(T), GROUP = kChunks * VEC;
  extern __shared__ __align__(16) uint8_t smem[];
  RowShared& sh = *reinterpret_cast<RowShared*>(smem);
  const uint32_t row = blockIdx.x / P.parts, part = blockIdx.x - row * P.parts;
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, width = P.a.width, V = P.a.V;
  const uint32_t b = row / P.a.beams, i = row - b * P.a.beams;
  const uint64_t out = uint64_t(row) * P.parts + part;
  if (i == 0 && part == 0 && tid == 0) P.came[b] = 0;
  if (!(P.a.d_scores[row] > -INFINITY)) {  // nothing of a beam that has no score is chosen
    for (uint32_t k = tid; k < width; k += kThreads) P.best[out * width + k] = 0;
    if (tid == 0) {
      P.tops[out] = -INFINITY;
      P.sums[out] = 0.0;
    }
    return;
  }
  if (tid == 0) sh.n = 0;
  const T* x0 = static_cast<const T*>(P.a.d_logits) + int64_t(b) * P.a.l_b + int64_t(i) * P.a.l_i;
  const uint32_t skew = uint32_t(reinterpret_cast<uintptr_t>(x0) & 15u) / uint32_t(sizeof(T));
  const uint32_t steps = ((V + skew + VEC - 1) / VEC + 32 * kChunks - 1) / (32 * kChunks);  // of a warp
  const uint32_t first = uint32_t(uint64_t(steps) * part / P.parts), last = uint32_t(uint64_t(steps) * (part + 1) / P.parts);
  // value `at - skew` is the first of the chunk at `at`
  auto whole = [&](uint32_t at) { return at >= skew && at + VEC <= V + skew; };
  auto fetch = [&](uint32_t step, uint32_t slot) {
    if (step < last) {
#pragma unroll
      for (uint32_t u = 0; u < kChunks; u++) {
        const uint32_t at = (step * 32 * kChunks + lane + 32 * u) * VEC;
        if (whole(at)) {
          copy16(&sh.raw[slot][u][tid], x0 - skew + at);
        } else {  // at the row's ends: value by value, and -inf for what is not the row's
          T x[VEC];
#pragma unroll
          for (uint32_t e = 0; e < VEC; e++) {
            const uint32_t t = at + e - skew;  // (before the row: wraps to a large number)
            const uint32_t none = kNone<T>;
            x[e] = t < V ? x0[t] : *reinterpret_cast<const T*>(&none);
          }
          sh.raw[slot][u][tid] = *reinterpret_cast<const uint4*>(x);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // sum + rest: of 2^(x log2 e - ref).  `ref` is a whole number, so that raising it scales both
  // exactly, however often a row rises, and x log2 e - ref is rounded once, as small as it is
  float top = -INFINITY, ref = -INFINITY, sum = 0.0f, rest = 0.0f;
  bool many = false;
  uint32_t slot = 0;
#pragma unroll
  for (uint32_t k = 0; k + 1 < kStages; k++) fetch(first + k * kWarps + warp, k);
  __syncthreads();  // sh.n is set
  for (uint32_t step0 = first; step0 < last; step0 += kSteps * kWarps) {
#pragma unroll 1
    for (uint32_t k = 0; k < kSteps && step0 + k * kWarps < last; k++) {
      const uint32_t step = step0 + k * kWarps + warp;
      float best = -INFINITY;
      if (step < last) {
        fetch(step + (kStages - 1) * kWarps, slot == 0 ? kStages - 1 : slot - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        uint4 raw[kChunks];
#pragma unroll
        for (uint32_t u = 0; u < kChunks; u++) raw[u] = sh.raw[slot][u][tid];
        slot = slot + 1 == kStages ? 0 : slot + 1;
        best = largest<T>(raw);
        if (best > top) {
          top = best;
          const float r = fminf(fmaxf(ceilf(best * kLog2e), -kFarRef), kFarRef);
          if (r > ref) {
            const float f = down2(r - ref);
            sum *= f;
            rest *= f;
            ref = r;
          }
        }
        const float base = ref == -INFINITY ? 0.0f : ref;
        const uint64_t nb = make2(-base, -base), l2 = make2(kLog2e, kLog2e);
        uint64_t acc[2] = {0, 0};
#pragma unroll
        for (uint32_t u = 0; u < kChunks; u++) {
          float x[VEC];
          unpack<T>(raw[u], x);
#pragma unroll
          for (uint32_t e = 0; e < VEC; e += 2) {
            float p, q;
            take2(fma2(make2(x[e], x[e + 1]), l2, nb), p, q);
            acc[e >> 1 & 1] = add2(acc[e >> 1 & 1], make2(exp2_fast(p), exp2_fast(q)));
          }
        }
        float s0, s1;
        take2(add2(acc[0], acc[1]), s0, s1);
        add_kept(sum, rest, s0 + s1);
      }
      sh.best[k][tid] = best;
    }
    if (tid == 0) sh.n_groups = 0;
    const float bar = fmaxf(find_bar(sh.bar, top, width), -FLT_MAX);  // (a logit of -inf is never chosen)
    const uint32_t rounds = min(kSteps, (last - step0 + kWarps - 1) / kWarps);
#pragma unroll 4
    for (uint32_t k = 0; k < rounds; k++)
      if (sh.best[k][tid] >= bar) {
        const uint32_t g = atomicAdd(&sh.n_groups, 1u);
        if (g < kFound) sh.groups[g] = (step0 + k * kWarps + warp) * 32 + lane;
      }
    __syncthreads();
    many |= sh.n_groups > kFound;
    const uint32_t groups = min(sh.n_groups, kFound);
    for (uint32_t q = warp * (32 / GROUP); q < groups; q += kWarps * (32 / GROUP)) {
      const uint32_t mine = q + lane / GROUP, e = lane % GROUP;
      if (mine >= groups) continue;
      const uint32_t g = sh.groups[mine], t = ((g >> 5) * 32 * kChunks + (g & 31u) + 32 * (e / VEC)) * VEC + e % VEC - skew;
      if (t >= V) continue;
      const float x = value(x0[t]);
      if (x >= bar) {
        const uint32_t at = atomicAdd(&sh.n, 1u);
        if (at < kFound) sh.found[at] = entry_of(x, t);
      }
    }
    __syncthreads();
  }
  const Part<T> part_of{x0, uint64_t(first) * 32 * kChunks * VEC, uint64_t(last) * 32 * kChunks * VEC, skew, V};
  if (many || sh.n > kFound) best_again(sh, part_of, width);
  // the warps' sums
  float all = top;
  for (int o = 16; o; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xFFFFFFFFu, all, o));
  // (a NaN value is not a maximum, but it is in the sum; far below the block's largest the sum is 0, far above made anew)
  double s = fabsf(top) > kFar ? double(sum) : (double(sum) + double(rest)) * exp2(double(ref) - double(all) * double(kLog2e));
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  if (lane == 0) {
    sh.top[warp] = all;
    sh.sum[warp] = s;
  }
  __syncthreads();
  float most = -INFINITY;
  for (uint32_t w = 0; w < kWarps; w++) most = fmaxf(most, sh.top[w]);
  if (fabsf(most) > kFar && fabsf(most) < INFINITY) {  // fp32 holds little of such an exponent
    double far = sum_far(part_of, most);
    for (int o = 16; o; o >>= 1) far += __shfl_xor_sync(0xFFFFFFFFu, far, o);
    __syncthreads();
    if (lane == 0) {
      sh.top[warp] = most;
      sh.sum[warp] = far;
    }
    __syncthreads();
  }
  if (warp == 0) {
    const float t = lane < kWarps ? sh.top[lane] : -INFINITY;
    float m = t;
    for (int o = kWarps / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    double y = lane < kWarps ? sh.sum[lane] : 0.0;
    if (t > -INFINITY) y *= exp(double(t) - double(m));
    for (int o = kWarps / 2; o; o >>= 1) y += __shfl_xor_sync(0xFFFFFFFFu, y, o);
    if (lane == 0) {
      P.tops[out] = m;
      P.sums[out] = y;
    }
  }
  const uint32_t n = sh.n;
  for (uint32_t k = tid; k < n; k += kThreads) {
    const uint64_t mine = sh.found[k];
    uint32_t rank = 0;
    for (uint32_t q = 0; q < n; q++) rank += sh.found[q] > mine;
    if (rank < width) P.best[out * width + rank] = mine;
  }
  for (uint32_t k = n + tid; k < width; k += kThreads) P.best[out * width + k] = 0;
}

// y = e^y for -inf <= y <= 0, in fp64, N at a time step by step: one alone waits for each
// result.  y = n ln 2 + r with ln 2 as its first 32 bits and the rest (Cody and Waite), and
// Taylor's series of e^r, |r| <= 0.347: the 14th term is below 5e-18.
template <int N>
__device__ __forceinline__ void exp_down(double (&y)[N]) {
  constexpr double whole = 6755399441055744.0;  // 1.5 * 2^52: what is added to it is rounded, and stands in the low word
  constexpr double hi = 2977044472.0 / 4294967296.0, lo = -4.2009150726810846e-11;
  constexpr double f[14] = {1.0,       1.0,        2.0,         6.0,          24.0,         120.0,         720.0,
                            5040.0,    40320.0,    362880.0,    3628800.0,    39916800.0,   479001600.0,   6227020800.0};
  double p[N];
  int n[N];
#pragma unroll
  for (int i = 0; i < N; i++) {
    const double t = fma(fmax(y[i], -700.0), 1.4426950408889634, whole);
    n[i] = __double2loint(t);
    y[i] = fma(whole - t, lo, fma(whole - t, hi, fmax(y[i], -700.0)));
    p[i] = 1.0 / f[13];
  }
#pragma unroll
  for (int k = 12; k >= 0; k--)
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = fma(p[i], y[i], 1.0 / f[k]);
#pragma unroll
  for (int i = 0; i < N; i++) y[i] = __hiloint2double(__double2hiint(p[i]) + (n[i] << 20), __double2loint(p[i]));
}

struct JoinShared {
  double lse[kMaxBeams];  // NaN: the beam has no candidates
  double part[kWarps];
  float score[kMaxBeams], top[kMaxBeams];
  Bar<float> bar;
  uint32_t n;
  unsigned long long near;  // beams whose candidates are too close to others'
  uint32_t last;
};

// Sum of e^(x - top) over tokens [t0, t1) of a row, in fp64 and an order that only the
// tokens decide; the whole block calls it, thread 0 gets it.
template <typename T>
__device__ __noinline__ double sum_exactly(JoinShared& sh, const T* row, double top, uint32_t t0, uint32_t t1) {
  constexpr int kDeep = 8;
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  double s = 0.0;
  for (uint32_t at = t0 + tid; at - tid < t1; at += kDeep * kThreads) {
    T x[kDeep];  // all under way together
    double y[kDeep];
#pragma unroll
    for (int u = 0; u < kDeep; u++) x[u] = at + u * kThreads < t1 ? row[at + u * kThreads] : T(-INFINITY);
#pragma unroll
    for (int u = 0; u < kDeep; u++) y[u] = double(value(x[u])) - top;
    exp_down(y);
#pragma unroll
    for (int u = 0; u < kDeep; u++) s += y[u];
  }
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  __syncthreads();  // the last row's parts are read
  if (lane == 0) sh.part[warp] = s;
  __syncthreads();
  s = 0.0;
  for (uint32_t w = 0; w < kWarps; w++) s += sh.part[w];
  return s;
}

// Makes the denominators of the beams in `near` again; false: another block goes on.
__device__ __noinline__ bool settle(const Beam& P, JoinShared& sh, uint32_t b, uint32_t slice, unsigned long long near) {
  const uint32_t tid = threadIdx.x, beams = P.a.beams;
  const uint32_t V = P.a.V, t0 = uint32_t(uint64_t(V) * slice / P.slices), t1 = uint32_t(uint64_t(V) * (slice + 1) / P.slices);
  for (unsigned long long left = near; left; left &= left - 1) {
    const uint32_t i = uint32_t(__ffsll(static_cast<long long>(left))) - 1;
    const int64_t row = int64_t(b) * P.a.l_b + int64_t(i) * P.a.l_i;
    const double top = double(sh.top[i]);
    double s;
    if (P.a.type == VOOM_BF16) s = sum_exactly(sh, static_cast<const __nv_bfloat16*>(P.a.d_logits) + row, top, t0, t1);
    else if (P.a.type == VOOM_FP16) s = sum_exactly(sh, static_cast<const __half*>(P.a.d_logits) + row, top, t0, t1);
    else s = sum_exactly(sh, static_cast<const float*>(P.a.d_logits) + row, top, t0, t1);
    if (tid == 0) P.exact[(uint64_t(b) * beams + i) * P.slices + slice] = s;
  }
  if (tid == 0) {
    __threadfence();
    sh.last = atomicAdd(P.came + b, 1u) + 1 == P.slices;
    __threadfence();
  }
  __syncthreads();
  if (!sh.last) return false;
  for (unsigned long long left = near; left; left &= left - 1) {
    const uint32_t i = uint32_t(__ffsll(static_cast<long long>(left))) - 1;
    if (tid != i) continue;
    double s = 0.0;
    for (uint32_t g = 0; g < P.slices; g++) s += __ldcg(P.exact + (uint64_t(b) * beams + i) * P.slices + g);
    sh.lse[i] = double(sh.top[i]) + log(s);
  }
  __syncthreads();
  return true;
}

// The candidates' scores come from beam_rows' sums, which are off by 8e-7 of themselves
// at most (ex2 2^-22, a group's additions 9 * 2^-24): enough for all but candidates of
// two beams that are closer than twice that.  Such beams' denominators are made again in
// fp64 (settle).  That is rare (one of twelve calls of 32 requests of 8 beams over 200019
// FP16 values, for one pair), but a row takes one block long: several blocks do the same
// for a request, each sums a slice of the rows if that is called for, and the last to
// come adds the slices up (nothing waits).  Without it the first block is done.  The pair
// 38 us more, all 256 rows of equal beams 142; the blocks that are not needed 1 us.
__global__ void __launch_bounds__(kThreads) beam_join(const __grid_constant__ Beam P) {
  extern __shared__ double s_z[];      // the candidates' scores; their entries, their beams
  __shared__ JoinShared sh;
  uint64_t* s_entry = reinterpret_cast<uint64_t*>(s_z + P.sorted);
  uint32_t* s_beam = reinterpret_cast<uint32_t*>(s_entry + P.sorted);
  const uint32_t b = blockIdx.x / P.slices, slice = blockIdx.x - b * P.slices, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t beams = P.a.beams, width = P.a.width, parts = P.parts, per = parts * width, all = beams * per;
  if (tid == 0) {
    sh.n = 0;
    sh.near = 0;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint64_t* best = P.best + uint64_t(b) * all;
  uint64_t ahead = tid < all ? best[tid] : 0;  // on its way while the denominators are made
  for (uint32_t i = warp; i < beams; i += kWarps) {
    const uint64_t at = (uint64_t(b) * beams + i) * parts;
    const float score = P.a.d_scores[b * beams + i];
    float m = -INFINITY;
    double s = 0.0;
    for (uint32_t p = lane; p < parts; p += 32) {
      const float t = P.tops[at + p];
      const double y = P.sums[at + p];
      if (t > m) {
        s = s * exp(double(m) - double(t)) + y;
        m = t;
      } else {
        s += t == -INFINITY ? y : y * exp(double(t) - double(m));
      }
    }
    float top = m;
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    if (m > -INFINITY && m != top) s *= exp(double(m) - double(top));
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    if (lane == 0) {
      sh.lse[i] = top > -INFINITY ? double(top) + log(s) : double(NAN);
      sh.score[i] = score;
      sh.top[i] = top;
    }
  }
  __syncthreads();
  // a candidate's score; NaN: it is none
  auto score_of = [&](uint32_t i, uint64_t x) {
    return x ? double(sh.score[i]) + (double(unordered(uint32_t(x >> 32))) - sh.lse[i]) : double(NAN);
  };
  float most = -INFINITY;
  for (uint32_t k = tid; k < all; k += kThreads) most = fmaxf(most, float(score_of(k / per, k == tid ? ahead : best[k])));
  float bar = find_bar(sh.bar, most, width);  // `width` candidates reach it, if there are as many
  // (and those that may be as good: what two scores are off, and the rounding to fp32)
  if (fabsf(bar) < INFINITY) bar -= 1.25f * kNear + fabsf(bar) * 0x1p-22f;
  for (uint32_t k = tid; k < all; k += kThreads) {
    const uint64_t x = k == tid ? ahead : best[k];
    const double z = score_of(k / per, x);
    if (z > -INFINITY && float(z) >= bar) {
      const uint32_t at = atomicAdd(&sh.n, 1u);
      s_z[at] = z;
      s_entry[at] = x;
      s_beam[at] = k / per;
    }
  }
  // equal scores: the lower beam, then the larger logit, then the lower token
  auto first = [&](uint32_t q, uint32_t k) { return s_beam[q] != s_beam[k] ? s_beam[q] < s_beam[k] : s_entry[q] > s_entry[k]; };
  auto put = [&](uint32_t rank, uint32_t k, bool some) {
    const uint64_t out = uint64_t(b) * width + rank;
    P.a.d_scores_out[out] = some ? float(s_z[k]) : -INFINITY;
    P.a.d_parents[out] = some ? int32_t(b * beams + s_beam[k]) : -1;
    P.a.d_tokens[out] = some ? int32_t(~uint32_t(s_entry[k])) : -1;
  };
  __syncthreads();
  const uint32_t n = sh.n;
  uint32_t sorted = 2;
  while (sorted < n) sorted *= 2;
  for (bool again = false;; again = true) {
    constexpr uint32_t kMine = kMaxCount / kThreads;
    uint32_t rank[kMine];
    if (n <= kMaxCount) {  // a candidate's place is the number of better ones
#pragma unroll
      for (uint32_t c = 0; c < kMine; c++) {
        const uint32_t k = tid + c * kThreads;
        rank[c] = width;
        if (k >= n) continue;
        const double z = s_z[k];
        uint32_t r = 0;
        unsigned long long near = 0;
#pragma unroll 4
        for (uint32_t q = 0; q < n; q++) {
          const double d = s_z[q] - z;
          r += d > 0.0;
          if (!(fabs(d) > double(kNear)) && q != k) {  // seldom (infinite ones are equal)
            if (!(fabs(d) > 0.0)) r += first(q, k);
            if (s_beam[q] != s_beam[k]) near |= 1ull << s_beam[q] | 1ull << s_beam[k];
          }
        }
        if (near && r < width && !again) atomicOr(&sh.near, near);
        rank[c] = r;
      }
    } else {
      for (uint32_t k = n + tid; k < sorted; k += kThreads) {
        s_z[k] = -INFINITY;
        s_beam[k] = kMaxBeams;
        s_entry[k] = sorted - k;
      }
      __syncthreads();
      for (uint32_t k = 2; k <= sorted; k <<= 1)
        for (uint32_t d = k >> 1; d; d >>= 1) {
          for (uint32_t q = tid; q < sorted / 2; q += kThreads) {
            const uint32_t lo = 2 * q - (q & (d - 1)), hi = lo + d;
            const double z = s_z[lo], y = s_z[hi];
            if ((z != y ? z < y : first(hi, lo)) == ((lo & k) == 0)) {  // (no two are equal)
              const uint64_t x = s_entry[lo];
              const uint32_t i = s_beam[lo];
              s_z[lo] = y;
              s_entry[lo] = s_entry[hi];
              s_beam[lo] = s_beam[hi];
              s_z[hi] = z;
              s_entry[hi] = x;
              s_beam[hi] = i;
            }
          }
          __syncthreads();
        }
      if (!again)  // (of two beams with close candidates, some are neighbours)
        for (uint32_t k = tid; k + 1 < n; k += kThreads)
          if (s_beam[k] != s_beam[k + 1] && !(s_z[k] - s_z[k + 1] > double(kNear))) atomicOr(&sh.near, 1ull << s_beam[k] | 1ull << s_beam[k + 1]);
    }
    __syncthreads();
    const unsigned long long near = again ? 0ull : sh.near;
    if (!near) {
      if (!again && slice) return;
      if (n <= kMaxCount) {
#pragma unroll
        for (uint32_t c = 0; c < kMine; c++)
          if (rank[c] < width) put(rank[c], tid + c * kThreads, true);
        for (uint32_t k = n + tid; k < width; k += kThreads) put(k, 0, false);
      } else {
        for (uint32_t k = tid; k < width; k += kThreads) put(k, k, true);  // (n > kMaxCount >= width)
      }
      return;
    }
    if (!settle(P, sh, b, slice, near)) return;
    for (uint32_t k = tid; k < n; k += kThreads) s_z[k] = score_of(s_beam[k], s_entry[k]);
    __syncthreads();
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
  // as many blocks as the SMs hold at once (a second wave of them, with half the
  // row each: 39 us against 32), a step to each of a block's warps at least
  uint64_t parts = std::max<uint64_t>(1, kSlots / std::max<uint64_t>(rows, 1));
  parts = std::min(parts, (steps + kWarps - 1) / kWarps);
  parts = std::min<uint64_t>(parts, std::max(1u, kMaxSort / (a.beams * a.width)));
  P.parts = uint32_t(std::max<uint64_t>(parts, 1));
  P.sorted = 2;
  while (P.sorted < a.beams * P.parts * a.width) P.sorted *= 2;
  // a slice of 4096 values at least, and no more blocks than two to an SM
  P.slices = uint32_t(std::max<uint64_t>(1, std::min<uint64_t>({32, 296 / std::max(a.B, 1u), (a.V + 4095) / 4096})));
  uint8_t* base = static_cast<uint8_t*>(scratch);
  const uint64_t n = rows * P.parts;
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    at += bytes;
    return base + (at - bytes);
  };
  P.best = reinterpret_cast<uint64_t*>(take(8 * n * a.width));
  P.sums = reinterpret_cast<double*>(take(8 * n));
  P.exact = reinterpret_cast<double*>(take(8 * rows * P.slices));
  P.tops = reinterpret_cast<float*>(take(4 * n));
  P.came = reinterpret_cast<uint32_t*>(take(4 * uint64_t(a.B)));
  return at;
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
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return VOOM_E_CUDA;
  if (!(allowed.load(std::memory_order_relaxed) >> (dev & 63) & 1u)) {
    const auto allow = [](const void* kernel, int n) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, n) == cudaSuccess; };
    if (!allow(reinterpret_cast<const void*>(beam_join), kMaxSort * kCandidate) ||
        !allow(reinterpret_cast<const void*>(beam_rows<__nv_bfloat16>), sizeof(RowShared)) ||
        !allow(reinterpret_cast<const void*>(beam_rows<__half>), sizeof(RowShared)) ||
        !allow(reinterpret_cast<const void*>(beam_rows<float>), sizeof(RowShared))) {
      cudaGetLastError();
      return VOOM_E_CUDA;
    }
    allowed.fetch_or(uint64_t(1) << (dev & 63), std::memory_order_relaxed);
  }
  if (a->type == VOOM_BF16) beam_rows<__nv_bfloat16><<<grid, kThreads, sizeof(RowShared), s>>>(P);
  else if (a->type == VOOM_FP16) beam_rows<__half><<<grid, kThreads, sizeof(RowShared), s>>>(P);
  else beam_rows<float><<<grid, kThreads, sizeof(RowShared), s>>>(P);
  if (cudaGetLastError() != cudaSuccess) return VOOM_E_CUDA;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute early{};
  cfg.gridDim = dim3(a->B * P.slices);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = P.sorted * kCandidate;
  cfg.stream = s;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, beam_join, P) == cudaSuccess) return VOOM_OK;
  cudaGetLastError();
  return VOOM_E_CUDA;
}
