// Launches of the cache attention's kernels.  Each pair of a type and a kind of
// scores is a source file of its own (kv_attn_*.cu): together they take minutes to compile.
#pragma once

#include <algorithm>
#include <atomic>

#include "kv_few.cuh"
#include "kv_rows.cuh"
#include "kv_sums.cuh"
#include "kv_tc.cuh"

namespace voom {
namespace kv {

// Lets a kernel use `bytes` of shared memory on the current device, once per device.
inline bool allow_smem(const void* kernel, uint32_t bytes, std::atomic<uint64_t>& devices) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  if (devices.load(std::memory_order_relaxed) >> (dev & 63) & 1u) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  devices.fetch_or(uint64_t(1) << (dev & 63), std::memory_order_relaxed);
  return true;
}

template <typename T, int DP, int MT, bool SCORED>
int launch_rows(const Attn& P, cudaStream_t s) {
  constexpr uint32_t smem = row_smem(DP, MT, SCORED);
  static std::atomic<uint64_t> allowed{0};
  if (!allow_smem(reinterpret_cast<const void*>(attn_rows<T, DP, MT, SCORED>), smem, allowed)) return VOOM_E_CUDA;
  const uint64_t grid = P.ctas ? P.ctas : uint64_t(P.c.v.B) * P.c.v.hk * P.mblocks;
  attn_rows<T, DP, MT, SCORED><<<uint32_t(grid), 32 * row_warps(DP, SCORED), smem, s>>>(P);
  return cudaGetLastError() == cudaSuccess ? VOOM_OK : VOOM_E_CUDA;
}

template <typename T, int DP, int MODE, bool SCORED>
int launch_tc(const Attn& P, cudaStream_t s) {
  constexpr uint32_t smem = tc_smem<DP, MODE>();
  static std::atomic<uint64_t> allowed{0};
  if (!allow_smem(reinterpret_cast<const void*>(attn_tc<T, DP, MODE, SCORED>), smem, allowed)) return VOOM_E_CUDA;
  const uint64_t grid = P.ctas ? P.ctas : uint64_t(P.c.v.B) * P.c.v.hk * P.mblocks;
  attn_tc<T, DP, MODE, SCORED><<<uint32_t(grid), Tc<DP, MODE>::THREADS, smem, s>>>(P);
  return cudaGetLastError() == cudaSuccess ? VOOM_OK : VOOM_E_CUDA;
}

template <typename T, int DP, bool SCORED>
int launch_sums_of(const Attn& P, cudaStream_t s) {
  constexpr uint32_t smem = sums_smem<DP>();
  static std::atomic<uint64_t> allowed{0};
  if (!allow_smem(reinterpret_cast<const void*>(attn_sums<T, DP, SCORED>), smem, allowed)) return VOOM_E_CUDA;
  attn_sums<T, DP, SCORED><<<P.ctas, Sums<DP>::THREADS, smem, s>>>(P);
  return cudaGetLastError() == cudaSuccess ? VOOM_OK : VOOM_E_CUDA;
}

template <typename T, int DP>
int launch_few(const Attn& P, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  if (!allow_smem(reinterpret_cast<const void*>(attn_few<T, DP>), Few<DP>::SMEM, allowed)) return VOOM_E_CUDA;
  const uint64_t grid = P.ctas ? P.ctas : uint64_t(P.c.v.B) * P.c.v.hk;
  attn_few<T, DP><<<uint32_t(grid), 32 * Few<DP>::W, Few<DP>::SMEM, s>>>(P);
  return cudaGetLastError() == cudaSuccess ? VOOM_OK : VOOM_E_CUDA;
}

template <typename T, bool SCORED>
int launch_attention(const Attn& P, cudaStream_t s) {
  if (P.tc == kSingle) return launch_tc<T, 256, kSingle, SCORED>(P, s);
  if (P.tc == kPair) return P.ld_o == 64 ? launch_tc<T, 64, kPair, SCORED>(P, s) : launch_tc<T, 128, kPair, SCORED>(P, s);
  if (P.tc == kAlternate)
    return P.ld_o == 64 ? launch_tc<T, 64, kAlternate, SCORED>(P, s) : launch_tc<T, 128, kAlternate, SCORED>(P, s);
  if constexpr (SCORED) {
    if (P.tc == kFew) return P.ld_o == 64 ? launch_few<T, 64>(P, s) : P.ld_o == 128 ? launch_few<T, 128>(P, s) : launch_few<T, 256>(P, s);
  }
  if (P.ld_o == 64) return P.rows == 16 ? launch_rows<T, 64, 1, SCORED>(P, s) : launch_rows<T, 64, 2, SCORED>(P, s);
  if (P.ld_o == 128) return P.rows == 16 ? launch_rows<T, 128, 1, SCORED>(P, s) : launch_rows<T, 128, 2, SCORED>(P, s);
  return launch_rows<T, 256, 1, SCORED>(P, s);
}

template <typename T, bool SCORED>
int launch_sums(const Attn& P, cudaStream_t s) {
  if (P.ld_o == 64) return launch_sums_of<T, 64, SCORED>(P, s);
  return P.ld_o == 128 ? launch_sums_of<T, 128, SCORED>(P, s) : launch_sums_of<T, 256, SCORED>(P, s);
}

}  // namespace kv
}  // namespace voom
