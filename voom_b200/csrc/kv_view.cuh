// Where a cached position's key and value lie (voom_kv_view on the device).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace voom {
namespace kv {

constexpr uint32_t kMaxD = 256;

// The view with the division by the page size as a multiplication: for
// s < 2^31, s / page = (s * magic) >> 32 >> shift with magic = ceil(2^(32+shift) / page).
struct View {
  voom_kv_view v;
  uint32_t magic, shift;

  __device__ __forceinline__ uint32_t page_of(uint32_t s) const {
    return magic ? __umulhi(s, magic) >> shift : s >> shift;
  }
  __device__ __forceinline__ uint32_t length(uint32_t b) const {
    const int32_t n = v.d_len[b];
    return n <= 0 ? 0u : min(uint32_t(n), v.max_len);
  }
  // Element offsets (from d_k, d_v) of the page that holds position s of
  // request b, head 0, position 0 of the page; false for a page that is none.
  __device__ __forceinline__ bool page_at(uint32_t b, uint32_t p, int64_t& k, int64_t& w) const {
    if (v.d_table) {
      const int32_t i = __ldg(v.d_table + uint64_t(b) * v.table_stride + p);
      if (uint32_t(i) >= v.n_pages) return false;
      k = int64_t(i) * v.k_page;
      w = int64_t(i) * v.v_page;
    } else if (v.d_offsets) {
      const longlong2 o = __ldg(reinterpret_cast<const longlong2*>(v.d_offsets) + uint64_t(b) * v.table_stride + p);
      if (o.x == VOOM_NO_PAGE) return false;
      k = o.x;
      w = o.y;
    } else {
      k = int64_t(b) * v.k_page;
      w = int64_t(b) * v.v_page;
    }
    return true;
  }
  // Element offsets of position s of head h of request b.
  __device__ __forceinline__ bool row_at(uint32_t b, uint32_t h, uint32_t s, int64_t& k, int64_t& w) const {
    const uint32_t p = page_of(s), o = s - p * v.page;
    if (!page_at(b, p, k, w)) return false;
    k += int64_t(h) * v.k_head + int64_t(o) * v.k_pos;
    w += int64_t(h) * v.v_head + int64_t(o) * v.v_pos;
    return true;
  }
};

// Host: checks the view (VOOM_OK or why not) and prepares the division.
inline int make_view(const voom_kv_view* c, View& out) {
  if (!c || !c->d_k || !c->d_v || !c->d_len) return VOOM_E_INVALID_ARG;
  if (!c->B || !c->hk || !c->D || !c->page || c->type > VOOM_FP16) return VOOM_E_INVALID_ARG;
  if (c->D % 8 || c->D > kMaxD) return VOOM_E_UNSUPPORTED;
  if (c->B > 65535u || c->hk > 65535u || c->max_len > 0x7FFFFFFFu || c->page > 0x7FFFFFFFu) return VOOM_E_UNSUPPORTED;
  if (c->d_table && c->d_offsets) return VOOM_E_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(c->d_k) | reinterpret_cast<uintptr_t>(c->d_v)) & 15u) return VOOM_E_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(c->d_offsets) & 15u) return VOOM_E_INVALID_ARG;
  for (int64_t s : {c->k_page, c->k_head, c->k_pos, c->v_page, c->v_head, c->v_pos})
    if (s % 8) return VOOM_E_INVALID_ARG;
  const bool paged = c->d_table || c->d_offsets;
  const uint64_t capacity = paged ? uint64_t(c->page) * c->table_stride : c->page;
  if (c->max_len > capacity) return VOOM_E_INVALID_ARG;
  out.v = *c;
  uint32_t up = 0;
  while ((1ull << up) < c->page) up++;
  if ((1ull << up) == c->page) {
    out.magic = 0;
    out.shift = up;
  } else {  // 2^(up-1) < page < 2^up: the rounded-up reciprocal is exact below 2^31
    out.shift = up - 1;
    out.magic = uint32_t(((uint64_t(1) << (32 + out.shift)) + c->page - 1) / c->page);
  }
  return VOOM_OK;
}

template <typename T>
__device__ __forceinline__ float elem(T v);
template <>
__device__ __forceinline__ float elem<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float elem<__half>(__half v) { return __half2float(v); }
}  // namespace kv
}  // namespace voom
