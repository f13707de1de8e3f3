// Pages of a KV cache: new tokens written to their places, rows of a page table
// forked, the pages in use brought together.
//
// kv_append: a group of lanes takes one new token, finds its place once and
// copies its heads, 16 bytes a lane.
//
// Forking needs three things of the whole table before it can move a byte: how
// often each page is held, which of an open page's holders may write on in it,
// and which pages are free, in order.  fork_tables counts (whole numbers, so
// their order does not matter) while it writes the new table; fork_plan, one
// block, numbers the wanted pages by row and the free ones by index, so that the
// k-th wanted meets the k-th free; fork_finish enters them and copies the open
// pages.  Compaction is alike: kv_mark, compact_plan, compact_finish.  For small
// tables one block does the first two (fork_small, compact_small).
//
// The copies are bound by HBM, the rest by latency: a chain of reads and barriers.
// Measured: 3 heads of 64 in 4 layers, 4 rows: 7.5 us a fork, 8.9 a compaction; 256
// rows in 2 layers, 28 MB of open pages copied: 19 us, 12 of it the copies (4.8 TB/s
// read and written); 1426 of 3001 pages of 256 KB moved: 128 us, 5.8 TB/s (89 % of
// what a copy reaches).  One block numbers the pages, whatever their number: 256 rows in
// a pool of 10^4, 10^5 and 10^6 pages take 13, 31 and 239 us to fork, 14, 39 and 283 to
// compact.  16376 new tokens of 8 heads of 128 written: 20.5 us, 6.5 TB/s.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "kv_view.cuh"
#include "rows.h"

namespace {

constexpr uint32_t kMaxPage = 32768, kMaxRows = 65535;
// Tables that one block does.  Entries: 4000 take 9.6 us forked by one block, 10.1 by
// many; 8000 12.2 and 10.4, but for 5 us that the host saves (a captured call has no
// host to save, and would want the limit at 4000); 16000 17.1 and 11.4.
// Pages and rows: what its shared memory holds.
constexpr uint32_t kSmallPages = 12288, kSmallRows = 4096, kSmallEntries = 8192;
constexpr uint32_t kSmallBytes = 8 * kSmallPages + 12 * kSmallRows;

__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A launch whose blocks may start before the last kernel has ended; they wait for it themselves.
template <typename... A>
int launch_early(void (*kernel)(A...), dim3 grid, uint32_t threads, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute early{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess) return VOOM_OK;
  cudaGetLastError();
  return VOOM_E_CUDA;
}

// A table entry may be a page that its row holds but cannot use: an open one whose copy
// found no fresh page.  It stands as page - 2^31, which no reader or writer takes for a
// page; the next fork takes it for the page that it is.
constexpr uint32_t kUnusable = 0x80000000u;
__device__ __forceinline__ int32_t page_in(int32_t entry, uint32_t n_pages) {
  const uint32_t t = uint32_t(entry) & ~kUnusable;
  return t < n_pages ? int32_t(t) : -1;
}

// ------------------------------------------------------------------- append
struct Append {
  voom::kv::View c;
  voom_kv_append_args a;
  uint32_t lanes, heads, parts;  // lanes of a row; heads that a group copies; groups of a token
  uint32_t capacity;
};

__global__ void __launch_bounds__(256) kv_append(const __grid_constant__ Append P) {
  const uint64_t group = (uint64_t(blockIdx.x) * 256 + threadIdx.x) / P.lanes;
  const uint32_t e = threadIdx.x & (P.lanes - 1), chunks = P.c.v.D / 8;
  const uint64_t token = group / P.parts;
  const uint32_t part = uint32_t(group - token * P.parts);
  const uint32_t b = uint32_t(token / P.a.m), j = uint32_t(token - uint64_t(b) * P.a.m);
  if (b >= P.c.v.B || e >= chunks) return;
  const int32_t i = P.a.d_index ? P.a.d_index[token] : int32_t(j);
  // (not length(b): a view's max_len bounds what is read, and must not turn a write back to what is cached)
  const uint64_t s = uint64_t(max(P.c.v.d_len[b], 0)) + j;
  int64_t ko, vo;
  if (uint32_t(i) >= P.a.n || s >= P.capacity || !P.c.row_at(b, 0, uint32_t(s), ko, vo)) return;
  const uint16_t* kn = static_cast<const uint16_t*>(P.a.d_kn) + int64_t(b) * P.a.kn_b + int64_t(i) * P.a.kn_t + 8 * e;
  const uint16_t* vn = static_cast<const uint16_t*>(P.a.d_vn) + int64_t(b) * P.a.vn_b + int64_t(i) * P.a.vn_t + 8 * e;
  uint16_t* k = static_cast<uint16_t*>(const_cast<void*>(P.c.v.d_k)) + ko + 8 * e;
  uint16_t* v = static_cast<uint16_t*>(const_cast<void*>(P.c.v.d_v)) + vo + 8 * e;
  const uint32_t h0 = part * P.heads, h1 = min(P.c.v.hk, h0 + P.heads);
  for (uint32_t h = h0; h < h1; h += 4) {
    uint4 x[4], y[4];
#pragma unroll
    for (uint32_t u = 0; u < 4; u++)
      if (h + u < h1) {
        x[u] = __ldcs(reinterpret_cast<const uint4*>(kn + int64_t(h + u) * P.a.kn_h));
        y[u] = __ldcs(reinterpret_cast<const uint4*>(vn + int64_t(h + u) * P.a.vn_h));
      }
#pragma unroll
    for (uint32_t u = 0; u < 4; u++)
      if (h + u < h1) {
        *reinterpret_cast<uint4*>(k + int64_t(h + u) * P.c.v.k_head) = x[u];
        *reinterpret_cast<uint4*>(v + int64_t(h + u) * P.c.v.v_head) = y[u];
      }
  }
}

// --------------------------------------------------------------------- fork
// A page's count: rows that hold it full in the low half, open in the high one.
struct CopyItem {
  uint32_t src, rank, fill;  // page; which fresh page it goes to; positions
};

struct Fork {
  voom_kv_fork_args a;
  uint32_t* count;  // n_pages, 0 at first
  uint32_t* owner;  // n_pages, 0 at first: (filled positions, then the first row) of its open holders, the largest
  uint32_t* words;  // free pages, copies
  uint4* rows;      // rows: rank of the row's first fresh page, its place in the row, the place behind the last one, and
                    // whether the first replaces an open page
  CopyItem* copies; // rows
  int32_t* fresh;   // free pages in order, as many as are wanted
  int32_t* table;   // the new table and lengths: the caller's, or scratch where those are still read
  int32_t* lengths;
};

struct RowState {
  uint32_t len, used, want, fill;
  uint32_t lost;  // pages that the table has no room for
  bool grows;
};

__device__ __forceinline__ uint32_t clamped_length(const int32_t* len, uint32_t r, uint64_t capacity) {
  const int32_t n = len[r];
  return n <= 0 ? 0u : uint32_t(min(uint64_t(n), capacity));
}

__device__ __forceinline__ bool parent_of(const Fork& P, uint32_t r, uint32_t& p) {
  p = P.a.d_parents ? uint32_t(P.a.d_parents[r]) : r;
  return p < P.a.rows;
}

__device__ __forceinline__ RowState row_state(const Fork& P, uint32_t r, uint32_t len, bool live) {
  RowState s;
  const int32_t g = !live ? 0 : P.a.d_grow ? P.a.d_grow[r] : int32_t(P.a.grow);
  s.len = len;
  s.used = (len + P.a.page - 1) / P.a.page;
  s.fill = len % P.a.page;
  s.grows = g > 0;
  const uint64_t want = s.grows ? (uint64_t(len) + uint32_t(g) + P.a.page - 1) / P.a.page : s.used;
  s.want = uint32_t(min(want, uint64_t(P.a.per)));
  s.lost = uint32_t(want - s.want);
  return s;
}

__device__ __forceinline__ uint32_t claim_of(uint32_t fill, uint32_t r) { return fill << 16 | (0xFFFFu - r); }

// The length that row r takes over.
__device__ __forceinline__ uint32_t taken_length(const Fork& P, uint32_t r, uint32_t& p) {
  return parent_of(P, r, p) ? clamped_length(P.a.d_lengths, p, uint64_t(P.a.per) * P.a.page) : 0u;
}

// Entry j of row r, which continues row p with `len` positions: written, counted, returned.
__device__ __forceinline__ int32_t take_entry(const Fork& P, uint32_t r, uint32_t j, uint32_t p, uint32_t len, uint32_t* count,
                                           uint32_t* owner) {
  int32_t t = -1;
  if (uint64_t(j) * P.a.page < len) t = page_in(P.a.d_table[uint64_t(p) * P.a.per + j], P.a.n_pages);
  P.table[uint64_t(r) * P.a.per + j] = t;
  if (t < 0) return t;
  const uint32_t fill = len - j * P.a.page;
  if (fill >= P.a.page) {
    atomicAdd(&count[t], 1u);
  } else {
    atomicAdd(&count[t], 1u << 16);
    atomicMax(&owner[t], claim_of(fill, r));
  }
  return t;
}

__global__ void __launch_bounds__(256) fork_tables(const __grid_constant__ Fork P) {
  const uint32_t r = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
  if (j >= P.a.per) return;
  uint32_t p;
  const uint32_t len = taken_length(P, r, p);
  if (j == 0) P.lengths[r] = int32_t(len);
  take_entry(P, r, j, p, len, P.count, P.owner);
}

// Exclusive sum of x over the block's threads, and the total; all threads call it.
__device__ __forceinline__ uint64_t block_before(uint64_t x, uint64_t* s_warp, uint64_t& total) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  uint64_t y = x;
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t z = __shfl_up_sync(0xFFFFFFFFu, y, o);
    if (int(lane) >= o) y += z;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = y;
  __syncthreads();
  uint64_t w = lane < warps ? s_warp[lane] : 0;
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t z = __shfl_up_sync(0xFFFFFFFFu, w, o);
    if (int(lane) >= o) w += z;
  }
  total = __shfl_sync(0xFFFFFFFFu, w, 31);
  const uint64_t before = __shfl_sync(0xFFFFFFFFu, w, (warp + 31) & 31u);
  return (warp ? before : 0) + y - x;
}

// Walks n pages in order, kPlanDeep at a time to a thread: `load` gives a page's
// count, `take` gets the page, its count, whether it is marked, and how many
// marked ones come before it.
constexpr uint32_t kPlanThreads = 1024, kPlanDeep = 8;
template <typename Load, typename Mark, typename Take>
__device__ __forceinline__ uint32_t walk_pages(uint32_t n, uint32_t* s_sum, Load load, Mark mark, Take take) {
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  uint32_t seen = 0;
  for (uint32_t p0 = 0; p0 < n; p0 += kPlanThreads * kPlanDeep) {
    uint32_t c[kPlanDeep], bits[kPlanDeep];
#pragma unroll
    for (uint32_t i = 0; i < kPlanDeep; i++) {
      const uint32_t p = p0 + i * kPlanThreads + tid;
      c[i] = p < n ? load(p) : 0u;
    }
    __syncthreads();  // the sums of the last round are read
#pragma unroll
    for (uint32_t i = 0; i < kPlanDeep; i++) {
      bits[i] = __ballot_sync(0xFFFFFFFFu, p0 + i * kPlanThreads + tid < n && mark(c[i]));
      if (lane == 0) s_sum[i * 32 + warp] = __popc(bits[i]);
    }
    __syncthreads();
    if (warp == 0) {  // sums before, over the 256 warps' counts: 8 to a lane
      uint32_t x[8], mine = 0;
#pragma unroll
      for (uint32_t i = 0; i < 8; i++) {
        x[i] = s_sum[lane * 8 + i];
        mine += x[i];
      }
      uint32_t upto = mine;
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t z = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (int(lane) >= o) upto += z;
      }
      uint32_t at = upto - mine;
#pragma unroll
      for (uint32_t i = 0; i < 8; i++) {
        s_sum[lane * 8 + i] = at;
        at += x[i];
      }
      if (lane == 31) s_sum[256] = at;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kPlanDeep; i++) {
      const uint32_t p = p0 + i * kPlanThreads + tid;
      if (p < n) take(p, c[i], (bits[i] >> lane & 1u) != 0, seen + s_sum[i * 32 + warp] + __popc(bits[i] & ((1u << lane) - 1u)));
    }
    seen += s_sum[256];
  }
  return seen;
}
static_assert(kPlanThreads / 32 * kPlanDeep == 256, "walk_pages sums 256 counts");

// `length`, `live` and `last` tell a row's length, whether it goes on, and its last page.
template <typename Length, typename Live, typename Last>
__device__ __forceinline__ void plan_fork(const Fork& P, uint32_t* count, const uint32_t* owner, Length length, Live live, Last last) {
  __shared__ uint64_t s_warp[32];
  __shared__ uint32_t s_sum[257];
  __shared__ uint32_t s_lost;
  if (threadIdx.x == 0) s_lost = 0;
  __syncthreads();
  uint64_t all = 0;  // copies, then pages wanted (low half), of the rows so far
  for (uint32_t r0 = 0; r0 < P.a.rows; r0 += kPlanThreads) {
    const uint32_t r = r0 + threadIdx.x;
    uint32_t src = 0, fill = 0, need = 0, first = 0, want = 0;
    bool copy = false;
    if (r < P.a.rows) {
      const RowState s = row_state(P, r, length(r), live(r));
      need = s.want - s.used;
      first = s.used;
      want = s.want;
      fill = s.fill;
      if (s.lost) atomicAdd(&s_lost, s.lost);
      if (s.grows && fill) {
        const int32_t t = last(r, s.used - 1);
        if (t >= 0) {
          src = uint32_t(t);
          copy = (count[src] & 0xFFFFu) || owner[src] != claim_of(fill, r);
        }
      }
      if (copy) {
        need++;
        first--;
        atomicSub(&count[src], 1u << 16);  // (the full holders, which others read, stay)
      }
    }
    uint64_t total;
    const uint64_t at = all + block_before(uint64_t(copy) << 32 | need, s_warp, total);
    if (r < P.a.rows) {
      P.rows[r] = make_uint4(uint32_t(at), first, want, uint32_t(copy));
      if (copy) P.copies[at >> 32] = CopyItem{src, uint32_t(at), fill};
    }
    all += total;
  }
  __syncthreads();
  const uint32_t wanted = uint32_t(all);
  const uint32_t free = walk_pages(
      P.a.n_pages, s_sum, [&](uint32_t p) { return count[p]; }, [](uint32_t c) { return c == 0; },
      [&](uint32_t p, uint32_t c, bool none, uint32_t rank) {
        if (none && rank < wanted) P.fresh[rank] = int32_t(p);
        P.a.d_refs[p] = none ? (rank < wanted ? 1 : 0) : int32_t((c & 0xFFFFu) + (c >> 16));
      });
  if (free < wanted) {  // rows whose open page has no copy hold it still
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < uint32_t(all >> 32); i += kPlanThreads)
      if (P.copies[i].rank >= free) atomicAdd(&P.a.d_refs[P.copies[i].src], 1);
  }
  if (threadIdx.x == 0) {
    const uint32_t lost = s_lost + (wanted > free ? wanted - free : 0u);
    *P.a.d_missing = int32_t(lost + (P.a.add_missing ? uint32_t(*P.a.d_missing) : 0u));
    P.words[0] = free;
    P.words[1] = uint32_t(all >> 32);
  }
}

__global__ void __launch_bounds__(kPlanThreads) fork_plan(const __grid_constant__ Fork P) {
  wait_for_last();
  plan_fork(
      P, P.count, P.owner, [&](uint32_t r) { return uint32_t(P.lengths[r]); },
      [&](uint32_t r) {
        uint32_t p;
        return parent_of(P, r, p);
      },
      [&](uint32_t r, uint32_t j) { return P.table[uint64_t(r) * P.a.per + j]; });
}

// Small tables: fork_tables and fork_plan in one block, the pages' counts in shared memory.
__global__ void __launch_bounds__(kPlanThreads) fork_small(const __grid_constant__ Fork P) {
  extern __shared__ uint32_t s_pages[];
  uint32_t *count = s_pages, *owner = count + P.a.n_pages, *len = owner + P.a.n_pages, *parent = len + P.a.rows;
  int32_t* last = reinterpret_cast<int32_t*>(parent + P.a.rows);
  for (uint32_t i = threadIdx.x; i < 2 * P.a.n_pages; i += kPlanThreads) s_pages[i] = 0;
  for (uint32_t r = threadIdx.x; r < P.a.rows; r += kPlanThreads) {
    len[r] = taken_length(P, r, parent[r]);
    P.lengths[r] = int32_t(len[r]);
  }
  __syncthreads();
  const uint32_t entries = P.a.rows * P.a.per;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < entries; i += kPlanThreads) {
    const uint32_t r = i / P.a.per;
    const uint32_t j = i - r * P.a.per;
    const int32_t t = take_entry(P, r, j, parent[r], len[r], count, owner);
    if (len[r] && j == (len[r] - 1) / P.a.page) last[r] = t;
  }
  __syncthreads();
  plan_fork(
      P, count, owner, [&](uint32_t r) { return len[r]; }, [&](uint32_t r) { return parent[r] < P.a.rows; },
      [&](uint32_t r, uint32_t) { return last[r]; });
}

// n rows of `chunks` 16-byte pieces, kDeep of them a thread under way.
__device__ __forceinline__ void copy_rows(uint16_t* to, const uint16_t* from, uint32_t n, uint32_t chunks, int64_t pos) {
  constexpr uint32_t kDeep = 4;
  const uint32_t all = n * chunks;
  for (uint32_t i0 = threadIdx.x; i0 < all; i0 += kDeep * blockDim.x) {
    uint4 x[kDeep];
#pragma unroll
    for (uint32_t u = 0; u < kDeep; u++) {
      const uint32_t i = i0 + u * blockDim.x, r = i / chunks, e = i - r * chunks;
      if (i < all) x[u] = __ldcs(reinterpret_cast<const uint4*>(from + int64_t(r) * pos + 8 * e));
    }
#pragma unroll
    for (uint32_t u = 0; u < kDeep; u++) {
      const uint32_t i = i0 + u * blockDim.x, r = i / chunks, e = i - r * chunks;
      if (i < all) *reinterpret_cast<uint4*>(to + int64_t(r) * pos + 8 * e) = x[u];
    }
  }
}

// One item's part of a page: head h of layer l, of keys and values.
template <typename A>
__device__ __forceinline__ void copy_page(const A& a, uint32_t src, uint32_t dst, uint32_t part, uint32_t n) {
  const uint32_t l = part / a.hk, h = part - l * a.hk;
  uint16_t* k = static_cast<uint16_t*>(a.d_k) + int64_t(l) * a.k_layer + int64_t(h) * a.k_head;
  uint16_t* v = static_cast<uint16_t*>(a.d_v) + int64_t(l) * a.v_layer + int64_t(h) * a.v_head;
  copy_rows(k + int64_t(dst) * a.k_page, k + int64_t(src) * a.k_page, n, a.D / 8, a.k_pos);
  copy_rows(v + int64_t(dst) * a.v_page, v + int64_t(src) * a.v_page, n, a.D / 8, a.v_pos);
}

__global__ void __launch_bounds__(256) fork_finish(const __grid_constant__ Fork P) {
  wait_for_last();
  const uint32_t free = P.words[0], parts = P.a.layers * P.a.hk;
  const bool back = P.table != P.a.d_table_out;
  for (uint32_t r = blockIdx.x; r < P.a.rows; r += gridDim.x) {
    const uint4 fresh = P.rows[r];
    const uint32_t want = fresh.z;
    const int32_t* from = P.table + uint64_t(r) * P.a.per;
    int32_t* to = P.a.d_table_out + uint64_t(r) * P.a.per;
    for (uint32_t j = (back ? 0u : fresh.y) + threadIdx.x; j < (back ? P.a.per : want); j += 256) {
      const uint32_t rank = fresh.x + (j - fresh.y);
      to[j] = j < fresh.y || j >= want ? from[j]
              : rank < free            ? P.fresh[rank]
              : fresh.w && j == fresh.y ? int32_t(uint32_t(from[j]) | kUnusable)
                                        : -1;
    }
    if (back && threadIdx.x == 0) P.a.d_lengths_out[r] = P.lengths[r];
  }
  const uint64_t items = uint64_t(P.words[1]) * parts;
  for (uint64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const uint32_t c = uint32_t(i / parts), part = uint32_t(i - uint64_t(c) * parts);
    const CopyItem x = P.copies[c];
    if (x.rank < free) copy_page(P.a, x.src, uint32_t(P.fresh[x.rank]), part, x.fill);
  }
}

// ------------------------------------------------------------------ compact
struct Compact {
  voom_kv_compact_args a;
  uint32_t* held;   // n_pages, 0 at first
  uint32_t* words;  // pages that move
  int32_t* from;    // the pages that move, in order, and
  int32_t* to;      // where they go
  int32_t* place;   // n_pages: where a page that moves goes
};

__device__ __forceinline__ int32_t held_page(const Compact& P, uint32_t r, uint32_t j) {
  const uint32_t len = clamped_length(P.a.d_lengths, r, uint64_t(P.a.per) * P.a.page);
  if (uint64_t(j) * P.a.page >= len && !P.a.room) return -1;
  return page_in(P.a.d_table[uint64_t(r) * P.a.per + j], P.a.n_pages);
}

__global__ void __launch_bounds__(256) kv_mark(const __grid_constant__ Compact P) {
  const uint32_t r = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
  const int32_t t = j < P.a.per ? held_page(P, r, j) : -1;
  if (t >= 0) P.held[t] = 1;
}

__device__ __forceinline__ void plan_compact(const Compact& P, const uint32_t* held) {
  __shared__ uint32_t s_sum[257];
  auto load = [&](uint32_t p) { return held[p]; };
  auto marked = [](uint32_t c) { return c != 0; };
  const uint32_t live = walk_pages(P.a.n_pages, s_sum, load, marked, [](uint32_t, uint32_t, bool, uint32_t) {});
  // below `live` the free pages are as many as the held ones past it
  const uint32_t stay = walk_pages(live, s_sum, load, marked, [&](uint32_t p, uint32_t, bool on, uint32_t rank) {
    if (!on) P.to[p - rank] = int32_t(p);
  });
  walk_pages(P.a.n_pages, s_sum, load, marked, [&](uint32_t p, uint32_t, bool on, uint32_t rank) {
    if (on && p >= live) P.from[rank - stay] = int32_t(p);
  });
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < live - stay; i += kPlanThreads) P.place[P.from[i]] = P.to[i];
  if (threadIdx.x == 0) {
    *P.a.d_live = int32_t(live);
    P.words[0] = live;
    P.words[1] = live - stay;
  }
}

__global__ void __launch_bounds__(kPlanThreads) compact_plan(const __grid_constant__ Compact P) {
  wait_for_last();
  plan_compact(P, P.held);
}

// Small tables: kv_mark and compact_plan in one block.
__global__ void __launch_bounds__(kPlanThreads) compact_small(const __grid_constant__ Compact P) {
  extern __shared__ uint32_t s_pages[];
  for (uint32_t i = threadIdx.x; i < P.a.n_pages; i += kPlanThreads) s_pages[i] = 0;
  __syncthreads();
  const uint32_t entries = P.a.rows * P.a.per;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < entries; i += kPlanThreads) {
    const uint32_t r = i / P.a.per;
    const int32_t t = held_page(P, r, i - r * P.a.per);
    if (t >= 0) s_pages[t] = 1;
  }
  __syncthreads();
  plan_compact(P, s_pages);
}

__global__ void __launch_bounds__(256) compact_finish(const __grid_constant__ Compact P) {
  wait_for_last();
  const uint32_t live = P.words[0], moves = P.words[1], parts = P.a.layers * P.a.hk;
  const uint64_t entries = uint64_t(P.a.rows) * P.a.per;
  for (uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x; i < entries; i += uint64_t(gridDim.x) * 256) {
    const uint32_t r = uint32_t(i / P.a.per);
    const int32_t t = held_page(P, r, uint32_t(i - uint64_t(r) * P.a.per)), to = t < int32_t(live) ? t : P.place[t];
    P.a.d_table_out[i] = int32_t(uint32_t(to) | (uint32_t(P.a.d_table[i]) & (t < 0 ? 0u : kUnusable)));
  }
  const uint64_t items = uint64_t(moves) * parts;
  for (uint64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const uint32_t c = uint32_t(i / parts);
    copy_page(P.a, uint32_t(P.from[c]), uint32_t(P.to[c]), uint32_t(i - uint64_t(c) * parts), P.a.page);
  }
}

int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

// What a pool's arguments have in common: VOOM_OK or why not.
template <typename A>
int check_pool(const A& a) {
  if (!a.d_k || !a.d_v || !a.d_table || !a.d_lengths || !a.d_table_out) return VOOM_E_INVALID_ARG;
  if (!a.layers || !a.n_pages || !a.hk || !a.page || !a.D || a.D % 8 || !a.per) return VOOM_E_INVALID_ARG;
  if (a.page > kMaxPage || a.rows > kMaxRows || a.n_pages > 0x7FFFFFFFu || uint64_t(a.layers) * a.hk > 0x7FFFFFFFu || a.D > voom::kv::kMaxD ||
      uint64_t(a.per) * a.page > 0x7FFFFFFFu || uint64_t(a.rows) * a.per > 0x7FFFFFFFu)
    return VOOM_E_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(a.d_k) | reinterpret_cast<uintptr_t>(a.d_v)) & 15u) return VOOM_E_INVALID_ARG;
  const int64_t steps[] = {a.k_layer, a.k_page, a.k_head, a.k_pos, a.v_layer, a.v_page, a.v_head, a.v_pos};
  for (int64_t s : steps)
    if (s % 8) return VOOM_E_INVALID_ARG;
  const int64_t L = a.layers, N = a.n_pages, hk = a.hk, p = a.page;
  const voom::RowsOf<4> k{a.d_k, {L, N, hk, p}, {a.k_layer, a.k_page, a.k_head, a.k_pos}, a.D, 2};
  const voom::RowsOf<4> v{a.d_v, {L, N, hk, p}, {a.v_layer, a.v_page, a.v_head, a.v_pos}, a.D, 2};
  return voom::separate(k) && voom::separate(v) && voom::disjoint(k, v) ? VOOM_OK : VOOM_E_OVERLAP;
}

struct Take {
  uint8_t* base;
  uint64_t at = 0;
  template <typename T>
  T* get(uint64_t n) {
    const uint64_t o = at;
    at += (n * sizeof(T) + 15) & ~uint64_t(15);
    return base ? reinterpret_cast<T*>(base + o) : nullptr;
  }
};

uint64_t layout(Fork& P, void* scratch) {
  Take take{static_cast<uint8_t*>(scratch)};
  const voom_kv_fork_args& a = P.a;
  const uint64_t entries = uint64_t(a.rows) * a.per;
  P.count = take.get<uint32_t>(2 * uint64_t(a.n_pages));  // cleared together
  P.owner = P.count ? P.count + a.n_pages : nullptr;
  P.words = take.get<uint32_t>(2);
  P.rows = take.get<uint4>(a.rows);
  P.copies = take.get<CopyItem>(a.rows);
  P.fresh = take.get<int32_t>(std::min<uint64_t>(entries, a.n_pages));
  const bool back = a.d_table_out == a.d_table;
  P.table = back ? take.get<int32_t>(entries) : a.d_table_out;
  P.lengths = back ? take.get<int32_t>(a.rows) : a.d_lengths_out;
  return take.at;
}

uint64_t layout(Compact& P, void* scratch) {
  Take take{static_cast<uint8_t*>(scratch)};
  const uint64_t n = P.a.n_pages;
  P.held = take.get<uint32_t>(n);
  P.words = take.get<uint32_t>(2);
  P.from = take.get<int32_t>(n / 2 + 1);
  P.to = take.get<int32_t>(n / 2 + 1);
  P.place = take.get<int32_t>(n);
  return take.at;
}

int check(const voom_kv_fork_args* a) {
  if (!a || !a->d_lengths_out || !a->d_refs || !a->d_missing) return VOOM_E_INVALID_ARG;
  if ((a->d_table_out == a->d_table) != (a->d_lengths_out == a->d_lengths)) return VOOM_E_INVALID_ARG;
  if (a->grow > 0x7FFFFFFFu) return VOOM_E_INVALID_ARG;
  return check_pool(*a);
}

int check(const voom_kv_compact_args* a) { return !a || !a->d_live ? VOOM_E_INVALID_ARG : check_pool(*a); }

// One block does the table: else its pages are counted in global memory, with a
// clear and two more launches.
template <typename A>
bool small(const A& a) {
  return a.n_pages <= kSmallPages && a.rows <= kSmallRows && uint64_t(a.rows) * a.per <= kSmallEntries;
}

// Lets a kernel use kSmallBytes of shared memory on the current device, once per device.
bool allow(const void* kernel, std::atomic<uint64_t>& devices) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  if (devices.load(std::memory_order_relaxed) >> (dev & 63) & 1u) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmallBytes)) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  devices.fetch_or(uint64_t(1) << (dev & 63), std::memory_order_relaxed);
  return true;
}

bool scratch_ok(const void* p) { return p && !(reinterpret_cast<uintptr_t>(p) & 15u); }

}  // namespace

VOOM_API int voom_kv_append(const voom_kv_view* c, const voom_kv_append_args* a, void* stream) {
  if (!a || !a->d_kn || !a->d_vn || (!a->d_index && a->m != a->n)) return VOOM_E_INVALID_ARG;
  Append P{};
  const int rc = voom::kv::make_view(c, P.c);
  if (rc != VOOM_OK) return rc;
  if ((reinterpret_cast<uintptr_t>(a->d_kn) | reinterpret_cast<uintptr_t>(a->d_vn)) & 15u) return VOOM_E_INVALID_ARG;
  const int64_t steps[] = {a->kn_b, a->kn_t, a->kn_h, a->vn_b, a->vn_t, a->vn_h};
  for (int64_t s : steps)
    if (s % 8) return VOOM_E_INVALID_ARG;
  if (a->n > 0x7FFFFFFFu || uint64_t(c->B) * a->m * c->hk > 0x7FFFFFFFu) return VOOM_E_UNSUPPORTED;
  if (!a->m || !a->n) return VOOM_OK;
  const int64_t B = c->B, n = a->n, hk = c->hk, D = c->D;
  // rows of the cache: of every page, or of one page anywhere
  const int64_t pages = c->d_offsets ? 1 : c->d_table ? c->n_pages : c->B;
  const voom::Rows k{c->d_k, {pages, hk, c->page}, {c->k_page, c->k_head, c->k_pos}, D, 2};
  const voom::Rows v{c->d_v, {pages, hk, c->page}, {c->v_page, c->v_head, c->v_pos}, D, 2};
  const voom::Rows kn{a->d_kn, {B, n, hk}, {a->kn_b, a->kn_t, a->kn_h}, D, 2};
  const voom::Rows vn{a->d_vn, {B, n, hk}, {a->vn_b, a->vn_t, a->vn_h}, D, 2};
  if (!voom::separate(k) || !voom::separate(v) || !voom::disjoint(k, v)) return VOOM_E_OVERLAP;
  if (!voom::disjoint(k, kn) || !voom::disjoint(k, vn) || !voom::disjoint(v, kn) || !voom::disjoint(v, vn)) return VOOM_E_OVERLAP;
  P.a = *a;
  P.lanes = 1;
  while (P.lanes < c->D / 8) P.lanes *= 2;
  const bool paged = c->d_table || c->d_offsets;
  P.capacity = uint32_t(std::min<uint64_t>(paged ? uint64_t(c->page) * c->table_stride : c->page, 0x7FFFFFFFu));
  // a group takes four heads, whose loads are under way together
  P.heads = std::min(c->hk, 4u);
  P.parts = (c->hk + P.heads - 1) / P.heads;
  const uint64_t threads = uint64_t(c->B) * a->m * P.parts * P.lanes;
  kv_append<<<uint32_t((threads + 255) / 256), 256, 0, static_cast<cudaStream_t>(stream)>>>(P);
  return cudaGetLastError() == cudaSuccess ? VOOM_OK : VOOM_E_CUDA;
}

VOOM_API uint64_t voom_kv_fork_scratch_bytes(uint32_t rows, uint32_t per, uint32_t n_pages, uint32_t in_place) {
  Fork P{};
  P.a.rows = rows;
  P.a.per = per;
  P.a.n_pages = n_pages;
  int32_t any;
  P.a.d_table = &any;
  P.a.d_table_out = in_place ? &any : nullptr;
  return layout(P, nullptr);
}

VOOM_API int voom_kv_fork(const voom_kv_fork_args* a, void* d_scratch, uint64_t bytes, void* stream) {
  const int rc = check(a);
  if (rc != VOOM_OK) return rc;
  Fork P{};
  P.a = *a;
  if (!scratch_ok(d_scratch)) return VOOM_E_INVALID_ARG;
  if (layout(P, d_scratch) > bytes) return VOOM_E_CAPACITY;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (small(*a)) {
    static std::atomic<uint64_t> allowed{0};
    if (!allow(reinterpret_cast<const void*>(fork_small), allowed)) return VOOM_E_CUDA;
    fork_small<<<1, kPlanThreads, 8 * a->n_pages + 12 * a->rows, s>>>(P);
    if (cudaGetLastError() != cudaSuccess) return VOOM_E_CUDA;
  } else {
    if (cudaMemsetAsync(P.count, 0, 8 * uint64_t(a->n_pages), s) != cudaSuccess) return VOOM_E_CUDA;
    if (a->rows) {
      fork_tables<<<dim3((a->per + 255) / 256, a->rows), 256, 0, s>>>(P);
      if (cudaGetLastError() != cudaSuccess) return VOOM_E_CUDA;
    }
    const int err = launch_early(fork_plan, dim3(1), kPlanThreads, s, P);
    if (err != VOOM_OK) return err;
  }
  if (!a->rows) return VOOM_OK;
  const uint64_t items = uint64_t(a->rows) * a->layers * a->hk;
  return launch_early(fork_finish, dim3(uint32_t(std::min<uint64_t>(items, 8ull * sm_count()))), 256, s, P);
}

VOOM_API uint64_t voom_kv_compact_scratch_bytes(uint32_t n_pages) {
  Compact P{};
  P.a.n_pages = n_pages;
  return layout(P, nullptr);
}

VOOM_API int voom_kv_compact(const voom_kv_compact_args* a, void* d_scratch, uint64_t bytes, void* stream) {
  const int rc = check(a);
  if (rc != VOOM_OK) return rc;
  Compact P{};
  P.a = *a;
  if (!scratch_ok(d_scratch)) return VOOM_E_INVALID_ARG;
  if (layout(P, d_scratch) > bytes) return VOOM_E_CAPACITY;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (small(*a)) {
    static std::atomic<uint64_t> allowed{0};
    if (!allow(reinterpret_cast<const void*>(compact_small), allowed)) return VOOM_E_CUDA;
    compact_small<<<1, kPlanThreads, 4 * a->n_pages, s>>>(P);
    if (cudaGetLastError() != cudaSuccess) return VOOM_E_CUDA;
  } else {
    if (cudaMemsetAsync(P.held, 0, 4 * uint64_t(a->n_pages), s) != cudaSuccess) return VOOM_E_CUDA;
    if (a->rows) {
      kv_mark<<<dim3((a->per + 255) / 256, a->rows), 256, 0, s>>>(P);
      if (cudaGetLastError() != cudaSuccess) return VOOM_E_CUDA;
    }
    const int err = launch_early(compact_plan, dim3(1), kPlanThreads, s, P);
    if (err != VOOM_OK) return err;
  }
  if (!a->rows) return VOOM_OK;
  return launch_early(compact_finish, dim3(8u * sm_count()), 256, s, P);
}
