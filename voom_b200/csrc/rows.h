// Host checks of the rows that an entry point writes: whether a strided tensor
// names an element twice, and whether two of them share one.
#pragma once

#include <stdint.h>

#include <initializer_list>

namespace voom {

// n[0] x n[1] x .. runs of `run` adjacent elements of `bytes` bytes, s apart.
template <int K>
struct RowsOf {
  const void* at;
  int64_t n[K], s[K];
  int64_t run, bytes;

  bool empty() const {
    for (int64_t x : n)
      if (!x) return true;
    return !run;
  }
};
using Rows = RowsOf<3>;

using Wide = __int128;  // strides and counts are the caller's: products of them pass 64 bits

inline Wide magnitude(int64_t s) { return s < 0 ? -Wide(s) : Wide(s); }

// No element twice: every dimension steps past all that the narrower ones
// cover.  (Refuses a few interleavings that do not overlap; none is a row layout.)
template <int K>
inline bool separate(const RowsOf<K>& x) {
  if (x.empty()) return true;
  bool done[K];
  for (int k = 0; k < K; k++) done[k] = x.n[k] == 1;
  Wide covered = x.run;
  for (;;) {
    int i = -1;
    for (int k = 0; k < K; k++)
      if (!done[k] && (i < 0 || magnitude(x.s[k]) < magnitude(x.s[i]))) i = k;
    if (i < 0) return true;
    if (magnitude(x.s[i]) < covered) return false;
    covered += magnitude(x.s[i]) * (x.n[i] - 1);
    done[i] = true;
  }
}

// The lowest address, and the bytes from it to the end, of the dimensions that
// step less than `below` (0: of all).
template <int K>
inline Wide low(const RowsOf<K>& x) {
  Wide p = Wide(reinterpret_cast<uintptr_t>(x.at));
  for (int k = 0; k < K; k++)
    if (x.s[k] < 0) p += Wide(x.s[k]) * (x.n[k] - 1) * x.bytes;
  return p;
}
template <int K>
inline Wide span(const RowsOf<K>& x, Wide below) {
  Wide n = x.run;
  for (int k = 0; k < K; k++)
    if (!below || magnitude(x.s[k]) * x.bytes < below) n += magnitude(x.s[k]) * (x.n[k] - 1);
  return n * x.bytes;
}
// Every dimension as wide as the period steps a multiple of it.
template <int K>
inline bool fits(const RowsOf<K>& x, Wide period) {
  for (int k = 0; k < K; k++)
    if (x.n[k] > 1 && magnitude(x.s[k]) * x.bytes >= period && magnitude(x.s[k]) * x.bytes % period) return false;
  return true;
}

// No element in both: their address ranges are apart, or they are parts of one
// layout with a period (the tokens of a fused projection): every wider stride
// of both is a multiple of it, and within it the two lie side by side.
template <int K, int L>
inline bool disjoint(const RowsOf<K>& a, const RowsOf<L>& b) {
  if (a.empty() || b.empty()) return true;
  const Wide la = low(a), lb = low(b);
  if (la + span(a, 0) <= lb || lb + span(b, 0) <= la) return true;
  auto side_by_side = [&](Wide period) {
    if (!period || !fits(a, period) || !fits(b, period)) return false;
    Wide r = (lb - la) % period;
    if (r < 0) r += period;
    return r >= span(a, period) && r + span(b, period) <= period;
  };
  for (int k = 0; k < K; k++)
    if (a.n[k] != 1 && side_by_side(magnitude(a.s[k]) * a.bytes)) return true;
  for (int k = 0; k < L; k++)
    if (b.n[k] != 1 && side_by_side(magnitude(b.s[k]) * b.bytes)) return true;
  return false;
}

// (for arguments in braces)
inline bool separate(const Rows& x) { return separate<3>(x); }
inline bool disjoint(const Rows& a, const Rows& b) { return disjoint<3, 3>(a, b); }

inline bool same_place(const Rows& a, const Rows& b) {
  if (a.at != b.at || a.run != b.run || a.bytes != b.bytes) return false;
  for (int k = 0; k < 3; k++)
    if (a.n[k] != b.n[k] || (a.n[k] > 1 && a.s[k] != b.s[k])) return false;
  return true;
}

}  // namespace voom
