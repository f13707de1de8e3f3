// Host checks of the rows that an entry point writes: whether a strided tensor
// names an element twice, and whether two of them share one.
#pragma once

#include <stdint.h>

#include <initializer_list>

namespace voom {

// n[0] x n[1] x n[2] runs of `run` adjacent elements of `bytes` bytes, s apart.
struct Rows {
  const void* at;
  int64_t n[3], s[3];
  int64_t run, bytes;

  bool empty() const { return !n[0] || !n[1] || !n[2] || !run; }
};

using Wide = __int128;  // strides and counts are the caller's: products of them pass 64 bits

inline Wide magnitude(int64_t s) { return s < 0 ? -Wide(s) : Wide(s); }

// No element twice: every dimension steps past all that the narrower ones
// cover.  (Refuses a few interleavings that do not overlap; none is a row layout.)
inline bool separate(const Rows& x) {
  if (x.empty()) return true;
  bool done[3] = {x.n[0] == 1, x.n[1] == 1, x.n[2] == 1};
  Wide covered = x.run;
  for (;;) {
    int i = -1;
    for (int k = 0; k < 3; k++)
      if (!done[k] && (i < 0 || magnitude(x.s[k]) < magnitude(x.s[i]))) i = k;
    if (i < 0) return true;
    if (magnitude(x.s[i]) < covered) return false;
    covered += magnitude(x.s[i]) * (x.n[i] - 1);
    done[i] = true;
  }
}

// No element in both: their address ranges are apart, or they are parts of one
// layout with a period (the tokens of a fused projection): every wider stride
// of both is a multiple of it, and within it the two lie side by side.
inline bool disjoint(const Rows& a, const Rows& b) {
  if (a.empty() || b.empty()) return true;
  auto low = [](const Rows& x) {  // lowest address
    Wide p = Wide(reinterpret_cast<uintptr_t>(x.at));
    for (int k = 0; k < 3; k++)
      if (x.s[k] < 0) p += Wide(x.s[k]) * (x.n[k] - 1) * x.bytes;
    return p;
  };
  // bytes from the lowest address to the end, of the dimensions that step less than `below` (0: of all)
  auto span = [](const Rows& x, Wide below) {
    Wide n = x.run;
    for (int k = 0; k < 3; k++)
      if (!below || magnitude(x.s[k]) * x.bytes < below) n += magnitude(x.s[k]) * (x.n[k] - 1);
    return n * x.bytes;
  };
  const Wide la = low(a), lb = low(b);
  if (la + span(a, 0) <= lb || lb + span(b, 0) <= la) return true;
  auto fits = [](const Rows& x, Wide period) {
    for (int k = 0; k < 3; k++)
      if (x.n[k] > 1 && magnitude(x.s[k]) * x.bytes >= period && magnitude(x.s[k]) * x.bytes % period) return false;
    return true;
  };
  for (const Rows* x : {&a, &b})
    for (int k = 0; k < 3; k++) {
      const Wide period = magnitude(x->s[k]) * x->bytes;
      if (x->n[k] == 1 || !period || !fits(a, period) || !fits(b, period)) continue;
      Wide r = (lb - la) % period;
      if (r < 0) r += period;
      if (r >= span(a, period) && r + span(b, period) <= period) return true;
    }
  return false;
}

inline bool same_place(const Rows& a, const Rows& b) {
  if (a.at != b.at || a.run != b.run || a.bytes != b.bytes) return false;
  for (int k = 0; k < 3; k++)
    if (a.n[k] != b.n[k] || (a.n[k] > 1 && a.s[k] != b.s[k])) return false;
  return true;
}

}  // namespace voom
