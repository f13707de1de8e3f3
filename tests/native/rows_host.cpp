// The overlap checks of voom_b200/csrc/rows.h for the host.  A tensor is eight
// numbers: address, three counts, three strides, run (elements of two bytes).
#include "../../voom_b200/csrc/rows.h"

static voom::Rows rows(const int64_t* v) {
  return voom::Rows{reinterpret_cast<const void*>(v[0]), {v[1], v[2], v[3]}, {v[4], v[5], v[6]}, v[7], 2};
}

extern "C" int rows_separate(const int64_t* a) { return voom::separate(rows(a)); }
extern "C" int rows_disjoint(const int64_t* a, const int64_t* b) { return voom::disjoint(rows(a), rows(b)); }
