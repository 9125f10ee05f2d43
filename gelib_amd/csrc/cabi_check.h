// What the C entry points of the operators on real channels and over points check their arguments with.
#pragma once

#include "real_ops.h"

namespace gelib_hip {

constexpr int64_t kMostElements = 1LL << 46;   // of one tensor: products of two extents below it do not overflow

// both factors are not below zero
inline bool product_ok(int64_t a, int64_t b) { return a == 0 || b <= kMostElements / a; }

inline int check_workspace(const void *ws, uint64_t have, uint64_t need) {
  if (need == 0) return GELIB_HIP_OK;
  if (!ws || have < need || ((uintptr_t)ws & 15)) return GELIB_HIP_ERR_WORKSPACE;
  return check_memory(ws, (int64_t)need);
}

// Collects the first refusal: missing pointers before memory that is not the device's.
struct Memory {
  int missing = GELIB_HIP_OK, foreign = GELIB_HIP_OK;
  void need(const void *p, int64_t bytes, unsigned align) {
    if (bytes == 0 || missing) return;
    if (!p) missing = GELIB_HIP_ERR_NULL;
    else if ((uintptr_t)p % align) missing = GELIB_HIP_ERR_ARG;
    else if (!foreign) foreign = check_memory(p, bytes);
  }
  void may(const void *p, int64_t bytes, unsigned align) {
    if (p) need(p, bytes, align);
  }
  int rc() const { return missing ? missing : foreign; }
};

// what rows of `cols` elements are aligned to: 16 bytes where they are a multiple of it long
inline unsigned row_align(unsigned e, int64_t cols) { return cols * e % 16 == 0 ? 16 : e; }

}  // namespace gelib_hip
