// tensor_list.cuh — many tensors in one launch: a table of them in the
// kernel's parameters (constant memory, captured with the launch), cut into
// chunks of equal length that blocks find by a binary search.
#pragma once

#include "common.cuh"

namespace frag {

// Tensors of one launch: 512 entries of up to 56 bytes stay below the 32764
// bytes that a kernel's parameters may have; a call with more is several
// launches.  A launch copies its whole parameter block, so lists of up to 32
// take a small one.
constexpr int kListSmall = 32, kListLarge = 512;

// The tensor that holds chunk c: the last one whose first chunk is not beyond
// it (a tensor without values has none).  `first` has `count` + 1 entries.
__device__ __forceinline__ int find_tensor(const uint32_t* first, int count, uint32_t c) {
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= c) lo = mid;
    else hi = mid;
  }
  return lo;
}

}  // namespace frag
