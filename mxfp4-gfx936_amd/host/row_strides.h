// Tensors [.., n] whose rows one stride steps through.
#pragma once
#include <cstdint>

namespace mx {

// Element (i, b) of a tensor [.., n], its leading dimensions taken together, lies at i * row
// + b * block.
struct RowStrides {
  int64_t row = 1, block = 1;

  // False: no two positive strides say where all of the tensor's values lie.
  bool read(const int64_t* sizes, const int64_t* strides, int64_t dims) {
    block = sizes[dims - 1] > 1 ? strides[dims - 1] : 1;
    if (block < 1) return false;
    int64_t next = 0;  // the stride that the next outer dimension must have; 0: any
    for (int64_t d = dims - 2; d >= 0; --d) {
      if (sizes[d] == 1) continue;
      if (strides[d] < 1) return false;  // expanded: no stride reaches its rows
      if (next == 0) row = strides[d];
      else if (strides[d] != next) return false;
      next = strides[d] * sizes[d];
    }
    return true;
  }
};

}  // namespace mx
