// Whether two ranges of memory share a byte: outputs that may not lie on inputs are refused before a launch.
#ifndef MLUOP_B200_CORE_OVERLAP_H_
#define MLUOP_B200_CORE_OVERLAP_H_

#include <cstddef>

#include "core/tensor.h"
#include "core/type.h"

namespace mluop {

inline bool overlap(const void *a, size_t a_bytes, const void *b, size_t b_bytes) {
  const size_t x = reinterpret_cast<size_t>(a), y = reinterpret_cast<size_t>(b);
  return a_bytes > 0 && b_bytes > 0 && x < y + b_bytes && y < x + a_bytes;
}
inline size_t denseBytes(const mluOpTensorDescriptor_t desc) {
  return (size_t)mluOpGetTensorElementNum(desc) * getSizeOfDataType(desc->getDtype());
}

}  // namespace mluop

#endif  // MLUOP_B200_CORE_OVERLAP_H_
