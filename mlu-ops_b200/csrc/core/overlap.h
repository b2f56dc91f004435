// Whether two ranges of memory share a byte: outputs that may not lie on inputs are refused before a launch.
#ifndef MLUOP_B200_CORE_OVERLAP_H_
#define MLUOP_B200_CORE_OVERLAP_H_

#include <cstddef>
#include <initializer_list>

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
// A tensor of a call (descriptor null: the call has none) or its workspace.
struct Span {
  const void *p;
  size_t bytes;
  Span(const void *p, size_t bytes) : p(p), bytes(p ? bytes : 0) {}
  Span(const mluOpTensorDescriptor_t desc, const void *p) : Span(p, desc ? denseBytes(desc) : 0) {}
};
// Whether no two of `written` share a byte, nor one of them and one of `read`.
inline bool writtenApart(std::initializer_list<Span> written, std::initializer_list<Span> read) {
  for (const Span *a = written.begin(); a != written.end(); ++a) {
    for (const Span *b = written.begin(); b != a; ++b)
      if (overlap(a->p, a->bytes, b->p, b->bytes)) return false;
    for (const Span &b : read)
      if (overlap(a->p, a->bytes, b.p, b.bytes)) return false;
  }
  return true;
}

}  // namespace mluop

#endif  // MLUOP_B200_CORE_OVERLAP_H_
