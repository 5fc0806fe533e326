// Host checks of operands: alignment, and buffers that overlap.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace lmoe {

inline bool misaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

struct Span {
  const void* p;
  size_t bytes;
};
inline bool overlap(const Span& a, const Span& b) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(a.p), q = reinterpret_cast<uintptr_t>(b.p);
  return p != 0 && q != 0 && p < q + b.bytes && q < p + a.bytes;
}

}  // namespace lmoe
