// Whether two pieces of device memory share a byte: rows of `width` bytes, `pitch` apart, as the
// matrices and arrays of a call are given. Host only.
#pragma once

#include <cstdint>
#include <initializer_list>
#include <utility>

namespace ovvs {
namespace rt {

struct Span {
  uint64_t at = 0;  // 0: there is none
  int64_t rows = 0, width = 0, pitch = 0;
};

inline Span span_of(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t bytes) {
  const uint64_t at = reinterpret_cast<uintptr_t>(p);
  if (ld == cols || rows == 1) return {at, 1, rows * cols * bytes, rows * cols * bytes};
  return {at, rows, cols * bytes, ld * bytes};
}
inline Span span_of(const void* p, int64_t count, int64_t bytes) {
  return span_of(p, 1, count, count, bytes);
}

// Exact where one of the two is in one piece or both have the same pitch (two column ranges of one
// buffer share nothing). Of two pitches, which no call here has a use for, only the first row of
// the later one is looked at.
inline bool overlap(Span a, Span b) {
  if (!a.at || !b.at) return false;
  if (b.at < a.at) std::swap(a, b);
  const uint64_t off = b.at - a.at;
  if (off >= static_cast<uint64_t>(a.rows - 1) * a.pitch + a.width) return false;
  // b begins in a row of a, or in the gap before one, which its own rows (the first like all of
  // one pitch) then reach if they are longer than what is left of the gap
  const int64_t in = static_cast<int64_t>(off % a.pitch);
  return in < a.width || b.width > a.pitch - in;
}

// Whether one of the outputs shares memory with another or with an input.
inline bool clash(std::initializer_list<Span> outs, std::initializer_list<Span> ins) {
  for (const Span* o = outs.begin(); o != outs.end(); ++o) {
    for (const Span* p = o + 1; p != outs.end(); ++p)
      if (overlap(*o, *p)) return true;
    for (const Span& i : ins)
      if (overlap(*o, i)) return true;
  }
  return false;
}

}  // namespace rt
}  // namespace ovvs
