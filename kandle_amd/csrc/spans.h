// Whether the memory that a call writes is also what it reads, or what it writes elsewhere (host side).
#pragma once

#include <cstdint>
#include <initializer_list>

namespace kh {

// Runs of `bytes` at `at`, repeated count[i] times every step[i] bytes (a tensor's outer dimensions).
struct Span {
  int64_t bytes, count[3], step[3];
  int64_t low = 0, high = 0;  // its first byte and the one behind its last; equal: no byte

  Span(const void* at, int64_t run, int64_t n0 = 1, int64_t s0 = 0, int64_t n1 = 1, int64_t s1 = 0, int64_t n2 = 1, int64_t s2 = 0)
      : bytes(run), count{n0, n1, n2}, step{s0, s1, s2} {
    if (at == nullptr || run <= 0 || n0 <= 0 || n1 <= 0 || n2 <= 0) return;
    low = (int64_t)(uintptr_t)at;
    high = low + run;
    for (int i = 0; i < 3; ++i) {
      int64_t far;
      if (__builtin_mul_overflow(count[i] - 1, step[i], &far)) far = step[i] < 0 ? INT64_MIN : INT64_MAX;
      int64_t& end = far < 0 ? low : high;
      if (__builtin_add_overflow(end, far, &end)) end = far < 0 ? INT64_MIN : INT64_MAX;
    }
  }
  // The bytes that it takes from its lowest address on, but for the repeats in whole multiples of s.
  __int128 within(int64_t s) const {
    __int128 x = bytes;
    for (int i = 0; i < 3; ++i)
      if (step[i] % s != 0) x += (__int128)(count[i] - 1) * (step[i] < 0 ? -(__int128)step[i] : step[i]);
    return x;
  }
};

// Whether two spans share no byte, as far as can be told: they do not reach each other, or for one of their steps s the
// addresses modulo s lie in intervals that do not meet (heads of one buffer, keys and values side by side).
inline bool apart(const Span& a, const Span& b) {
  if (a.low == a.high || b.low == b.high || a.high <= b.low || b.high <= a.low) return true;
  for (const Span* x : {&a, &b})
    for (int i = 0; i < 3; ++i) {
      const int64_t s = x->step[i] < 0 ? -x->step[i] : x->step[i];
      if (x->count[i] < 2 || s == 0) continue;
      const __int128 na = a.within(s), nb = b.within(s);
      __int128 d = ((__int128)b.low - a.low) % s;
      if (d < 0) d += s;
      if (d >= na && d + nb <= s) return true;
    }
  return false;
}

// Whether any of the memory that a call writes may be what it reads, or other memory that it writes.
inline bool overlap(std::initializer_list<Span> written, std::initializer_list<Span> read) {
  for (const Span& a : written) {
    for (const Span& b : read)
      if (!apart(a, b)) return true;
    for (const Span& b : written)
      if (&a < &b && !apart(a, b)) return true;
  }
  return false;
}

// Of n int32 values; of a page table.
inline Span ints(const void* at, int64_t n) { return Span(at, 4 * n); }
inline Span table_span(const int32_t* at, int64_t stride, int64_t rows, int64_t width) {
  return Span(at, 4 * width, rows, 4 * stride);
}

}  // namespace kh
