// Host side of the serving operators: whether buffers of a call share memory. A start address alone does not say so -
// two views of one buffer may begin at different elements.
#pragma once
#include <stdint.h>

// `rows` rows of `bytes` bytes, `stride` bytes apart (0: all rows are one).
struct Span {
  const void* p;
  long long rows, bytes, stride;
};
inline Span span(const void* p, long long bytes) { return Span{p, 1, bytes, bytes}; }
inline Span span_rows(const void* p, long long rows, long long bytes, long long stride) {
  return Span{p, stride == 0 && rows > 1 ? 1 : rows, bytes, stride};
}

// Exact, also for rows that lie in each other's gaps. Rows are searched only where the whole ranges meet and the strides
// differ.
inline bool spans_meet(const Span& x, const Span& y) {
  if (!x.p || !y.p || x.rows <= 0 || y.rows <= 0 || x.bytes <= 0 || y.bytes <= 0) return false;
  const uintptr_t xp = reinterpret_cast<uintptr_t>(x.p), yp = reinterpret_cast<uintptr_t>(y.p);
  if (xp + (x.rows - 1) * x.stride + x.bytes <= yp || yp + (y.rows - 1) * y.stride + y.bytes <= xp) return false;
  const Span &a = x.rows <= y.rows ? x : y, &b = x.rows <= y.rows ? y : x;
  const long long ap = (long long)(reinterpret_cast<uintptr_t>(a.p) - reinterpret_cast<uintptr_t>(b.p));
  if (a.stride == b.stride && a.bytes <= a.stride && b.bytes <= b.stride) {
    // row i of a lies `ap + (i - j) * stride` behind row j of b: less than a stride for two neighbouring i - j at most
    const long long near = -ap / a.stride;
    for (long long k = near - 1; k <= near + 1; ++k) {
      const long long at = ap + k * a.stride;
      if (k > -b.rows && k < a.rows && at < b.bytes && at + a.bytes > 0) return true;
    }
    return false;
  }
  for (long long i = 0; i < a.rows; ++i) {
    const long long from = ap + i * a.stride, to = from + a.bytes;  // relative to b's first row
    // the first row of b that ends behind `from`
    const long long over = from - b.bytes;
    const long long r = over < 0 || b.rows == 1 ? 0 : over / b.stride + 1;
    if (r < b.rows && r * b.stride < to && r * b.stride + b.bytes > from) return true;
  }
  return false;
}

// whether an output shares memory with another buffer of the call
template <int O, int I>
inline bool outputs_shared(const Span (&out)[O], const Span (&in)[I]) {
  for (int i = 0; i < O; ++i) {
    for (int j = i + 1; j < O; ++j)
      if (spans_meet(out[i], out[j])) return true;
    for (int j = 0; j < I; ++j)
      if (spans_meet(out[i], in[j])) return true;
  }
  return false;
}
