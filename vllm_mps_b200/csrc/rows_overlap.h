// Whether two sets of strided rows share memory: host arithmetic that the entry points use to
// refuse outputs in their inputs' place, plain C++ so that it can be checked without a GPU.
#pragma once

#include <stdint.h>

namespace vmps {

// `rows` rows each, from `a` and `b`, their strides and lengths in bytes (strides at least a
// row).  Rows of one buffer that lie beside each other do not overlap.  Strides that differ
// are only told apart where one of the two is contiguous; otherwise rows whose ranges meet
// count as overlapping.
inline bool rows_overlap(const void* a, int64_t a_stride, int64_t a_row, const void* b,
                         int64_t b_stride, int64_t b_row, int64_t rows) {
  if (rows <= 0 || a_row <= 0 || b_row <= 0) return false;
  const int64_t at = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b) -
                                          reinterpret_cast<uintptr_t>(a));
  if (at >= (rows - 1) * a_stride + a_row || -at >= (rows - 1) * b_stride + b_row) return false;
  if (rows == 1) return true;
  // From the start of one of the first's rows: does [from, from + size) stay in its gap?
  auto in_gap = [](int64_t from, int64_t stride, int64_t row, int64_t size) {
    const int64_t d = ((from % stride) + stride) % stride;
    return d >= row && d + size <= stride;
  };
  if (a_stride == b_stride) return !in_gap(at, a_stride, a_row, b_row);
  if (b_stride == b_row && in_gap(at, a_stride, a_row, rows * b_row)) return false;
  if (a_stride == a_row && in_gap(-at, b_stride, b_row, rows * a_row)) return false;
  return true;
}

}  // namespace vmps
