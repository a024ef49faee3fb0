// Where rows lie among the vectors of a tensor: plain C++, for the launch code of gn_rms.cu and for tests on the host.
#pragma once
#include <cstdint>

namespace gnb200 {

// Rows at either end of a tensor whose edge vectors may reach out of it.  Vectors of `width` elements begin up to width - 1 elements before a
// row or end as many behind it; a row with as much of the tensor on both sides may be read in whole vectors.  One row at either end where rows are no
// shorter than that, several where they are, or where they overlap.  stride: from row to row, not 0.
inline int edge_rows(int width, int64_t stride) {
  const int64_t step = stride < 0 ? -stride : stride;
  return step < width - 1 ? (int)((width - 1 + step - 1) / (step > 0 ? step : 1)) : 1;
}

}  // namespace gnb200
