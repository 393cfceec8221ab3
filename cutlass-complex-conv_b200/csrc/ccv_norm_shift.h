// Which elements layer norm's shifted vectors read (dense rows of odd width):
// plain arithmetic, compiled for the kernels and for the host.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define CCV_HD __host__ __device__ __forceinline__
#else
#define CCV_HD inline
#endif

namespace ccv {

// Whether rows of this width can be read as shifted vectors of v.  A vector
// that begins in its row ends at most v - 1 elements behind it.  The last row
// is fetched element by element there; a row before it must find that many
// elements in the one row that is sure to follow.
CCV_HD bool shift_fits(int64_t features, int v) { return features >= v - 1; }

// Element of a vector of v at which row `row` begins.
CCV_HD int shift_of_row(int64_t row, int features, int v) {
  return static_cast<int>(row * features % v);
}

// Column of the row at which a lane's vector i begins (negative: in the row
// before).
CCV_HD int shifted_column(int i, int g, int lane, int v, int shift) {
  return (i * g + lane) * v - shift;
}

// Whether the vector at column c of row r reaches past the tensor and is
// fetched element by element, the row's own elements only.
CCV_HD bool past_the_end(int64_t r, int64_t rows, int c, int features, int v) {
  return r == rows - 1 && c + v > features;
}

}  // namespace ccv
