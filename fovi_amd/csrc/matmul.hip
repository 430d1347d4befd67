// Copies of operands whose rows are not whole 16-byte pieces, for the matrix products of matmul.h.
#include "matmul.h"

namespace fovi {

__global__ __launch_bounds__(256) void mat_copy_kernel(MatCopies c) {
  for (int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; id < c.first[c.n]; id += static_cast<int64_t>(gridDim.x) * 256) {
    int i = 0;
    while (id >= c.first[i + 1]) ++i;
    const auto& m = c.m[i];
    const int64_t at = id - c.first[i], pieces = (m.len + 15) / 16, r = at / pieces, p = at - r * pieces;
    *reinterpret_cast<u32x4*>(m.to + at * 16) = mat_piece(m.from + r * m.stride, p * 16, m.len);
  }
}

void MatInputs::copy(hipStream_t s) const {
  const int64_t groups = (copies_.first[copies_.n] + 255) / 256;
  if (groups) mat_copy_kernel<<<static_cast<unsigned>(groups < 16384 ? groups : 16384), 256, 0, s>>>(copies_);
}

}  // namespace fovi
