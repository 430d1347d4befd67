// Copies of operands whose rows are not whole 16-byte pieces, for the matrix products of matmul.h.
#include "matmul.h"

namespace fovi {

__global__ __launch_bounds__(256) void mat_copy_kernel(MatCopies c) {
  for (int i = 0; i < c.n; ++i) {
    const auto& m = c.m[i];
    const int64_t pieces = (m.len + 15) / 16, all = m.rows * pieces;
    for (int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; id < all; id += static_cast<int64_t>(gridDim.x) * 256) {
      const int64_t r = id / pieces, p = id - r * pieces;
      *reinterpret_cast<u32x4*>(m.to + id * 16) = mat_piece(m.from + r * m.stride, p * 16, m.len);
    }
  }
}

void MatInputs::copy(hipStream_t s) const {
  int64_t most = 0;
  for (int i = 0; i < copies_.n; ++i) {
    const int64_t n = (copies_.m[i].rows * ((copies_.m[i].len + 15) / 16) + 255) / 256;
    if (n > most) most = n;
  }
  if (most) mat_copy_kernel<<<static_cast<unsigned>(most < 4096 ? most : 4096), 256, 0, s>>>(copies_);
}

}  // namespace fovi
