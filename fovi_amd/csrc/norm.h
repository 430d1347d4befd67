// What the row norms share: rows in 16-byte pieces at any alignment, sums over groups of lanes, and the shape of a call.
#pragma once

#include "common.h"

namespace fovi {

__device__ __forceinline__ float norm_param(const void* p, int64_t c, int bf16, float none) {
  if (!p) return none;
  return bf16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(p)[c]) : static_cast<const float*>(p)[c];
}

// Sum over the workgroup of 256; every thread gets the result.
__device__ __forceinline__ float block_sum(float v, float* sh) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// VEC adjacent channels (16 bytes) from c on as floats; zeros from C on. The accesses need no alignment, so
// that rows of any width and offset come in whole pieces. short_piece (a constant): the piece may pass the
// end of the row; then it is read as the row's last 16 bytes and shifted down (reading it by elements cost
// rows of 385 bf16 channels 15 %), and written in parts of 8, 4 and 2 bytes.
template <typename T, int VEC>
__device__ __forceinline__ void norm_load(const T* row, int64_t c, int64_t C, float (&v)[VEC], bool short_piece) {
  T e[VEC];
  if (!short_piece) {
    u32x4 u = {0, 0, 0, 0};
    if (c < C) __builtin_memcpy(&u, row + c, 16);
    __builtin_memcpy(e, &u, sizeof(e));
  } else if (C >= VEC) {
    const int64_t at = c + VEC <= C ? c : C - VEC;
    u32x4 u;
    __builtin_memcpy(&u, row + at, 16);
    uint64_t w[2];
    __builtin_memcpy(w, &u, 16);
    const int64_t over = (c - at) * 8 * static_cast<int>(sizeof(T));
    const int bits = static_cast<int>(over) & 63;
    if (over >= 64) { w[0] = over < 128 ? w[1] : 0; w[1] = 0; }
    w[0] = (w[0] >> bits) | (w[1] << 1 << (63 - bits));
    w[1] >>= bits;
    __builtin_memcpy(e, w, sizeof(e));
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = c + i < C ? row[c + i] : T(0);
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = Elem<T>::load(e + i);
}
template <typename T, int VEC>
__device__ __forceinline__ void norm_store(T* row, int64_t c, int64_t C, const float (&v)[VEC], bool short_piece) {
  T e[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) Elem<T>::store(e + i, v[i]);
  if (c + (short_piece ? VEC - 1 : 0) < C) {
    u32x4 u;
    __builtin_memcpy(&u, e, sizeof(e));
    __builtin_memcpy(row + c, &u, 16);
  } else if (short_piece && c < C) {
    T* at = row + c;
    const int n = static_cast<int>(C - c);
    uint64_t w[2];
    __builtin_memcpy(w, e, sizeof(e));
    if (n * sizeof(T) & 8) { __builtin_memcpy(at, w, 8); at += 8 / sizeof(T); w[0] = w[1]; }
    if (n * sizeof(T) & 4) { __builtin_memcpy(at, w, 4); at += 4 / sizeof(T); w[0] >>= 32; }
    if (n * sizeof(T) & 2) __builtin_memcpy(at, w, 2);
  }
}

// VEC parameters from channel c on (wide loads: a workgroup's first work), `none` without any.
template <int VEC>
__device__ __forceinline__ void norm_params_at(const void* p, int64_t c, int64_t C, int bf16, float none, float (&v)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = none;
  if (!p || c >= C) return;
  if (c + VEC > C) {
#pragma unroll
    for (int i = 0; i < VEC - 1; ++i)
      if (c + i < C) v[i] = norm_param(p, c + i, bf16, none);
  } else if (bf16) {
    uint16_t e[VEC];
    __builtin_memcpy(e, static_cast<const uint16_t*>(p) + c, sizeof(e));
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = bf16_bits_to_f32(e[i]);
  } else {
    __builtin_memcpy(v, static_cast<const float*>(p) + c, sizeof(v));
  }
}

// Sum over a group of LANES; every lane gets the result.
template <int LANES>
__device__ __forceinline__ float group_sum(float v, float* sh) {
  if (LANES == 256) return block_sum(v, sh);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// The shape of a call: the lanes of a row and the 16-byte pieces a lane holds (nv 0: too wide for registers).
// Rows of up to 64 pieces take 16 lanes (4 rows a wave: a shorter reduction, no idle lanes at 48 pieces),
// unless there are too few rows to fill the card that way. Rows that are not whole pieces take pieces too
// (element by element, 60000 bf16 rows of 385 took 39 and 133 us forward and backward, now 26 and 35; fp32
// rows of 771 take 13 and 18 us either way within 10 %).
struct NormPlan { bool tail; int lanes, nv; };

inline NormPlan norm_plan(int64_t rows, int64_t C, int es) {
  NormPlan f;
  f.tail = C * es % 16 != 0;
  const int64_t n = (C * es + 15) / 16;
  f.lanes = n <= 64 ? (rows >= 4096 ? 16 : 64) : n <= 256 ? 64 : 256;
  f.nv = n <= 1024 ? static_cast<int>((n + f.lanes - 1) / f.lanes) : 0;
  return f;
}

inline int64_t norm_groups(int64_t rows, const NormPlan& f, int64_t most) {
  const int64_t per = 256 / f.lanes, n = (rows + per - 1) / per;
  return n < most ? n : most;
}

inline int64_t norm_chunks(int64_t rows, int64_t C) {
  const int64_t cols = (C + 63) / 64;
  int64_t chunks = (1024 + cols - 1) / cols;        // about four workgroups a compute unit
  if (chunks > (rows + 15) / 16) chunks = (rows + 15) / 16;
  return chunks < 1 ? 1 : chunks;
}

// Workgroups of `columns` columns each, by `y`: along x no more than 2^20, the rest along z. (A launch whose threads along one
// dimension pass 2^32 runs without an error, and without the threads in excess: a workgroup for every 8 of 2^27 columns.)
inline dim3 norm_grid(int64_t C, int columns, int64_t y) {
  const int64_t n = (C + columns - 1) / columns, most = 1 << 20;
  return dim3(static_cast<unsigned>(n < most ? n : most), static_cast<unsigned>(y), static_cast<unsigned>((n + most - 1) / most));
}
__device__ __forceinline__ int64_t norm_group() { return static_cast<int64_t>(blockIdx.z) * gridDim.x + blockIdx.x; }

// CALL(lanes, pieces, short last piece) of a plan.
#define FOVI_NORM_TAIL(CALL, L, N) \
  if (f.tail) CALL(L, N, true) else CALL(L, N, false)
#define FOVI_NORM_CASES(CALL)                                                                            \
  if (f.lanes == 16) {                                                                                   \
    if (f.nv == 1) { FOVI_NORM_TAIL(CALL, 16, 1) } else if (f.nv == 2) { FOVI_NORM_TAIL(CALL, 16, 2) }   \
    else if (f.nv == 3) { FOVI_NORM_TAIL(CALL, 16, 3) } else { FOVI_NORM_TAIL(CALL, 16, 4) }             \
  } else if (f.lanes == 64) {                                                                            \
    if (f.nv == 1) { FOVI_NORM_TAIL(CALL, 64, 1) } else if (f.nv == 2) { FOVI_NORM_TAIL(CALL, 64, 2) }   \
    else if (f.nv == 3) { FOVI_NORM_TAIL(CALL, 64, 3) } else { FOVI_NORM_TAIL(CALL, 64, 4) }             \
  } else {                                                                                               \
    if (f.nv == 2) { FOVI_NORM_TAIL(CALL, 256, 2) } else if (f.nv == 3) { FOVI_NORM_TAIL(CALL, 256, 3) } \
    else { FOVI_NORM_TAIL(CALL, 256, 4) }                                                                \
  }

}  // namespace fovi
