// RMS norm over the channels of token rows, with the residual's addition in front: forward (in the rows' type, or
// in 8 bits with a scale a row), and the gradients of rows and weight.
//
//   t = round(x + residual), rstd = 1 / sqrt(mean(t^2) + eps), y = t * rstd * w
//   dt = dtotal + rstd * (g - h * mean(g * h)), g = dy * w, h = t * rstd; dw = sum dy * h
//   8 bits: scale = max|y| / 127, q = rint(y / scale)
//
// Bound by memory. As in the layer norm a row is read once into the registers of a group of lanes (16, 64 or 256):
// the sum, its rounding, the mean of squares, the largest value and the quantised row all come from there. The
// backward keeps the weight's sums of its rows in registers too; each workgroup leaves one row of them, which a
// second launch adds in a fixed order. Rows too wide for registers go through kernels of a workgroup per row.
//
// 131072 bf16 rows of 384 with a residual: forward 68 us (403 MB, 5.9 TB/s), backward 83 (403 MB, 4.9 TB/s) and 5 for the
// join; 32768 of 1024 to 8 bits 48 us (235 MB, 4.9 TB/s), 7421 fp32 rows of 771 11 and 16 us.
#include "norm.h"

namespace fovi {

struct RmsParams {
  const void* x; const void* r; const void* w;
  void* total; void* y; int8_t* q; float* scale; float* rstd;
  const void* dy; const void* dtotal; void* dx;
  int64_t rows0, rows1, C;
  int64_t xs[2], rs[2], dys[2], dts[2];
  float eps;
  int p_bf16, norm;
};

// Largest bit pattern of |v| over a group of LANES: unsigned order is the order of the values, with infinity and
// then NaN on top, so that neither is lost.
template <int LANES>
__device__ __forceinline__ uint32_t group_max(uint32_t v, uint32_t* sh) {
#pragma unroll
  for (int o = (LANES < 64 ? LANES : 64) / 2; o > 0; o >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o)));
  if (LANES < 256) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return max(max(sh[0], sh[1]), max(sh[2], sh[3]));
}

// A row's step, and the numbers that its values are multiplied by: first `up`, a power of two (1 but for rows whose
// largest value is so small that 127 over it would be infinite), then `inv`. A row without a finite largest
// value is 0 times a step that is not finite: NaN, as such rows are.
struct Quantum {
  float scale, up, inv;
  __device__ __forceinline__ explicit Quantum(uint32_t top) {
    const float m = __uint_as_float(top);
    scale = m / 127.0f;
    up = m < 0x1p-64f ? 0x1p64f : 1.0f;
    inv = top > 0 && top < 0x7f800000u ? 127.0f / (m * up) : 0.0f;
  }
  __device__ __forceinline__ int8_t operator()(float v) const {
    return inv > 0 ? static_cast<int8_t>(static_cast<int>(rintf(v * up * inv))) : static_cast<int8_t>(0);
  }
};

// 1 / sqrt(mean of squares + eps). Where the squares' sum has passed fp32's range (values beyond 1.8e19 / sqrt(C)), from
// scaled_mean(), that of the values times 2^-80: exact for those that count, and finite for any finite row. A row with
// an infinity stays infinite. All lanes of a row have the same mean, so that they go the same way.
template <typename ScaledMean>
__device__ __forceinline__ float rms_rstd(float mean, float eps, const ScaledMean& scaled_mean) {
  if (mean != INFINITY) return 1.0f / sqrtf(mean + eps);
  return 0x1p-80f / sqrtf(scaled_mean() + eps * 0x1p-80f * 0x1p-80f);
}
__device__ __forceinline__ float scaled_square(float v, float s) {
  v *= 0x1p-80f;
  return fmaf(v, v, s);
}

template <typename T> __device__ __forceinline__ float round_to(float v) { T e; Elem<T>::store(&e, v); return Elem<T>::load(&e); }

template <typename T, int VEC, int LANES, int NV, bool TAIL, bool INT8>
__global__ __launch_bounds__(256) void rms_fwd_rows_kernel(RmsParams p) {
  __shared__ float sh[4];
  __shared__ uint32_t shm[4];
  const int lane = threadIdx.x % LANES;
  float w[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k)
    norm_params_at<VEC>(p.w, static_cast<int64_t>(lane + k * LANES) * VEC, p.C, p.p_bf16, 1.0f, w[k]);
  const float n = 1.0f / static_cast<float>(p.C);
  const int64_t rows = p.rows0 * p.rows1, step = static_cast<int64_t>(gridDim.x) * (256 / LANES);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES; row < rows; row += step) {
    const int64_t i0 = p.rows0 == 1 ? 0 : row / p.rows1, i1 = row - i0 * p.rows1;
    const T* xr = static_cast<const T*>(p.x) + i0 * p.xs[0] + i1 * p.xs[1];
    float x[NV][VEC], s = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) norm_load<T, VEC>(xr, static_cast<int64_t>(lane + k * LANES) * VEC, p.C, x[k], TAIL && k == NV - 1);
    if (p.r) {
      const T* rr = static_cast<const T*>(p.r) + i0 * p.rs[0] + i1 * p.rs[1];
      T* tr = static_cast<T*>(p.total) + row * p.C;
      float r[NV][VEC];
#pragma unroll
      for (int k = 0; k < NV; ++k) norm_load<T, VEC>(rr, static_cast<int64_t>(lane + k * LANES) * VEC, p.C, r[k], TAIL && k == NV - 1);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[k][i] = round_to<T>(x[k][i] + r[k][i]);
        norm_store<T, VEC>(tr, static_cast<int64_t>(lane + k * LANES) * VEC, p.C, x[k], TAIL && k == NV - 1);
      }
    }
    float rstd = 1.0f;
    if (!INT8 || p.norm) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) s = fmaf(x[k][i], x[k][i], s);
      rstd = rms_rstd(group_sum<LANES>(s, sh) * n, p.eps, [&]() __attribute__((always_inline)) {
        float t = 0;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int i = 0; i < VEC; ++i) t = scaled_square(x[k][i], t);
        return group_sum<LANES>(t, sh) * n;
      });
      if (lane == 0 && p.rstd) p.rstd[row] = rstd;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[k][i] = x[k][i] * rstd * w[k][i];
    if (!INT8) {
      T* yr = static_cast<T*>(p.y) + row * p.C;
#pragma unroll
      for (int k = 0; k < NV; ++k)
        norm_store<T, VEC>(yr, static_cast<int64_t>(lane + k * LANES) * VEC, p.C, x[k], TAIL && k == NV - 1);
      continue;
    }
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if ((lane + k * LANES) * VEC + (TAIL ? i : 0) < p.C) top = max(top, __float_as_uint(x[k][i]) & 0x7fffffffu);
    const Quantum quantum(group_max<LANES>(top, shm));
    if (lane == 0) p.scale[row] = quantum.scale;
    int8_t* qr = p.q + row * p.C;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = static_cast<int64_t>(lane + k * LANES) * VEC;
      int8_t e[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[i] = quantum(x[k][i]);
      if (c + (TAIL && k == NV - 1 ? VEC - 1 : 0) < p.C) {
        __builtin_memcpy(qr + c, e, VEC);
      } else if (TAIL && k == NV - 1 && c < p.C) {
#pragma unroll
        for (int i = 0; i < VEC - 1; ++i)
          if (c + i < p.C) qr[c + i] = e[i];
      }
    }
  }
}

// dt of the rows and, with `partial`, the workgroup's sums of dy * h: partial[block * C + c].
template <typename T, int VEC, int LANES, int NV, bool TAIL>
__global__ __launch_bounds__(256) void rms_bwd_rows_kernel(RmsParams p, float* partial) {
  __shared__ float sh[4];
  const int lane = threadIdx.x % LANES;
  float w[NV][VEC], dw[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    norm_params_at<VEC>(p.w, static_cast<int64_t>(lane + k * LANES) * VEC, p.C, p.p_bf16, 1.0f, w[k]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[k][i] = 0;
  }
  const float n = 1.0f / static_cast<float>(p.C);
  const int64_t rows = p.rows0 * p.rows1, step = static_cast<int64_t>(gridDim.x) * (256 / LANES);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES; row < rows; row += step) {
    const int64_t i0 = p.rows0 == 1 ? 0 : row / p.rows1, i1 = row - i0 * p.rows1;
    const T* xr = static_cast<const T*>(p.x) + i0 * p.xs[0] + i1 * p.xs[1];
    const T* gr = static_cast<const T*>(p.dy) + i0 * p.dys[0] + i1 * p.dys[1];
    const float rstd = p.rstd[row];
    float h[NV][VEC], g[NV][VEC], sgh = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = static_cast<int64_t>(lane + k * LANES) * VEC;
      norm_load<T, VEC>(xr, c, p.C, h[k], TAIL && k == NV - 1);
      norm_load<T, VEC>(gr, c, p.C, g[k], TAIL && k == NV - 1);
    }
    // read ahead of the sums, which wait for what was read so far
    float d[NV][VEC];
    if (p.dx && p.dtotal) {
      const T* dr = static_cast<const T*>(p.dtotal) + i0 * p.dts[0] + i1 * p.dts[1];
#pragma unroll
      for (int k = 0; k < NV; ++k) norm_load<T, VEC>(dr, static_cast<int64_t>(lane + k * LANES) * VEC, p.C, d[k], TAIL && k == NV - 1);
    } else {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) d[k][i] = 0;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        h[k][i] *= rstd;
        dw[k][i] = fmaf(g[k][i], h[k][i], dw[k][i]);
        g[k][i] *= w[k][i];
        sgh = fmaf(g[k][i], h[k][i], sgh);
      }
    if (!p.dx) continue;
    sgh = group_sum<LANES>(sgh, sh) * n;
    T* dxr = static_cast<T*>(p.dx) + row * p.C;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) d[k][i] = fmaf(rstd, g[k][i] - h[k][i] * sgh, d[k][i]);
      norm_store<T, VEC>(dxr, static_cast<int64_t>(lane + k * LANES) * VEC, p.C, d[k], TAIL && k == NV - 1);
    }
  }
  if (!partial) return;
  float* out = partial + static_cast<int64_t>(blockIdx.x) * p.C;
  if (LANES == 256) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = static_cast<int64_t>(lane + k * LANES) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (c + i < p.C) out[c + i] = dw[k][i];
    }
    return;
  }
  // the groups of a wave by shuffles, the waves through LDS
  constexpr int WIDTH = LANES * NV * VEC;
  extern __shared__ float sums[];                    // [4][WIDTH]
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float a = dw[k][i];
#pragma unroll
      for (int o = 32; o >= LANES; o >>= 1) a += __shfl_xor(a, o);
      if ((threadIdx.x & 63) < LANES) sums[wave * WIDTH + (lane + k * LANES) * VEC + i] = a;
    }
  __syncthreads();
  for (int at = threadIdx.x; at < WIDTH && at < p.C; at += 256)
    out[at] = (sums[at] + sums[WIDTH + at]) + (sums[2 * WIDTH + at] + sums[3 * WIDTH + at]);
}

template <typename T, bool INT8>
__global__ __launch_bounds__(256) void rms_fwd_kernel(RmsParams p) {
  __shared__ float sh[4];
  __shared__ uint32_t shm[4];
  for (int64_t row = blockIdx.x; row < p.rows0 * p.rows1; row += gridDim.x) {
    const int64_t i0 = row / p.rows1, i1 = row - i0 * p.rows1;
    const T* x = static_cast<const T*>(p.x) + i0 * p.xs[0] + i1 * p.xs[1];
    const T* r = p.r ? static_cast<const T*>(p.r) + i0 * p.rs[0] + i1 * p.rs[1] : nullptr;
    T* total = static_cast<T*>(p.total) + row * p.C;
    float s = 0;
    for (int64_t c = threadIdx.x; c < p.C; c += 256) {
      float t = Elem<T>::load(x + c);
      if (r) {
        t = round_to<T>(t + Elem<T>::load(r + c));
        Elem<T>::store(total + c, t);
      }
      s = fmaf(t, t, s);
    }
    const T* from = r ? total : x;                    // each thread reads the places that it wrote
    float rstd = 1.0f;
    if (!INT8 || p.norm) {
      rstd = rms_rstd(block_sum(s, sh) / static_cast<float>(p.C), p.eps, [&]() __attribute__((always_inline)) {
        float t = 0;
        for (int64_t c = threadIdx.x; c < p.C; c += 256) t = scaled_square(Elem<T>::load(from + c), t);
        return block_sum(t, sh) / static_cast<float>(p.C);
      });
      if (threadIdx.x == 0 && p.rstd) p.rstd[row] = rstd;
    }
    if (!INT8) {
      for (int64_t c = threadIdx.x; c < p.C; c += 256)
        Elem<T>::store(static_cast<T*>(p.y) + row * p.C + c, Elem<T>::load(from + c) * rstd * norm_param(p.w, c, p.p_bf16, 1.0f));
      continue;
    }
    uint32_t top = 0;
    for (int64_t c = threadIdx.x; c < p.C; c += 256)
      top = max(top, __float_as_uint(Elem<T>::load(from + c) * rstd * norm_param(p.w, c, p.p_bf16, 1.0f)) & 0x7fffffffu);
    const Quantum quantum(group_max<256>(top, shm));
    if (threadIdx.x == 0) p.scale[row] = quantum.scale;
    for (int64_t c = threadIdx.x; c < p.C; c += 256)
      p.q[row * p.C + c] = quantum(Elem<T>::load(from + c) * rstd * norm_param(p.w, c, p.p_bf16, 1.0f));
  }
}

template <typename T>
__global__ __launch_bounds__(256) void rms_dx_kernel(RmsParams p) {
  __shared__ float sh[4];
  for (int64_t row = blockIdx.x; row < p.rows0 * p.rows1; row += gridDim.x) {
    const int64_t i0 = row / p.rows1, i1 = row - i0 * p.rows1;
    const T* x = static_cast<const T*>(p.x) + i0 * p.xs[0] + i1 * p.xs[1];
    const T* dy = static_cast<const T*>(p.dy) + i0 * p.dys[0] + i1 * p.dys[1];
    const T* dt = p.dtotal ? static_cast<const T*>(p.dtotal) + i0 * p.dts[0] + i1 * p.dts[1] : nullptr;
    const float rstd = p.rstd[row];
    float sgh = 0;
    for (int64_t c = threadIdx.x; c < p.C; c += 256)
      sgh = fmaf(Elem<T>::load(dy + c) * norm_param(p.w, c, p.p_bf16, 1.0f), Elem<T>::load(x + c) * rstd, sgh);
    sgh = block_sum(sgh, sh) / static_cast<float>(p.C);
    for (int64_t c = threadIdx.x; c < p.C; c += 256) {
      const float g = Elem<T>::load(dy + c) * norm_param(p.w, c, p.p_bf16, 1.0f);
      const float d = dt ? Elem<T>::load(dt + c) : 0.0f;
      Elem<T>::store(static_cast<T*>(p.dx) + row * p.C + c, fmaf(rstd, g - Elem<T>::load(x + c) * rstd * sgh, d));
    }
  }
}

// partial[chunk * C + c] over the chunk's rows; workgroup: 64 columns, 4 rows at a time
template <typename T>
__global__ __launch_bounds__(256) void rms_dw_kernel(RmsParams p, int64_t per, float* partial) {
  __shared__ float sw[256];
  const int64_t c = norm_group() * 64 + (threadIdx.x & 63);
  const int64_t r0 = blockIdx.y * per, rows = p.rows0 * p.rows1, r1 = r0 + per < rows ? r0 + per : rows;
  float dw = 0;
  if (c < p.C)
    for (int64_t row = r0 + (threadIdx.x >> 6); row < r1; row += 4) {
      const int64_t i0 = row / p.rows1, i1 = row - i0 * p.rows1;
      dw = fmaf(Elem<T>::load(static_cast<const T*>(p.dy) + i0 * p.dys[0] + i1 * p.dys[1] + c),
                Elem<T>::load(static_cast<const T*>(p.x) + i0 * p.xs[0] + i1 * p.xs[1] + c) * p.rstd[row], dw);
    }
  sw[threadIdx.x] = dw;
  __syncthreads();
  if (threadIdx.x < 64 && c < p.C) {
    const int t = threadIdx.x;
    partial[static_cast<int64_t>(blockIdx.y) * p.C + c] = (sw[t] + sw[t + 64]) + (sw[t + 128] + sw[t + 192]);
  }
}

// dweight[c]: the partial sums added up; workgroup: 8 columns by 32 partial rows at a time
__global__ __launch_bounds__(256) void rms_dw_join_kernel(const float* partial, int64_t chunks, int64_t C, void* dw, int p_bf16) {
  __shared__ float sh[4][8];
  const int64_t c = norm_group() * 8 + (threadIdx.x & 7);
  float s = 0;
  if (c < C) {
#pragma unroll 4
    for (int64_t q = threadIdx.x >> 3; q < chunks; q += 32) s += partial[q * C + c];
  }
#pragma unroll
  for (int o = 32; o >= 8; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) < 8) sh[threadIdx.x >> 6][threadIdx.x & 7] = s;
  __syncthreads();
  if (threadIdx.x >= 8 || c >= C) return;
  const float t = (sh[0][threadIdx.x] + sh[1][threadIdx.x]) + (sh[2][threadIdx.x] + sh[3][threadIdx.x]);
  if (p_bf16) static_cast<uint16_t*>(dw)[c] = f32_to_bf16_bits(t);
  else static_cast<float*>(dw)[c] = t;
}

// The values that 8-bit rows stand for, 8 at a time.
template <typename T>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(const int8_t* q, const float* scale, T* y, int64_t rows, int64_t C,
                                                              int64_t stride, int64_t pieces) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < rows * pieces; i += step) {
    const int64_t row = i / pieces, c = (i - row * pieces) * 8;
    const float s = scale[row];
    const int8_t* from = q + row * stride + c;
    T* to = y + row * C + c;
    T e[8];
    if (c + 8 <= C) {
      int8_t v[8];
      __builtin_memcpy(v, from, 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) Elem<T>::store(e + j, static_cast<float>(v[j]) * s);
      __builtin_memcpy(to, e, sizeof(e));
    } else {
      for (int j = 0; c + j < C; ++j) Elem<T>::store(to + j, static_cast<float>(from[j]) * s);
    }
  }
}

static unsigned row_groups(int64_t rows) { return static_cast<unsigned>(rows < (1 << 16) ? rows : (1 << 16)); }

template <typename T, bool INT8>
static void rms_fwd_launch(const RmsParams& p, hipStream_t s) {
  const int64_t rows = p.rows0 * p.rows1;
  const NormPlan f = norm_plan(rows, p.C, sizeof(T));
  if (f.nv == 0) {
    rms_fwd_kernel<T, INT8><<<row_groups(rows), 256, 0, s>>>(p);
    return;
  }
  const unsigned grid = static_cast<unsigned>(norm_groups(rows, f, 2048));
#define CALL(L, N, TAIL) rms_fwd_rows_kernel<T, 16 / sizeof(T), L, N, TAIL, INT8><<<grid, 256, 0, s>>>(p);
  FOVI_NORM_CASES(CALL)
#undef CALL
}

constexpr int64_t kRmsBlocks = 512;                  // workgroups of the backward: rows of partial sums

template <typename T>
static int64_t rms_bwd_launch(const RmsParams& p, float* partial, hipStream_t s) {
  const int64_t rows = p.rows0 * p.rows1;
  const NormPlan f = norm_plan(rows, p.C, sizeof(T));
  if (f.nv == 0) {
    if (p.dx) rms_dx_kernel<T><<<row_groups(rows), 256, 0, s>>>(p);
    if (!partial) return 0;
    const int64_t chunks = norm_chunks(rows, p.C), per = (rows + chunks - 1) / chunks;
    rms_dw_kernel<T><<<norm_grid(p.C, 64, chunks), 256, 0, s>>>(p, per, partial);
    return chunks;
  }
  const int64_t groups = norm_groups(rows, f, kRmsBlocks);
  const unsigned grid = static_cast<unsigned>(groups);
#define CALL(L, N, TAIL)                                   \
  rms_bwd_rows_kernel<T, 16 / sizeof(T), L, N, TAIL>       \
      <<<grid, 256, partial && L < 256 ? 4 * L * N * (16 / sizeof(T)) * 4 : 0, s>>>(p, partial);
  FOVI_NORM_CASES(CALL)
#undef CALL
  return groups;
}

static int rms_check(const fovi_rms_norm_args* a, const char* what) {
  if (!a || !a->x) { set_error("%s: null pointer", what); return 1; }
  if ((a->dtype != FOVI_F32 && a->dtype != FOVI_BF16) || (a->p_dtype != FOVI_F32 && a->p_dtype != FOVI_BF16)) {
    set_error("%s: dtypes must be F32 or BF16", what);
    return 1;
  }
  if (a->rows0 < 0 || a->rows1 < 0 || a->channels < 1) { set_error("%s: bad sizes", what); return 1; }
  if (a->channels > (1 << 30)) { set_error("%s: more than 2^30 channels", what); return 1; }
  if (!(a->eps >= 0)) { set_error("%s: eps must not be negative", what); return 1; }
  return 0;
}

static RmsParams rms_params(const fovi_rms_norm_args* a) {
  RmsParams p;
  p.x = a->x; p.r = a->residual; p.w = a->weight; p.total = a->total; p.y = a->y; p.q = a->q; p.scale = a->scale; p.rstd = a->rstd;
  p.dy = a->dy; p.dtotal = a->dtotal; p.dx = a->dx;
  p.rows0 = a->rows0; p.rows1 = a->rows1; p.C = a->channels;
  for (int i = 0; i < 2; ++i) {
    p.xs[i] = a->x_stride[i]; p.rs[i] = a->residual_stride[i]; p.dys[i] = a->dy_stride[i]; p.dts[i] = a->dtotal_stride[i];
  }
  p.eps = a->eps;
  p.p_bf16 = a->p_dtype == FOVI_BF16;
  p.norm = 1;
  return p;
}

}  // namespace fovi

using namespace fovi;

extern "C" int fovi_rms_norm_fwd(const fovi_rms_norm_args* a, void* stream) {
  clear_error();
  if (rms_check(a, "fovi_rms_norm_fwd")) return 1;
  if (!a->y == !a->q || !a->q != !a->scale || !a->residual != !a->total) {
    set_error("fovi_rms_norm_fwd: either y, or q with scale; total with residual");
    return 1;
  }
  if (a->rows0 * a->rows1 == 0) return 0;
  const RmsParams p = rms_params(a);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == FOVI_BF16) {
    if (p.q) rms_fwd_launch<uint16_t, true>(p, s);
    else rms_fwd_launch<uint16_t, false>(p, s);
  } else {
    if (p.q) rms_fwd_launch<float, true>(p, s);
    else rms_fwd_launch<float, false>(p, s);
  }
  return check_launch("fovi_rms_norm_fwd");
}

extern "C" int64_t fovi_rms_norm_workspace_bytes(int64_t rows, int64_t channels) {
  if (rows < 1 || channels < 1) return 0;
  const int64_t chunks = norm_chunks(rows, channels), blocks = rows < kRmsBlocks ? rows : kRmsBlocks;
  return (chunks > blocks ? chunks : blocks) * channels * 4;
}

extern "C" int fovi_rms_norm_bwd(const fovi_rms_norm_args* a, void* stream) {
  clear_error();
  if (rms_check(a, "fovi_rms_norm_bwd")) return 1;
  const int64_t rows = a->rows0 * a->rows1;
  if (!a->dy || !a->rstd) { set_error("fovi_rms_norm_bwd: null pointer"); return 1; }
  const int64_t need = fovi_rms_norm_workspace_bytes(rows, a->channels);
  if (a->dweight && need && (!a->workspace || a->workspace_bytes < need)) {
    set_error("fovi_rms_norm_bwd: workspace of %lld bytes needed", static_cast<long long>(need));
    return 1;
  }
  const RmsParams p = rms_params(a);
  hipStream_t s = static_cast<hipStream_t>(stream);
  int64_t chunks = 0;
  float* partial = a->dweight ? static_cast<float*>(a->workspace) : nullptr;
  if (rows) {
    chunks = a->dtype == FOVI_BF16 ? rms_bwd_launch<uint16_t>(p, partial, s) : rms_bwd_launch<float>(p, partial, s);
    if (check_launch("fovi_rms_norm_bwd")) return 1;
  }
  if (!a->dweight) return 0;
  rms_dw_join_kernel<<<norm_grid(p.C, 8, 1), 256, 0, s>>>(partial, chunks, p.C, a->dweight, p.p_bf16);
  return check_launch("fovi_rms_norm_bwd");
}

extern "C" int fovi_quantize_rows(const void* x, int32_t dtype, int64_t rows0, int64_t rows1, int64_t channels, const int64_t* stride,
                                  int8_t* q, float* scale, void* stream) {
  clear_error();
  if (!x || !stride || !q || !scale) { set_error("fovi_quantize_rows: null pointer"); return 1; }
  if (dtype != FOVI_F32 && dtype != FOVI_BF16) { set_error("fovi_quantize_rows: dtype must be F32 or BF16"); return 1; }
  if (rows0 < 0 || rows1 < 0 || channels < 1 || channels > (1 << 30)) { set_error("fovi_quantize_rows: bad sizes"); return 1; }
  if (rows0 * rows1 == 0) return 0;
  RmsParams p = {};
  p.x = x; p.q = q; p.scale = scale;
  p.rows0 = rows0; p.rows1 = rows1; p.C = channels;
  p.xs[0] = stride[0]; p.xs[1] = stride[1];
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == FOVI_BF16) rms_fwd_launch<uint16_t, true>(p, s);
  else rms_fwd_launch<float, true>(p, s);
  return check_launch("fovi_quantize_rows");
}

extern "C" int fovi_dequantize_rows(const int8_t* q, const float* scale, int64_t rows, int64_t channels, int64_t stride, void* y,
                                    int32_t dtype, void* stream) {
  clear_error();
  if (!q || !scale || !y) { set_error("fovi_dequantize_rows: null pointer"); return 1; }
  if (dtype != FOVI_F32 && dtype != FOVI_BF16) { set_error("fovi_dequantize_rows: dtype must be F32 or BF16"); return 1; }
  if (rows < 0 || channels < 1) { set_error("fovi_dequantize_rows: bad sizes"); return 1; }
  if (rows == 0) return 0;
  const int64_t pieces = (channels + 7) / 8, groups = (rows * pieces + 255) / 256;
  const unsigned grid = static_cast<unsigned>(groups < (1 << 14) ? groups : (1 << 14));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == FOVI_BF16) dequantize_rows_kernel<uint16_t><<<grid, 256, 0, s>>>(q, scale, static_cast<uint16_t*>(y), rows, channels, stride, pieces);
  else dequantize_rows_kernel<float><<<grid, 256, 0, s>>>(q, scale, static_cast<float*>(y), rows, channels, stride, pieces);
  return check_launch("fovi_dequantize_rows");
}
