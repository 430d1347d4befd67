// Layer norm over the channels of token rows: forward, and the gradients of rows, weight and bias.
//
//   h = (x - mean) * rstd, y = h * w + b
//   dx = rstd * (g - mean(g) - h * mean(g * h)), g = dy * w; dw = sum dy * h; db = sum dy
//
// One workgroup per row; the row is read once for the mean, once for the centred squares (no
// cancellation between large sums) and once to write. The weight gradients are summed by columns:
// a workgroup takes 64 columns of a chunk of rows into fp32 partial sums, which a second launch
// adds in a fixed order, so results do not change from run to run.
#include "common.h"

namespace fovi {

struct NormParams {
  const void* x; const void* w; const void* b; void* y;
  const void* dy; void* dx;
  float* mean; float* rstd;
  int64_t rows0, rows1, C;
  int64_t xs[2], ys[2], dys[2], dxs[2];
  float eps;
  int p_bf16;
};

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

template <typename T>
__global__ __launch_bounds__(256) void norm_fwd_kernel(NormParams p) {
  __shared__ float sh[4];
  for (int64_t row = blockIdx.x; row < p.rows0 * p.rows1; row += gridDim.x) {
    const int64_t i0 = row / p.rows1, i1 = row - i0 * p.rows1;
    const T* x = static_cast<const T*>(p.x) + i0 * p.xs[0] + i1 * p.xs[1];
    T* y = static_cast<T*>(p.y) + i0 * p.ys[0] + i1 * p.ys[1];
    float s = 0;
    for (int64_t c = threadIdx.x; c < p.C; c += 256) s += Elem<T>::load(x + c);
    const float mean = block_sum(s, sh) / static_cast<float>(p.C);
    s = 0;
    for (int64_t c = threadIdx.x; c < p.C; c += 256) {
      const float d = Elem<T>::load(x + c) - mean;
      s = fmaf(d, d, s);
    }
    const float rstd = 1.0f / sqrtf(block_sum(s, sh) / static_cast<float>(p.C) + p.eps);
    if (threadIdx.x == 0 && p.mean) { p.mean[row] = mean; p.rstd[row] = rstd; }
    for (int64_t c = threadIdx.x; c < p.C; c += 256) {
      const float h = (Elem<T>::load(x + c) - mean) * rstd;
      Elem<T>::store(y + c, fmaf(h, norm_param(p.w, c, p.p_bf16, 1.0f), norm_param(p.b, c, p.p_bf16, 0.0f)));
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void norm_dx_kernel(NormParams p) {
  __shared__ float sh[4];
  for (int64_t row = blockIdx.x; row < p.rows0 * p.rows1; row += gridDim.x) {
    const int64_t i0 = row / p.rows1, i1 = row - i0 * p.rows1;
    const T* x = static_cast<const T*>(p.x) + i0 * p.xs[0] + i1 * p.xs[1];
    const T* dy = static_cast<const T*>(p.dy) + i0 * p.dys[0] + i1 * p.dys[1];
    T* dx = static_cast<T*>(p.dx) + i0 * p.dxs[0] + i1 * p.dxs[1];
    const float mean = p.mean[row], rstd = p.rstd[row];
    float sg = 0, sgh = 0;
    for (int64_t c = threadIdx.x; c < p.C; c += 256) {
      const float g = Elem<T>::load(dy + c) * norm_param(p.w, c, p.p_bf16, 1.0f);
      sg += g;
      sgh = fmaf(g, (Elem<T>::load(x + c) - mean) * rstd, sgh);
    }
    sg = block_sum(sg, sh) / static_cast<float>(p.C);
    sgh = block_sum(sgh, sh) / static_cast<float>(p.C);
    for (int64_t c = threadIdx.x; c < p.C; c += 256) {
      const float g = Elem<T>::load(dy + c) * norm_param(p.w, c, p.p_bf16, 1.0f);
      const float h = (Elem<T>::load(x + c) - mean) * rstd;
      Elem<T>::store(dx + c, rstd * (g - sg - h * sgh));
    }
  }
}

// partial[(chunk * 2 + {0: dw, 1: db}) * C + c] over the chunk's rows; workgroup: 64 columns, 4 rows at a time
template <typename T>
__global__ __launch_bounds__(256) void norm_dw_kernel(NormParams p, int64_t per, float* partial) {
  __shared__ float sw[256], sb[256];
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + (threadIdx.x & 63);
  const int64_t r0 = blockIdx.y * per, rows = p.rows0 * p.rows1, r1 = r0 + per < rows ? r0 + per : rows;
  float dw = 0, db = 0;
  if (c < p.C)
    for (int64_t row = r0 + (threadIdx.x >> 6); row < r1; row += 4) {
      const int64_t i0 = row / p.rows1, i1 = row - i0 * p.rows1;
      const float d = Elem<T>::load(static_cast<const T*>(p.dy) + i0 * p.dys[0] + i1 * p.dys[1] + c);
      const float h = (Elem<T>::load(static_cast<const T*>(p.x) + i0 * p.xs[0] + i1 * p.xs[1] + c) - p.mean[row]) * p.rstd[row];
      dw = fmaf(d, h, dw);
      db += d;
    }
  sw[threadIdx.x] = dw;
  sb[threadIdx.x] = db;
  __syncthreads();
  if (threadIdx.x < 64 && c < p.C) {
    const int t = threadIdx.x;
    float* out = partial + static_cast<int64_t>(blockIdx.y) * 2 * p.C + c;
    out[0] = (sw[t] + sw[t + 64]) + (sw[t + 128] + sw[t + 192]);
    out[p.C] = (sb[t] + sb[t + 64]) + (sb[t + 128] + sb[t + 192]);
  }
}

// dweight[c], dbias[c]: the partial sums added up; workgroup: 16 columns by 16 chunks at a time
__global__ __launch_bounds__(256) void norm_dw_join_kernel(const float* partial, int64_t chunks, int64_t C, void* dw,
                                                           void* db, int p_bf16) {
  __shared__ float sh[256];
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x & 15);
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  float s = 0;
  if (c < C)
    for (int64_t q = threadIdx.x >> 4; q < chunks; q += 16) s += partial[(q * 2 + blockIdx.y) * C + c];
  sh[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x >= 16 || c >= C) return;
  float t = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) t += sh[threadIdx.x + 16 * i];
  if (p_bf16) static_cast<uint16_t*>(out)[c] = f32_to_bf16_bits(t);
  else static_cast<float*>(out)[c] = t;
}

static int64_t norm_chunks(int64_t rows, int64_t C) {
  const int64_t cols = (C + 63) / 64;
  int64_t chunks = (1024 + cols - 1) / cols;        // about four workgroups a compute unit
  if (chunks > (rows + 15) / 16) chunks = (rows + 15) / 16;
  return chunks < 1 ? 1 : chunks;
}

static int norm_check(const fovi_layer_norm_args* a, const char* what) {
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

static NormParams norm_params(const fovi_layer_norm_args* a) {
  NormParams p;
  p.x = a->x; p.w = a->weight; p.b = a->bias; p.y = a->y; p.dy = a->dy; p.dx = a->dx;
  p.mean = a->mean; p.rstd = a->rstd;
  p.rows0 = a->rows0; p.rows1 = a->rows1; p.C = a->channels;
  for (int i = 0; i < 2; ++i) {
    p.xs[i] = a->x_stride[i]; p.ys[i] = a->y_stride[i]; p.dys[i] = a->dy_stride[i]; p.dxs[i] = a->dx_stride[i];
  }
  p.eps = a->eps;
  p.p_bf16 = a->p_dtype == FOVI_BF16;
  return p;
}

}  // namespace fovi

using namespace fovi;

extern "C" int fovi_layer_norm_fwd(const fovi_layer_norm_args* a, void* stream) {
  clear_error();
  if (norm_check(a, "fovi_layer_norm_fwd")) return 1;
  if (!a->y || !a->mean != !a->rstd) { set_error("fovi_layer_norm_fwd: null pointer"); return 1; }
  const int64_t rows = a->rows0 * a->rows1;
  if (rows == 0) return 0;
  const NormParams p = norm_params(a);
  const unsigned grid = static_cast<unsigned>(rows < (1 << 16) ? rows : (1 << 16));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == FOVI_BF16) norm_fwd_kernel<uint16_t><<<grid, 256, 0, s>>>(p);
  else norm_fwd_kernel<float><<<grid, 256, 0, s>>>(p);
  return check_launch("fovi_layer_norm_fwd");
}

extern "C" int64_t fovi_layer_norm_workspace_bytes(int64_t rows, int64_t channels, int32_t dtype) {
  (void)dtype;
  if (rows < 1 || channels < 1) return 0;
  return norm_chunks(rows, channels) * 2 * channels * 4;
}

extern "C" int fovi_layer_norm_bwd(const fovi_layer_norm_args* a, void* stream) {
  clear_error();
  if (norm_check(a, "fovi_layer_norm_bwd")) return 1;
  const int64_t rows = a->rows0 * a->rows1;
  if (!a->dy || !a->mean || !a->rstd) { set_error("fovi_layer_norm_bwd: null pointer"); return 1; }
  const bool params = a->dweight || a->dbias;
  const int64_t need = fovi_layer_norm_workspace_bytes(rows, a->channels, a->dtype);
  if (params && need && (!a->workspace || a->workspace_bytes < need)) {
    set_error("fovi_layer_norm_bwd: workspace of %lld bytes needed", static_cast<long long>(need));
    return 1;
  }
  const NormParams p = norm_params(a);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dx && rows) {
    const unsigned grid = static_cast<unsigned>(rows < (1 << 16) ? rows : (1 << 16));
    if (a->dtype == FOVI_BF16) norm_dx_kernel<uint16_t><<<grid, 256, 0, s>>>(p);
    else norm_dx_kernel<float><<<grid, 256, 0, s>>>(p);
    if (check_launch("fovi_layer_norm_bwd")) return 1;
  }
  if (!params) return 0;
  const int64_t chunks = rows ? norm_chunks(rows, p.C) : 0;
  float* partial = static_cast<float*>(a->workspace);
  if (chunks) {
    const dim3 grid(static_cast<unsigned>((p.C + 63) / 64), static_cast<unsigned>(chunks));
    const int64_t per = (rows + chunks - 1) / chunks;
    if (a->dtype == FOVI_BF16) norm_dw_kernel<uint16_t><<<grid, 256, 0, s>>>(p, per, partial);
    else norm_dw_kernel<float><<<grid, 256, 0, s>>>(p, per, partial);
    if (check_launch("fovi_layer_norm_bwd")) return 1;
  }
  norm_dw_join_kernel<<<dim3(static_cast<unsigned>((p.C + 15) / 16), 2), 256, 0, s>>>(partial, chunks, p.C, a->dweight,
                                                                                    a->dbias, p.p_bf16);
  return check_launch("fovi_layer_norm_bwd");
}
