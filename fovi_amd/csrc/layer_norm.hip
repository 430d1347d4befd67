// Layer norm over the channels of token rows: forward, and the gradients of rows, weight and bias.
//
//   h = (x - mean) * rstd, y = h * w + b
//   dx = rstd * (g - mean(g) - h * mean(g * h)), g = dy * w; dw = sum dy * h; db = sum dy
//
// Bound by memory. A row is read once into the registers of a group of lanes (16, 64 or 256), which
// takes the mean and then the centred squares from there (no cancellation between large sums), and
// writes from there too. Groups walk the rows with the parameters in registers. The backward keeps
// the sums of dy * h and dy of its channels over all its rows in registers as well, so that x and dy
// are read once for all three gradients; each workgroup leaves one row of partial sums, and a second
// launch adds those in a fixed order (no atomics: results do not change from run to run).
// 131072 bf16 rows of 384: forward 34 us (201 MB, 6.0 TB/s), backward 52 (302 MB, 5.8 TB/s) and 4 for the join.
// Rows too wide for registers go through kernels of a workgroup per row that read them again.
#include "norm.h"

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

template <typename T, int VEC, int LANES, int NV, bool TAIL>
__global__ __launch_bounds__(256) void norm_fwd_rows_kernel(NormParams p) {
  __shared__ float sh[4];
  const int lane = threadIdx.x % LANES;
  float w[NV][VEC], b[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    norm_params_at<VEC>(p.w, static_cast<int64_t>(lane + k * LANES) * VEC, p.C, p.p_bf16, 1.0f, w[k]);
    norm_params_at<VEC>(p.b, static_cast<int64_t>(lane + k * LANES) * VEC, p.C, p.p_bf16, 0.0f, b[k]);
  }
  const float n = 1.0f / static_cast<float>(p.C);
  const int64_t rows = p.rows0 * p.rows1, step = static_cast<int64_t>(gridDim.x) * (256 / LANES);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES; row < rows; row += step) {
    const int64_t i0 = p.rows0 == 1 ? 0 : row / p.rows1, i1 = row - i0 * p.rows1;
    const T* xr = static_cast<const T*>(p.x) + i0 * p.xs[0] + i1 * p.xs[1];
    T* yr = static_cast<T*>(p.y) + i0 * p.ys[0] + i1 * p.ys[1];
    float x[NV][VEC], s = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) norm_load<T, VEC>(xr, static_cast<int64_t>(lane + k * LANES) * VEC, p.C, x[k], TAIL && k == NV - 1);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) s += x[k][i];
    const float mean = group_sum<LANES>(s, sh) * n;
    s = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = static_cast<int64_t>(lane + k * LANES) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        x[k][i] = c + (TAIL ? i : 0) < p.C ? x[k][i] - mean : 0.0f;
        s = fmaf(x[k][i], x[k][i], s);
      }
    }
    const float rstd = 1.0f / sqrtf(group_sum<LANES>(s, sh) * n + p.eps);
    if (lane == 0 && p.mean) { p.mean[row] = mean; p.rstd[row] = rstd; }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float y[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) y[i] = fmaf(x[k][i] * rstd, w[k][i], b[k][i]);
      norm_store<T, VEC>(yr, static_cast<int64_t>(lane + k * LANES) * VEC, p.C, y, TAIL && k == NV - 1);
    }
  }
}

// dx of the rows and, with `partial`, the workgroup's sums of dy * h and dy: partial[(block * 2 + {0, 1}) * C + c].
template <typename T, int VEC, int LANES, int NV, bool TAIL>
__global__ __launch_bounds__(256) void norm_bwd_rows_kernel(NormParams p, float* partial) {
  __shared__ float sh[4];
  const int lane = threadIdx.x % LANES;
  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    norm_params_at<VEC>(p.w, static_cast<int64_t>(lane + k * LANES) * VEC, p.C, p.p_bf16, 1.0f, w[k]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[k][i] = db[k][i] = 0;
  }
  const float n = 1.0f / static_cast<float>(p.C);
  const int64_t rows = p.rows0 * p.rows1, step = static_cast<int64_t>(gridDim.x) * (256 / LANES);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES; row < rows; row += step) {
    const int64_t i0 = p.rows0 == 1 ? 0 : row / p.rows1, i1 = row - i0 * p.rows1;
    const T* xr = static_cast<const T*>(p.x) + i0 * p.xs[0] + i1 * p.xs[1];
    const T* gr = static_cast<const T*>(p.dy) + i0 * p.dys[0] + i1 * p.dys[1];
    const float mean = p.mean[row], rstd = p.rstd[row];
    float h[NV][VEC], g[NV][VEC], sg = 0, sgh = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = static_cast<int64_t>(lane + k * LANES) * VEC;
      norm_load<T, VEC>(xr, c, p.C, h[k], TAIL && k == NV - 1);
      norm_load<T, VEC>(gr, c, p.C, g[k], TAIL && k == NV - 1);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = static_cast<int64_t>(lane + k * LANES) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        h[k][i] = c + (TAIL ? i : 0) < p.C ? (h[k][i] - mean) * rstd : 0.0f;
        dw[k][i] = fmaf(g[k][i], h[k][i], dw[k][i]);
        db[k][i] += g[k][i];
        g[k][i] *= w[k][i];
        sg += g[k][i];
        sgh = fmaf(g[k][i], h[k][i], sgh);
      }
    }
    if (!p.dx) continue;
    sg = group_sum<LANES>(sg, sh) * n;
    sgh = group_sum<LANES>(sgh, sh) * n;
    T* dxr = static_cast<T*>(p.dx) + i0 * p.dxs[0] + i1 * p.dxs[1];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float dx[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) dx[i] = rstd * (g[k][i] - sg - h[k][i] * sgh);
      norm_store<T, VEC>(dxr, static_cast<int64_t>(lane + k * LANES) * VEC, p.C, dx, TAIL && k == NV - 1);
    }
  }
  if (!partial) return;
  float* out = partial + static_cast<int64_t>(blockIdx.x) * 2 * p.C;
  if (LANES == 256) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t c = static_cast<int64_t>(lane + k * LANES) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (c + i < p.C) { out[c + i] = dw[k][i]; out[p.C + c + i] = db[k][i]; }
    }
    return;
  }
  // the groups of a wave by shuffles, the waves through LDS
  constexpr int WIDTH = LANES * NV * VEC;
  extern __shared__ float sums[];                    // [4][2][WIDTH]
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float a = dw[k][i], c = db[k][i];
#pragma unroll
      for (int o = 32; o >= LANES; o >>= 1) {
        a += __shfl_xor(a, o);
        c += __shfl_xor(c, o);
      }
      const int at = (lane + k * LANES) * VEC + i;
      if ((threadIdx.x & 63) < LANES) {
        sums[(wave * 2) * WIDTH + at] = a;
        sums[(wave * 2 + 1) * WIDTH + at] = c;
      }
    }
  __syncthreads();
  for (int x = threadIdx.x; x < 2 * WIDTH; x += 256) {
    const int which = x / WIDTH, at = x - which * WIDTH;
    if (at < p.C)
      out[which * p.C + at] = (sums[x] + sums[2 * WIDTH + x]) + (sums[4 * WIDTH + x] + sums[6 * WIDTH + x]);
  }
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
  const int64_t c = norm_group() * 64 + (threadIdx.x & 63);
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

// dweight[c], dbias[c]: the partial sums added up; workgroup: 8 columns by 32 partial rows at a time
__global__ __launch_bounds__(256) void norm_dw_join_kernel(const float* partial, int64_t chunks, int64_t C, void* dw,
                                                           void* db, int p_bf16) {
  __shared__ float sh[4][8];
  const int64_t c = norm_group() * 8 + (threadIdx.x & 7);
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  float s = 0;
  if (c < C) {
#pragma unroll 4
    for (int64_t q = threadIdx.x >> 3; q < chunks; q += 32) s += partial[(q * 2 + blockIdx.y) * C + c];
  }
#pragma unroll
  for (int o = 32; o >= 8; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) < 8) sh[threadIdx.x >> 6][threadIdx.x & 7] = s;
  __syncthreads();
  if (threadIdx.x >= 8 || c >= C) return;
  const float t = (sh[0][threadIdx.x] + sh[1][threadIdx.x]) + (sh[2][threadIdx.x] + sh[3][threadIdx.x]);
  if (p_bf16) static_cast<uint16_t*>(out)[c] = f32_to_bf16_bits(t);
  else static_cast<float*>(out)[c] = t;
}

template <typename T>
static void norm_fwd_launch(const NormParams& p, hipStream_t s) {
  const int64_t rows = p.rows0 * p.rows1;
  const NormPlan f = norm_plan(rows, p.C, sizeof(T));
  if (f.nv == 0) {
    norm_fwd_kernel<T><<<static_cast<unsigned>(rows < (1 << 16) ? rows : (1 << 16)), 256, 0, s>>>(p);
    return;
  }
  const unsigned grid = static_cast<unsigned>(norm_groups(rows, f, 2048));
#define CALL(L, N, TAIL) norm_fwd_rows_kernel<T, 16 / sizeof(T), L, N, TAIL><<<grid, 256, 0, s>>>(p);
  FOVI_NORM_CASES(CALL)
#undef CALL
}

constexpr int64_t kNormBlocks = 512;                 // workgroups of the backward: rows of partial sums

template <typename T>
static int64_t norm_bwd_launch(const NormParams& p, float* partial, hipStream_t s) {
  const int64_t rows = p.rows0 * p.rows1;
  const NormPlan f = norm_plan(rows, p.C, sizeof(T));
  if (f.nv == 0) {
    if (p.dx) norm_dx_kernel<T><<<static_cast<unsigned>(rows < (1 << 16) ? rows : (1 << 16)), 256, 0, s>>>(p);
    if (!partial) return 0;
    const int64_t chunks = norm_chunks(rows, p.C), per = (rows + chunks - 1) / chunks;
    norm_dw_kernel<T><<<norm_grid(p.C, 64, chunks), 256, 0, s>>>(p, per, partial);
    return chunks;
  }
  const int64_t groups = norm_groups(rows, f, kNormBlocks);
  const unsigned grid = static_cast<unsigned>(groups);
#define CALL(L, N, TAIL)                                       \
  norm_bwd_rows_kernel<T, 16 / sizeof(T), L, N, TAIL>          \
      <<<grid, 256, partial && L < 256 ? 4 * 2 * L * N * (16 / sizeof(T)) * 4 : 0, s>>>(p, partial);
  FOVI_NORM_CASES(CALL)
#undef CALL
  return groups;
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
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == FOVI_BF16) norm_fwd_launch<uint16_t>(p, s);
  else norm_fwd_launch<float>(p, s);
  return check_launch("fovi_layer_norm_fwd");
}

extern "C" int64_t fovi_layer_norm_workspace_bytes(int64_t rows, int64_t channels, int32_t dtype) {
  (void)dtype;
  if (rows < 1 || channels < 1) return 0;
  const int64_t chunks = norm_chunks(rows, channels), blocks = rows < kNormBlocks ? rows : kNormBlocks;
  return (chunks > blocks ? chunks : blocks) * 2 * channels * 4;
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
  int64_t chunks = 0;
  float* partial = params ? static_cast<float*>(a->workspace) : nullptr;
  if (rows) {
    chunks = a->dtype == FOVI_BF16 ? norm_bwd_launch<uint16_t>(p, partial, s) : norm_bwd_launch<float>(p, partial, s);
    if (check_launch("fovi_layer_norm_bwd")) return 1;
  }
  if (!params) return 0;
  norm_dw_join_kernel<<<norm_grid(p.C, 8, 2), 256, 0, s>>>(partial, chunks, p.C, a->dweight, a->dbias, p.p_bf16);
  return check_launch("fovi_layer_norm_bwd");
}
