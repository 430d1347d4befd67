// The gated feed-forward block of token rows and its gradients.
//
//   gate = x Wg^T, up = x Wu^T, h = act(gate) * up, y = h Wd^T (+ residual)
//   dh = dy Wd, dgate = dh * up * act'(gate), dup = dh * act(gate)
//   dx = dgate Wg + dup Wu, dWg = dgate^T x, dWu = dup^T x, dWd = dy^T h
//
// Both first projections run over one tile of x, and h is all that leaves them. The backward forms gate and up again
// beside dh, in the registers of one kernel, whose epilogue writes dgate, dup and h (bf16; fp32 calls keep gate and up
// from the forward). The weights' gradients reduce over the tokens: the tokens are split over workgroups, whose
// partial sums a second launch adds in a fixed order.
#include "matmul.h"

namespace fovi {

struct MatSegments {
  MatOperand x[2], w[2];
  int64_t k[2];
  int n;
};

template <typename T> struct MlpLinear {               // out = sums (+ residual)
  T* out; int64_t stride;
  const T* residual; int64_t residual_stride;
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, int count, const float (&v)[1][4]) const {
    float y[4] = {v[0][0], v[0][1], v[0][2], v[0][3]};
    if (residual) {
      float r[4];
      load_four(residual + m * residual_stride + n, count, r);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] += r[i];
    }
    store_four(out + m * stride + n, count, y);
  }
};

template <typename T> struct MlpTwoRows {              // rows below `rows` to one output, the others to the next
  T* out[2]; int64_t rows, stride;
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, int count, const float (&v)[1][4]) const {
    store_four(m < rows ? out[0] + m * stride + n : out[1] + (m - rows) * stride + n, count, v[0]);
  }
};

struct MlpPartial {                                    // the sums of a share of the reduction
  float* part; int64_t M, N;
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, int count, const float (&v)[1][4]) const {
    store_four(part + (blockIdx.y * M + m) * N + n, count, v[0]);
  }
};

template <typename T> struct MlpGated {                // h, and gate and up where a backward will read them
  T* h; int64_t stride; int act;
  T* gate; T* up; int64_t saved_stride;
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, int count, const float (&v)[2][4]) const {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = mat_act<sizeof(T) == 4>(v[0][i], act) * v[1][i];
    store_four(h + m * stride + n, count, y);
    if (gate) {
      store_four(gate + m * saved_stride + n, count, v[0]);
      store_four(up + m * saved_stride + n, count, v[1]);
    }
  }
};

template <typename T> struct MlpGatedGrad {            // dgate, dup and h from gate, up and dh
  T* dgate; T* dup; T* h; int64_t stride, h_stride; int act;
  const T* gate; const T* up; int64_t saved_stride;
  __device__ __forceinline__ void write(int64_t m, int64_t n, int count, const float (&g)[4], const float (&u)[4],
                                        const float (&dh)[4]) const {
    float a[4], b[4], c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float value, slope;
      mat_act_grad<sizeof(T) == 4>(g[i], act, value, slope);
      a[i] = dh[i] * u[i] * slope;
      b[i] = dh[i] * value;
      c[i] = value * u[i];
    }
    store_four(dgate + m * stride + n, count, a);
    store_four(dup + m * stride + n, count, b);
    store_four(h + m * h_stride + n, count, c);
  }
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, int count, const float (&v)[3][4]) const {
    write(m, n, count, v[0], v[1], v[2]);
  }
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, int count, const float (&v)[1][4]) const {
    float g[4], u[4];
    load_four(gate + m * saved_stride + n, count, g);
    load_four(up + m * saved_stride + n, count, u);
    write(m, n, count, g, u, v[0]);
  }
};

template <typename T, int BM, int BN, bool CX, bool CW, typename Epilogue>
__global__ __launch_bounds__(256) void mlp_linear_kernel(MatSegments s, int64_t M, int64_t N, int64_t share, Epilogue epilogue) {
  typedef MatCore<T, BM, BN, 1, CX, CW> Core;
  __shared__ __attribute__((aligned(16))) char lds[Core::LDS];
  int64_t tm, tn;
  if (!mat_tile((M + BM - 1) / BM, (N + BN - 1) / BN, tm, tn)) return;
  typename Core::Acc acc[1][Core::MB][Core::NN];
  mat_clear(acc);
  for (int i = 0; i < s.n; ++i) {
    const int64_t from = blockIdx.y * share, to = from + share < s.k[i] ? from + share : s.k[i];
    if (from < to) Core::run(s.x[i], &s.w[i], tm * BM, tn * BN, from, to, lds, acc);
  }
  mat_finish<BM, BN, float>(acc, tm * BM, tn * BN, M, N, epilogue);
}

// out = the shares' sums added up, through the epilogue.
template <typename Epilogue>
__global__ __launch_bounds__(256) void mlp_join_kernel(const float* part, int64_t shares, int64_t M, int64_t N, Epilogue epilogue) {
  const int64_t per = (N + 3) / 4, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= M * per) return;
  const int64_t m = i / per, n = (i - m * per) * 4;
  const int count = static_cast<int>(N - n < 4 ? N - n : 4);
  float v[1][4] = {{0, 0, 0, 0}};
  for (int64_t z = 0; z < shares; ++z) {
    float t[4];
    load_four(part + (z * M + m) * N + n, count, t);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[0][e] += t[e];
  }
  epilogue(m, n, count, v);
}

template <typename T, int BM, int BN>
__global__ __launch_bounds__(256) void mlp_gated_kernel(MatOperand x, MatOperand wg, MatOperand wu, int64_t K, int64_t M, int64_t N,
                                                        MlpGated<T> epilogue) {
  typedef MatCore<T, BM, BN, 2, false, false> Core;
  __shared__ __attribute__((aligned(16))) char lds[Core::LDS];
  int64_t tm, tn;
  if (!mat_tile((M + BM - 1) / BM, (N + BN - 1) / BN, tm, tn)) return;
  typename Core::Acc acc[2][Core::MB][Core::NN];
  mat_clear(acc);
  const MatOperand w[2] = {wg, wu};
  Core::run(x, w, tm * BM, tn * BN, 0, K, lds, acc);
  mat_finish<BM, BN, float>(acc, tm * BM, tn * BN, M, N, epilogue);
}

// gate, up and dh of a tile, one after the other, and what the epilogue makes of them.
template <typename T, int BM, int BN>
__global__ __launch_bounds__(256) void mlp_gated_grad_kernel(MatOperand x, MatOperand wg, MatOperand wu, MatOperand dy, MatOperand wd,
                                                             int64_t K, int64_t M, int64_t N, MlpGatedGrad<T> epilogue) {
  typedef MatCore<T, BM, BN, 2, false, false> Both;
  typedef MatCore<T, BM, BN, 1, false, true> Down;
  __shared__ __attribute__((aligned(16))) char lds[Both::LDS];
  int64_t tm, tn;
  if (!mat_tile((M + BM - 1) / BM, (N + BN - 1) / BN, tm, tn)) return;
  typename Both::Acc acc[3][Both::MB][Both::NN];
  mat_clear(acc);
  const MatOperand w[2] = {wg, wu};
  Both::run(x, w, tm * BM, tn * BN, 0, K, lds, acc);
  Down::run(dy, &wd, tm * BM, tn * BN, 0, K, lds, acc, 2);
  mat_finish<BM, BN, float>(acc, tm * BM, tn * BN, M, N, epilogue);
}

static int64_t tiles_of(int64_t n, int64_t b) { return (n + b - 1) / b; }

template <typename T, bool CX, bool CW, typename Epilogue>
static void mlp_linear(const MatSegments& s, int64_t M, int64_t N, const Epilogue& epilogue, hipStream_t stream) {
  const int64_t tiles = tiles_of(M, 128) * tiles_of(N, 128);
  mlp_linear_kernel<T, 128, 128, CX, CW, Epilogue><<<mat_grid(tiles), 256, 0, stream>>>(s, M, N, s.k[0] > s.k[1] ? s.k[0] : s.k[1], epilogue);
}

// Shares of a reduction over the tokens: workgroups for the whole card twice over, at least 512 tokens each.
static int64_t token_shares(int64_t tokens, int64_t M, int64_t N) {
  const int64_t tiles = tiles_of(M, 128) * tiles_of(N, 128);
  int64_t shares = (512 + tiles - 1) / tiles;
  const int64_t most = (tokens + 511) / 512;
  if (shares > most) shares = most;
  return shares < 1 ? 1 : shares;
}

// x and w by columns, reduced over the tokens.
template <typename T, typename Epilogue>
static void token_product(const MatOperand& x, const MatOperand& w, int64_t tokens, int64_t M, int64_t N, float* part,
                          const Epilogue& epilogue, hipStream_t stream) {
  const int64_t shares = token_shares(tokens, M, N);
  MatSegments s = {{x}, {w}, {tokens, 0}, 1};
  if (shares == 1) {
    mlp_linear<T, true, true>(s, M, N, epilogue, stream);
    return;
  }
  const int64_t bk = Mat<T>::BK, share = ((tokens + shares - 1) / shares + bk - 1) / bk * bk;
  const int64_t used = (tokens + share - 1) / share;
  const dim3 grid(mat_grid(tiles_of(M, 128) * tiles_of(N, 128)), static_cast<unsigned>(used));
  mlp_linear_kernel<T, 128, 128, true, true, MlpPartial><<<grid, 256, 0, stream>>>(s, M, N, share, MlpPartial{part, M, N});
  mlp_join_kernel<Epilogue><<<static_cast<unsigned>((M * ((N + 3) / 4) + 255) / 256), 256, 0, stream>>>(part, used, M, N, epilogue);
}

static int mlp_check(const fovi_gated_mlp_args* a, const char* what) {
  if (!a || !a->x || !a->w_gate || !a->w_up || !a->w_down) { set_error("%s: null pointer", what); return 1; }
  if (a->dtype != FOVI_F32 && a->dtype != FOVI_BF16) { set_error("%s: dtype must be F32 or BF16", what); return 1; }
  if (a->activation != FOVI_GATE_SILU && a->activation != FOVI_GATE_GELU) { set_error("%s: unknown activation", what); return 1; }
  if (a->rows < 0 || a->dim < 1 || a->hidden < 1 || a->dim > (1 << 24) || a->hidden > (1 << 24) || a->rows > (1ll << 31)) {
    set_error("%s: bad sizes (rows to 2^31, dim and hidden to 2^24)", what);
    return 1;
  }
  const int64_t tiles = (a->rows + 127) / 128 * ((a->hidden > a->dim ? a->hidden : a->dim) / 64 + 1);
  if (tiles > 0x7ffffff0ll || a->dim * a->hidden > (1ll << 39)) { set_error("%s: too large", what); return 1; }
  return 0;
}

template <typename T>
static MatOperand operand(const void* p, int64_t stride, int64_t extent) {
  return MatOperand{static_cast<const char*>(p), stride * static_cast<int64_t>(sizeof(T)), extent};
}

template <typename T> static void mlp_fwd(const fovi_gated_mlp_args* a, hipStream_t s) {
  const int64_t M = a->rows, C = a->dim, F = a->hidden;
  T* h = static_cast<T*>(a->workspace);
  T* gate = static_cast<T*>(a->saved);
  const MlpGated<T> gated = {h, F, a->activation, gate, gate + F, 2 * F};
  mlp_gated_kernel<T, 128, 64><<<mat_grid(tiles_of(M, 128) * tiles_of(F, 64)), 256, 0, s>>>(
      operand<T>(a->x, a->x_stride, M), operand<T>(a->w_gate, a->w_gate_stride, F), operand<T>(a->w_up, a->w_up_stride, F), C, M, F, gated);
  const MatSegments down = {{operand<T>(h, F, M)}, {operand<T>(a->w_down, a->w_down_stride, C)}, {F, 0}, 1};
  const MlpLinear<T> linear = {static_cast<T*>(a->y), a->y_stride, static_cast<const T*>(a->residual), a->residual_stride};
  mlp_linear<T, false, false>(down, M, C, linear, s);
}

static int64_t aligned(int64_t n) { return (n + 255) & ~static_cast<int64_t>(255); }

template <typename T> static void mlp_bwd(const fovi_gated_mlp_args* a, hipStream_t s) {
  const int64_t M = a->rows, C = a->dim, F = a->hidden;
  char* work = static_cast<char*>(a->workspace);
  T* grad = reinterpret_cast<T*>(work);                             // [M, 2 F]: dgate, dup
  T* h = reinterpret_cast<T*>(work + aligned(M * 2 * F * sizeof(T)));
  float* part = reinterpret_cast<float*>(reinterpret_cast<char*>(h) + aligned(M * F * sizeof(T)));
  const MatOperand x = operand<T>(a->x, a->x_stride, M), dy = operand<T>(a->dy, a->dy_stride, M);
  const MatOperand wg = operand<T>(a->w_gate, a->w_gate_stride, F), wu = operand<T>(a->w_up, a->w_up_stride, F);
  const MatOperand wd = operand<T>(a->w_down, a->w_down_stride, F); // by columns: k runs over its rows
  const T* gate = static_cast<const T*>(a->saved);
  const MlpGatedGrad<T> gated = {grad, grad + F, h, 2 * F, F, a->activation, gate, gate + F, 2 * F};
  if (gate) {
    const MatSegments down = {{dy}, {wd}, {C, 0}, 1};
    mlp_linear<T, false, true>(down, M, F, gated, s);
  } else {
    mlp_gated_grad_kernel<T, 128, 64><<<mat_grid(tiles_of(M, 128) * tiles_of(F, 64)), 256, 0, s>>>(x, wg, wu, dy, wd, C, M, F, gated);
  }
  if (a->dx) {
    const MatSegments both = {{operand<T>(grad, 2 * F, M), operand<T>(grad + F, 2 * F, M)},
                              {operand<T>(a->w_gate, a->w_gate_stride, C), operand<T>(a->w_up, a->w_up_stride, C)}, {F, F}, 2};
    mlp_linear<T, false, true>(both, M, C, MlpLinear<T>{static_cast<T*>(a->dx), C, nullptr, 0}, s);
  }
  if (a->dw_gate)
    token_product<T>(operand<T>(grad, 2 * F, 2 * F), operand<T>(a->x, a->x_stride, C), M, 2 * F, C, part,
                     MlpTwoRows<T>{{static_cast<T*>(a->dw_gate), static_cast<T*>(a->dw_up)}, F, C}, s);
  if (a->dw_down)
    token_product<T>(operand<T>(a->dy, a->dy_stride, C), operand<T>(h, F, F), M, C, F, part,
                     MlpLinear<T>{static_cast<T*>(a->dw_down), F, nullptr, 0}, s);
}

}  // namespace fovi

using namespace fovi;

extern "C" int64_t fovi_gated_mlp_saved_bytes(int64_t rows, int64_t dim, int64_t hidden, int32_t dtype) {
  (void)dim;
  return dtype == FOVI_F32 && rows > 0 && hidden > 0 ? rows * 2 * hidden * 4 : 0;
}

extern "C" int64_t fovi_gated_mlp_fwd_workspace_bytes(int64_t rows, int64_t dim, int64_t hidden, int32_t dtype) {
  (void)dim;
  return rows > 0 && hidden > 0 ? rows * hidden * (dtype == FOVI_F32 ? 4 : 2) : 0;
}

extern "C" int64_t fovi_gated_mlp_bwd_workspace_bytes(int64_t rows, int64_t dim, int64_t hidden, int32_t dtype) {
  if (rows < 1 || dim < 1 || hidden < 1) return 0;
  const int64_t es = dtype == FOVI_F32 ? 4 : 2;
  const int64_t a = token_shares(rows, 2 * hidden, dim) * 2 * hidden * dim, b = token_shares(rows, dim, hidden) * dim * hidden;
  return aligned(rows * 2 * hidden * es) + aligned(rows * hidden * es) + (a > b ? a : b) * 4;
}

extern "C" int fovi_gated_mlp_fwd(const fovi_gated_mlp_args* a, void* stream) {
  clear_error();
  if (mlp_check(a, "fovi_gated_mlp_fwd")) return 1;
  if (a->rows == 0) return 0;
  const int64_t need = fovi_gated_mlp_fwd_workspace_bytes(a->rows, a->dim, a->hidden, a->dtype);
  if (!a->y || !a->workspace || a->workspace_bytes < need) {
    set_error("fovi_gated_mlp_fwd: y and a workspace of %lld bytes needed", static_cast<long long>(need));
    return 1;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == FOVI_BF16) mlp_fwd<uint16_t>(a, s);
  else mlp_fwd<float>(a, s);
  return check_launch("fovi_gated_mlp_fwd");
}

extern "C" int fovi_gated_mlp_bwd(const fovi_gated_mlp_args* a, void* stream) {
  clear_error();
  if (mlp_check(a, "fovi_gated_mlp_bwd")) return 1;
  if (!a->dy || !a->dw_gate != !a->dw_up) { set_error("fovi_gated_mlp_bwd: null pointer"); return 1; }
  if (a->rows == 0) { set_error("fovi_gated_mlp_bwd: no rows"); return 1; }
  if (!a->saved && fovi_gated_mlp_saved_bytes(a->rows, a->dim, a->hidden, a->dtype)) {
    set_error("fovi_gated_mlp_bwd: the forward's gate and up are needed");
    return 1;
  }
  const int64_t need = fovi_gated_mlp_bwd_workspace_bytes(a->rows, a->dim, a->hidden, a->dtype);
  if (!a->workspace || a->workspace_bytes < need) {
    set_error("fovi_gated_mlp_bwd: workspace of %lld bytes needed", static_cast<long long>(need));
    return 1;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == FOVI_BF16) mlp_bwd<uint16_t>(a, s);
  else mlp_bwd<float>(a, s);
  return check_launch("fovi_gated_mlp_bwd");
}
