// Products of 8-bit integers with a scale for each token and for each output channel, for serving:
//
//   y[m, n] = (sum_k x[m, k] w[n, k]) * sx[m] * sw[n] + bias[n] + residual[m, n]
//   gated: act(gate[m, n]) * up[m, n] of two such products over the same rows
//
// The sums are exact (int32 holds 133,000 products of 127 * 127); they become floats once, times the two scales.
#include "matmul.h"

namespace fovi {

struct Int8Scales {
  const float* x; const float* w; const float* w2;
};

template <typename TO> struct Int8Linear {
  Int8Scales s;
  const float* bias; const TO* residual; int64_t residual_stride;
  TO* out; int64_t stride;
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, int count, const int32_t (&v)[1][4]) const {
    const float sx = s.x[m];
    float y[4], w[4], t[4];
    load_four(s.w + n, count, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = static_cast<float>(v[0][i]) * sx * w[i];
    if (bias) {
      load_four(bias + n, count, t);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] += t[i];
    }
    if (residual) {
      load_four(residual + m * residual_stride + n, count, t);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] += t[i];
    }
    store_four(out + m * stride + n, count, y);
  }
};

template <typename TO> struct Int8Gated {
  Int8Scales s;
  int act;
  TO* out; int64_t stride;
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, int count, const int32_t (&v)[2][4]) const {
    const float sx = s.x[m];
    float y[4], g[4], u[4];
    load_four(s.w + n, count, g);
    load_four(s.w2 + n, count, u);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      y[i] = mat_act<false>(static_cast<float>(v[0][i]) * sx * g[i], act) * (static_cast<float>(v[1][i]) * sx * u[i]);
    store_four(out + m * stride + n, count, y);
  }
};

template <int BM, int BN, int NB, typename Epilogue>
__global__ __launch_bounds__(256) void int8_kernel(MatOperand x, MatOperand w0, MatOperand w1, int64_t K, int64_t M, int64_t N,
                                                   Epilogue epilogue) {
  typedef MatCore<int8_t, BM, BN, NB, false, false> Core;
  __shared__ __attribute__((aligned(16))) char lds[Core::LDS];
  int64_t tm, tn;
  if (!mat_tile((M + BM - 1) / BM, (N + BN - 1) / BN, tm, tn)) return;
  typename Core::Acc acc[NB][Core::MB][Core::NN];
  mat_clear(acc);
  const MatOperand w[2] = {w0, w1};
  Core::run(x, w, tm * BM, tn * BN, 0, K, lds, acc);
  mat_finish<BM, BN, int32_t>(acc, tm * BM, tn * BN, M, N, epilogue);
}

template <typename TO> static void int8_launch(const fovi_linear_int8_args* a, hipStream_t stream) {
  const int64_t M = a->rows, N = a->outputs, K = a->inputs;
  const MatOperand x = {reinterpret_cast<const char*>(a->x), a->x_stride, M}, w = {reinterpret_cast<const char*>(a->weight), a->weight_stride, N},
                   w2 = {reinterpret_cast<const char*>(a->weight2), a->weight2_stride, N};
  const Int8Scales scales = {a->x_scale, a->weight_scale, a->weight2_scale};
  TO* out = static_cast<TO*>(a->out);
  const int64_t tm = (M + 127) / 128;
  if (a->weight2) {
    const Int8Gated<TO> gated = {scales, a->activation, out, a->out_stride};
    int8_kernel<128, 64, 2, Int8Gated<TO>><<<mat_grid(tm * ((N + 63) / 64)), 256, 0, stream>>>(x, w, w2, K, M, N, gated);
  } else {
    const Int8Linear<TO> linear = {scales, a->bias, static_cast<const TO*>(a->residual), a->residual_stride, out, a->out_stride};
    int8_kernel<128, 128, 1, Int8Linear<TO>><<<mat_grid(tm * ((N + 127) / 128)), 256, 0, stream>>>(x, w, w, K, M, N, linear);
  }
}

}  // namespace fovi

using namespace fovi;

extern "C" int64_t fovi_linear_int8_workspace_bytes(int64_t rows, int64_t inputs, int64_t outputs, int32_t gated) {
  (void)rows; (void)inputs; (void)outputs; (void)gated;
  return 0;
}

extern "C" int fovi_linear_int8(const fovi_linear_int8_args* a, void* stream) {
  clear_error();
  if (!a || !a->x || !a->x_scale || !a->weight || !a->weight_scale || !a->out || !a->weight2 != !a->weight2_scale) {
    set_error("fovi_linear_int8: null pointer");
    return 1;
  }
  if (a->out_dtype != FOVI_F32 && a->out_dtype != FOVI_BF16) { set_error("fovi_linear_int8: out_dtype must be F32 or BF16"); return 1; }
  if (a->weight2 && (a->bias || a->residual)) { set_error("fovi_linear_int8: no bias or residual beside weight2"); return 1; }
  if (a->weight2 && a->activation != FOVI_GATE_SILU && a->activation != FOVI_GATE_GELU) {
    set_error("fovi_linear_int8: unknown activation");
    return 1;
  }
  if (a->rows < 0 || a->outputs < 0 || a->inputs < 1 || a->inputs > 131072) {
    set_error("fovi_linear_int8: bad sizes (1 to 131072 inputs)");
    return 1;
  }
  if (a->rows == 0 || a->outputs == 0) return 0;
  if ((a->rows + 127) / 128 > 0x7fffff00ll / ((a->outputs + 63) / 64)) { set_error("fovi_linear_int8: too large"); return 1; }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->out_dtype == FOVI_BF16) int8_launch<uint16_t>(a, s);
  else int8_launch<float>(a, s);
  return check_launch("fovi_linear_int8");
}
