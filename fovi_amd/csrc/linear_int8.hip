// Products of 8-bit integers with a scale for each token and for each output channel, for serving:
//
//   y[m, n] = (sum_k x[m, k] w[n, k]) * sx[m] * sw[n] + bias[n] + residual[m, n]
//   gated: act(gate[m, n]) * up[m, n] of two such products over the same rows
//
// The sums are exact (int32 holds 131,071 products of -128 * -128); they become floats once, times the two scales.
//
// Bound by products and epilogue one after the other where there are many rows (16384 x 1024 by 2 x 2752: 124 us, 1.49 POP/s; 91
// without the epilogue, 112 without the loads, or without the activation), by the weights' way from memory where there are few
// (48 x 4096 by 11008: 12.7 us, 3.6 TB/s). fp32 results pay for the library's exponential and division: 143 us for 16384 rows.
#include "matmul_few.h"

namespace fovi {

struct Int8Scales {
  const float* x; const float* w; const float* w2;
};

template <typename TO> struct Int8Linear {
  static constexpr int STORES = sizeof(TO) / 2;        // of 16 bytes for a run of eight
  struct Column { Run<float> w, bias; };
  struct Extra { Run<TO> residual; float x; };
  Int8Scales s;
  const float* bias; const TO* residual; int64_t residual_stride;
  TO* out; int64_t stride;
  __device__ __forceinline__ Column column(int64_t n, int count) const {
    Column c = {};
    c.w.load(s.w + n, count);
    if (bias) c.bias.load(bias + n, count);
    return c;
  }
  __device__ __forceinline__ Extra load(int64_t m, int64_t n, int count) const {
    Extra e = {};
    e.x = s.x[m];
    if (residual) e.residual.load(residual + m * residual_stride + n, count);
    return e;
  }
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, int count, const int32_t (&v)[1][8], const Column& c, const Extra& e) const {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = static_cast<float>(v[0][i]) * e.x * c.w[i];
      if (bias) y[i] += c.bias[i];
      if (residual) y[i] += e.residual[i];
    }
    store_run(out + m * stride + n, count, y);
  }
};

template <typename TO> struct Int8Gated {
  static constexpr int STORES = sizeof(TO) / 2;
  struct Column { Run<float> gate, up; };
  typedef float Extra;
  Int8Scales s;
  int act;
  TO* out; int64_t stride;
  __device__ __forceinline__ Column column(int64_t n, int count) const {
    Column c;
    c.gate.load(s.w + n, count);
    c.up.load(s.w2 + n, count);
    return c;
  }
  __device__ __forceinline__ Extra load(int64_t m, int64_t, int) const { return s.x[m]; }
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, int count, const int32_t (&v)[2][8], const Column& c, const Extra& x) const {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      y[i] = mat_act<sizeof(TO) == 4>(static_cast<float>(v[0][i]) * x * c.gate[i], act) * (static_cast<float>(v[1][i]) * x * c.up[i]);
    store_run(out + m * stride + n, count, y);
  }
};

template <int BM, int BN, typename Epilogue> struct Int8GatedTile {
  typedef MatPhase<int8_t, BM, BN, 2, false, false> Phase;
  typedef MatRing<Phase::BYTES, 2 * Phase::MB * Phase::NN * Epilogue::STORES> Ring;
};

template <int BM, int BN, typename Epilogue>
__global__ __launch_bounds__((MatUsual<BM, BN>::THREADS), 2) void int8_gated_kernel(MatOperand x, MatOperand w0, MatOperand w1, int64_t K, int64_t M, int64_t N, MatWork work,
                                                      Epilogue epilogue) {
  typedef typename Int8GatedTile<BM, BN, Epilogue>::Phase Phase;
  typedef typename Int8GatedTile<BM, BN, Epilogue>::Ring Ring;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  MatItem item(work), ahead(work);
  if (!item.live()) return;
  const MatOperand w[2] = {w0, w1};
  Phase phase;
  int64_t left = -1;                                   // of the tile `ahead`; -1: not begun
  auto produce = [&](uint32_t to) __attribute__((always_inline)) {
    if (left <= 0) {
      if (left == 0) ahead.next();
      if (!ahead.live()) return false;
      left = K;
      int64_t tm, tn;
      ahead.place(work, tm, tn);
      phase.open(x, w, tm * BM, tn * BN, 0);
    }
    phase.start(to, left);
    left = left > Phase::BK ? left - Phase::BK : 0;
    return true;
  };
  Ring ring(lds, produce);
  typename Phase::Step step[2];
  auto first_step = [&](const char* now) __attribute__((always_inline)) { step[0].read(now, 0); };
  first_step(ring.now());
  const int64_t stages = (K + Phase::BK - 1) / Phase::BK;
  for (; item.live(); item.next()) {
    typename Phase::Acc acc[2][Phase::MB][Phase::NN];
    mat_clear(acc);
    Phase::run(ring, stages, step, acc, 0, produce, first_step);
    int64_t tm, tn;
    item.place(work, tm, tn);
    ring.stored = mat_finish<typename Phase::Waves, BM, BN, int32_t>(acc, tm * BM, tn * BN, M, N, epilogue);
  }
}

template <int BM, int BN, typename Epilogue>
static void int8_gated_tiles(const MatOperand& x, const MatOperand& w0, const MatOperand& w1, int64_t K, int64_t M, int64_t N,
                             const Epilogue& epilogue, hipStream_t s) {
  const MatWork work = mat_work(M, N, BM, BN, 1);
  mat_launch(int8_gated_kernel<BM, BN, Epilogue>, mat_grid(work, 256 / BM), (MatUsual<BM, BN>::THREADS),
             Int8GatedTile<BM, BN, Epilogue>::Ring::LDS, s, x, w0, w1, K, M, N, work, epilogue);
}
template <typename Epilogue>
static void int8_gated(const MatOperand& x, const MatOperand& w0, const MatOperand& w1, int64_t K, int64_t M, int64_t N,
                       const Epilogue& epilogue, hipStream_t s) {
  const int size = mat_tile_size(M, 2 * N, 1, false, 256);
  if (size == 256) int8_gated_tiles<256, 128>(x, w0, w1, K, M, N, epilogue, s);
  else if (size == 128) int8_gated_tiles<128, 64>(x, w0, w1, K, M, N, epilogue, s);
  else int8_gated_tiles<64, 64>(x, w0, w1, K, M, N, epilogue, s);
}

struct Int8Inputs {
  MatInputs in;
  MatOperand x, w, w2;
  Int8Inputs(const fovi_linear_int8_args* a, void* workspace) : in(workspace) {
    x = in.take(a->x, a->x_stride, a->rows, a->inputs, 1);
    w = in.take(a->weight, a->weight_stride, a->outputs, a->inputs, 1);
    w2 = a->weight2 ? in.take(a->weight2, a->weight2_stride, a->outputs, a->inputs, 1) : w;
  }
};

static bool int8_few(const fovi_linear_int8_args* a) { return few_rows_best(a->rows, a->outputs, a->weight2 != nullptr); }

template <typename TO> static void int8_launch(const fovi_linear_int8_args* a, hipStream_t stream) {
  const int64_t M = a->rows, N = a->outputs, K = a->inputs;
  const Int8Scales scales = {a->x_scale, a->weight_scale, a->weight2_scale};
  TO* out = static_cast<TO*>(a->out);
  const Int8Gated<TO> gated = {scales, a->activation, out, a->out_stride};
  const Int8Linear<TO> linear = {scales, a->bias, static_cast<const TO*>(a->residual), a->residual_stride, out, a->out_stride};
  if (int8_few(a)) {
    const MatOperand x = {reinterpret_cast<const char*>(a->x), a->x_stride, M}, w = {reinterpret_cast<const char*>(a->weight), a->weight_stride, N},
                     w2 = {reinterpret_cast<const char*>(a->weight2), a->weight2_stride, N};
    if (a->weight2) few_product<int8_t, 2>(x, w, w2, K, M, N, gated, stream);
    else few_product<int8_t, 1>(x, w, w, K, M, N, linear, stream);
    return;
  }
  const Int8Inputs in(a, a->workspace);
  in.in.copy(stream);
  if (a->weight2) {
    int8_gated(in.x, in.w, in.w2, K, M, N, gated, stream);
  } else {
    const MatSegments s = {{in.x}, {in.w}, {K, 0}, 1};
    mat_linear<int8_t, false, false>(s, M, N, in.in.rest(), false, linear, stream);
  }
}

}  // namespace fovi

using namespace fovi;

extern "C" int64_t fovi_linear_int8_workspace_bytes(const fovi_linear_int8_args* a) {
  if (!a || a->rows < 1 || a->inputs < 1 || a->outputs < 1 || int8_few(a)) return 0;
  return Int8Inputs(a, nullptr).in.used() + (a->weight2 ? 0 : mat_part_bytes<int8_t>(a->rows, a->outputs, a->inputs, false));
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
  if (a->rows < 0 || a->outputs < 0 || a->inputs < 1 || a->inputs > 131071) {
    set_error("fovi_linear_int8: bad sizes (1 to 131071 inputs)");
    return 1;
  }
  if (a->rows == 0 || a->outputs == 0) return 0;
  if (a->rows > (1ll << 31) || (a->rows + 63) / 64 > (1ll << 30) / ((a->outputs + 63) / 64)) { set_error("fovi_linear_int8: too large"); return 1; }
  const int64_t need = fovi_linear_int8_workspace_bytes(a);
  if (need && (!a->workspace || a->workspace_bytes < need)) {
    set_error("fovi_linear_int8: workspace of %lld bytes needed", static_cast<long long>(need));
    return 1;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->out_dtype == FOVI_BF16) int8_launch<uint16_t>(a, s);
  else int8_launch<float>(a, s);
  return check_launch("fovi_linear_int8");
}
