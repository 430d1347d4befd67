// The gated feed-forward block of token rows and its gradients.
//
//   gate = x Wg^T, up = x Wu^T, h = act(gate) * up, y = h Wd^T (+ residual)
//   dh = dy Wd, dgate = dh * up * act'(gate), dup = dh * act(gate)
//   dx = dgate Wg + dup Wu, dWg = dgate^T x, dWu = dup^T x, dWd = dy^T h
//
// Both first projections run over one tile of x, and h is all that leaves them, but for gate and up where they are kept
// for the backward (fp32, wide bf16 rows). The backward forms dh, or gate, up and dh in the registers of one kernel,
// whose epilogue writes dgate, dup and h. The weights' gradients reduce over the tokens: the tokens are split over workgroups, whose
// partial sums a second launch adds in a fixed order.
//
// 131072 rows of 384, hidden 1024, in bf16: gate, up and h 281 us (206 GFLOP), y 126 (103), gate, up and dh 615 (309), dx 238
// (206), dWg and dWu 222 + 10 (206), dWd 141 + 13 (103): 1646 us. What bounds the first and the third is that a compute
// unit's waves are in the epilogue together: without it they take 180 and 371 us, without their loads 207 and 427. 32 rows
// of 2048, hidden 5504: 13.0 and 8.0 us (68 MB).
#include "matmul_few.h"

namespace fovi {

// Runs of h, dgate and dup are written whole, with zeros behind the last column: the products that read them go by 16 bytes.
__device__ __forceinline__ void clear_behind(int count, float (&v)[8]) {
#pragma unroll
  for (int i = 1; i < 8; ++i) v[i] = i < count ? v[i] : 0.0f;
}

template <typename T> struct MlpLinear : NoColumn {               // out = sums (+ residual)
  static constexpr int STORES = sizeof(T) / 2;         // of 16 bytes for a run of eight
  typedef Run<T> Extra;
  T* out; int64_t stride;
  const T* residual; int64_t residual_stride;
  __device__ __forceinline__ Extra load(int64_t m, int64_t n, int count) const {
    Extra r = {};
    if (residual) r.load(residual + m * residual_stride + n, count);
    return r;
  }
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, int count, const float (&v)[1][8], const NoExtra&, const Extra& r) const {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = residual ? v[0][i] + r[i] : v[0][i];
    store_run(out + m * stride + n, count, y);
  }
};

template <typename T> struct MlpTwoRows : Plain {              // `rows` rows to one output, those from `next` on to the other
  static constexpr int STORES = 0;                     // rows between the two are not stored
  T* out[2]; int64_t rows, next, stride;
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, int count, const float (&v)[1][8], const NoExtra&, const NoExtra&) const {
    if (m < rows) store_run(out[0] + m * stride + n, count, v[0]);
    else if (m >= next) store_run(out[1] + (m - next) * stride + n, count, v[0]);
  }
};

template <typename T> struct MlpGated : Plain {                // h, and gate and up where a backward will read them
  static constexpr int STORES = sizeof(T) / 2;
  T* h; int64_t stride; int act;
  T* gate; T* up; int64_t saved_stride;
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, int count, const float (&v)[2][8], const NoExtra&, const NoExtra&) const {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = mat_act<sizeof(T) == 4>(v[0][i], act) * v[1][i];
    clear_behind(count, y);
    store_run(h + m * stride + n, 8, y);
    if (gate) {
      store_run(gate + m * saved_stride + n, count, v[0]);
      store_run(up + m * saved_stride + n, count, v[1]);
    }
  }
};

// dgate, dup and h of a run of gate, up and dh.
template <typename T> struct MlpGradRows {
  static constexpr int STORES = 3 * sizeof(T) / 2;
  T* dgate; T* dup; T* h; int64_t stride, h_stride; int act;
  template <typename G, typename U>
  __device__ __forceinline__ void write(int64_t m, int64_t n, int count, const G& g, const U& u, const float (&dh)[8]) const {
    float a[8], b[8], c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float value, slope;
      mat_act_grad<sizeof(T) == 4>(g[i], act, value, slope);
      a[i] = dh[i] * u[i] * slope;
      b[i] = dh[i] * value;
      c[i] = value * u[i];
    }
    clear_behind(count, a);
    clear_behind(count, b);
    clear_behind(count, c);
    store_run(dgate + m * stride + n, 8, a);
    store_run(dup + m * stride + n, 8, b);
    store_run(h + m * h_stride + n, 8, c);
  }
};
template <typename T> struct MlpGatedGrad : Plain, MlpGradRows<T> {   // of all three sums
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, int count, const float (&v)[3][8], const NoExtra&, const NoExtra&) const {
    this->write(m, n, count, v[0], v[1], v[2]);
  }
};
template <typename T> struct MlpSavedGrad : NoColumn, MlpGradRows<T> { // of dh's sums and the gate and up of the forward
  struct Extra { Run<T> gate, up; };
  const T* gate; const T* up; int64_t saved_stride;
  __device__ __forceinline__ Extra load(int64_t m, int64_t n, int count) const {
    Extra x;
    x.gate.load(gate + m * saved_stride + n, count);
    x.up.load(up + m * saved_stride + n, count);
    return x;
  }
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, int count, const float (&v)[1][8], const NoExtra&, const Extra& x) const {
    this->write(m, n, count, x.gate, x.up, v[0]);
  }
};
template <typename T> constexpr bool mat_narrow<MlpSavedGrad<T>> = true;

template <typename T, int BM, int BN> struct MlpGatedTile {
  typedef MatPhase<T, BM, BN, 2, false, false> Both;
  typedef MatRing<Both::BYTES, 2 * Both::MB * Both::NN * MlpGated<T>::STORES> Ring;
};
template <typename T, int BM, int BN, typename W> struct MlpGradTile {
  typedef MatPhase<T, BM, BN, 2, false, false, W> Both;
  typedef MatPhase<T, BM, BN, 1, false, true, W> Down;
  typedef MatRing<Both::BYTES, 2 * Both::MB * Both::NN * MlpGatedGrad<T>::STORES> Ring;
};

template <typename T, int BM, int BN>
__global__ __launch_bounds__((MatUsual<BM, BN>::THREADS), 2) void mlp_gated_kernel(MatOperand x, MatOperand wg, MatOperand wu, int64_t K, int64_t M, int64_t N,
                                                           MatWork work, MlpGated<T> epilogue) {
  typedef typename MlpGatedTile<T, BM, BN>::Both Phase;
  typedef typename MlpGatedTile<T, BM, BN>::Ring Ring;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  MatItem item(work), ahead(work);
  if (!item.live()) return;
  const MatOperand w[2] = {wg, wu};
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
    ring.stored = mat_finish<typename Phase::Waves, BM, BN, float>(acc, tm * BM, tn * BN, M, N, epilogue);
  }
}

// gate, up and dh of a tile, one after the other, and what the epilogue makes of them.
template <typename T, int BM, int BN, typename W>
__global__ __launch_bounds__(W::THREADS, 2) void mlp_gated_grad_kernel(MatOperand x, MatOperand wg, MatOperand wu, MatOperand dy, MatOperand wd,
                                                                int64_t K, int64_t M, int64_t N, MatWork work, MlpGatedGrad<T> epilogue) {
  typedef typename MlpGradTile<T, BM, BN, W>::Both Both;
  typedef typename MlpGradTile<T, BM, BN, W>::Down Down;
  typedef typename MlpGradTile<T, BM, BN, W>::Ring Ring;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  MatItem item(work), ahead(work);
  if (!item.live()) return;
  const MatOperand w[2] = {wg, wu}, d[1] = {wd};
  Both both;
  Down down;
  int64_t left = -1;
  bool second = true;                                  // which of the two runs of stages `left` belongs to
  auto produce = [&](uint32_t to) __attribute__((always_inline)) {
    if (left <= 0) {
      if (left == 0 && second) ahead.next();
      if (!ahead.live()) return false;
      left = K;
      second = !second;
      int64_t tm, tn;
      ahead.place(work, tm, tn);
      if (second) down.open(dy, d, tm * BM, tn * BN, 0);
      else both.open(x, w, tm * BM, tn * BN, 0);
    }
    if (second) down.start(to, left);
    else both.start(to, left);
    left = left > Both::BK ? left - Both::BK : 0;
    return true;
  };
  Ring ring(lds, produce);
  const int64_t stages = (K + Both::BK - 1) / Both::BK;
  for (; item.live(); item.next()) {
    typename Both::Acc acc[3][Both::MB][Both::NN];
    mat_clear(acc);
    Both::run_lean(ring, stages, acc, 0, produce);
    Down::run_lean(ring, stages, acc, 2, produce);
    int64_t tm, tn;
    item.place(work, tm, tn);
    ring.stored = mat_finish<W, BM, BN, float>(acc, tm * BM, tn * BN, M, N, epilogue);
  }
}

static int mlp_check(const fovi_gated_mlp_args* a, const char* what) {
  if (!a || !a->x || !a->w_gate || !a->w_up || !a->w_down) { set_error("%s: null pointer", what); return 1; }
  if (a->dtype != FOVI_F32 && a->dtype != FOVI_BF16) { set_error("%s: dtype must be F32 or BF16", what); return 1; }
  if (a->activation != FOVI_GATE_SILU && a->activation != FOVI_GATE_GELU) { set_error("%s: unknown activation", what); return 1; }
  if (a->rows < 0 || a->dim < 1 || a->hidden < 1 || a->dim > (1 << 19) || a->hidden > (1 << 19) || a->rows > (1ll << 31)) {
    set_error("%s: bad sizes (rows to 2^31, dim and hidden to 2^19)", what);
    return 1;
  }
  const int64_t widest = a->hidden > a->dim ? a->hidden : a->dim;
  if (((a->rows > widest ? a->rows : widest) + 63) / 64 > (1ll << 30) / ((widest + 63) / 64)) { set_error("%s: too large", what); return 1; }
  return 0;
}

static int64_t mlp_element(const fovi_gated_mlp_args* a) { return a->dtype == FOVI_F32 ? 4 : 2; }
static int64_t aligned(int64_t n) { return (n + 255) & ~static_cast<int64_t>(255); }
static int64_t wide(int64_t n) { return (n + 7) & ~static_cast<int64_t>(7); }

struct MlpInputs {
  MatInputs in;
  MatOperand x, wg, wu, wd, dy;
  MlpInputs(const fovi_gated_mlp_args* a, void* workspace, bool backward) : in(workspace) {
    const int64_t es = mlp_element(a);
    x = in.take(a->x, a->x_stride, a->rows, a->dim, es);
    wg = in.take(a->w_gate, a->w_gate_stride, a->hidden, a->dim, es);
    wu = in.take(a->w_up, a->w_up_stride, a->hidden, a->dim, es);
    wd = in.take(a->w_down, a->w_down_stride, a->dim, a->hidden, es);
    if (backward) dy = in.take(a->dy, a->dy_stride, a->rows, a->dim, es);
  }
};

// The operand's columns as rows of an operand by columns.
static MatOperand columns(const MatOperand& o, int64_t n, int64_t es) { return MatOperand{o.p, o.stride, (n * es + 15) / 16 * 16 / es}; }

template <typename T, int BM, int BN>
static void mlp_gated_tiles(const MlpInputs& in, int64_t C, int64_t M, int64_t F, const MlpGated<T>& epilogue, hipStream_t s) {
  const MatWork work = mat_work(M, F, BM, BN, 1);
  mat_launch(mlp_gated_kernel<T, BM, BN>, mat_grid(work, 256 / BM), (MatUsual<BM, BN>::THREADS), MlpGatedTile<T, BM, BN>::Ring::LDS, s, in.x, in.wg, in.wu, C, M, F, work,
             epilogue);
}
template <typename T, int BM, int BN, typename W>
static void mlp_gated_grad_tiles(const MlpInputs& in, const MatOperand& wd, int64_t C, int64_t M, int64_t F, const MlpGatedGrad<T>& epilogue,
                                 hipStream_t s) {
  const MatWork work = mat_work(M, F, BM, BN, 1);
  mat_launch(mlp_gated_grad_kernel<T, BM, BN, W>, mat_grid(work, BM == 64 ? 3 : 2), W::THREADS, MlpGradTile<T, BM, BN, W>::Ring::LDS, s, in.x, in.wg, in.wu, in.dy, wd, C,
             M, F, work, epilogue);
}

// Whether the forward keeps gate and up for the backward: 4 bytes a pair and row in bf16, where forming them again costs
// 4 dim operations. Both directions in bf16, us, kept and formed again: 131072 x 384 by 1024 1735 and 1640, 65536 x 512 by
// 1344 1412 and 1355, 32768 x 768 by 2048 1485 and 1493, 8192 x 1536 by 4096 1270 and 1362, 4572 x 2048 by 5504 1266
// and 1412. fp32 products are slow enough to keep always.
constexpr int64_t kKeepDim = 768;
static bool mlp_keeps(int64_t dim, int32_t dtype) { return dtype == FOVI_F32 || dim >= kKeepDim; }
static bool mlp_keeps(const fovi_gated_mlp_args* a) { return mlp_keeps(a->dim, a->dtype); }
static bool mlp_few(const fovi_gated_mlp_args* a) {
  return few_rows_best(a->rows, a->hidden > a->dim ? a->hidden : a->dim, a->dtype == FOVI_F32);
}

template <typename T> static MatOperand as_is(const void* p, int64_t stride, int64_t rows) {
  return MatOperand{static_cast<const char*>(p), stride * static_cast<int64_t>(sizeof(T)), rows};
}

template <typename T> static void mlp_fwd(const fovi_gated_mlp_args* a, hipStream_t s) {
  const int64_t M = a->rows, C = a->dim, F = a->hidden, Fp = wide(F);
  T* gate = static_cast<T*>(a->saved);
  const MlpLinear<T> linear = {{}, static_cast<T*>(a->y), a->y_stride, static_cast<const T*>(a->residual), a->residual_stride};
  MlpGated<T> gated = {{}, static_cast<T*>(a->workspace), Fp, a->activation, gate, gate + F, 2 * F};
  if (mlp_few(a)) {
    few_product<T, 2>(as_is<T>(a->x, a->x_stride, M), as_is<T>(a->w_gate, a->w_gate_stride, F), as_is<T>(a->w_up, a->w_up_stride, F), C, M, F,
                      gated, s);
    const MatOperand wd = as_is<T>(a->w_down, a->w_down_stride, C);
    few_product<T, 1>(as_is<T>(gated.h, Fp, M), wd, wd, F, M, C, linear, s);
    return;
  }
  const MlpInputs in(a, a->workspace, false);
  in.in.copy(s);
  gated.h = reinterpret_cast<T*>(in.in.rest());
  const int size = mat_tile_size(M, 2 * F, 1, sizeof(T) == 4, 256);
  if constexpr (sizeof(T) == 2) {
    if (size == 256) mlp_gated_tiles<T, 256, 128>(in, C, M, F, gated, s);
  }
  if (size == 128) mlp_gated_tiles<T, 128, 64>(in, C, M, F, gated, s);
  else if (size == 64) mlp_gated_tiles<T, 64, 64>(in, C, M, F, gated, s);
  const MatSegments down = {{as_is<T>(gated.h, Fp, M)}, {in.wd}, {F, 0}, 1};
  mat_linear<T, false, false>(down, M, C, reinterpret_cast<char*>(gated.h) + aligned(M * Fp * sizeof(T)), false, linear, s);
}

template <typename T> static void mlp_bwd(const fovi_gated_mlp_args* a, hipStream_t s) {
  const int64_t M = a->rows, C = a->dim, F = a->hidden, Fp = wide(F), es = sizeof(T);
  const MlpInputs in(a, a->workspace, true);
  in.in.copy(s);
  T* grad = reinterpret_cast<T*>(in.in.rest());                     // [M, 2 Fp]: dgate, dup
  T* h = reinterpret_cast<T*>(in.in.rest() + aligned(M * 2 * Fp * es));
  char* part = reinterpret_cast<char*>(h) + aligned(M * Fp * es);
  const MatOperand wd = columns(in.wd, F, es);
  const MlpGradRows<T> rows = {grad, grad + Fp, h, 2 * Fp, Fp, a->activation};
  if (mlp_keeps(a)) {
    const T* gate = static_cast<const T*>(a->saved);
    const MatSegments down = {{in.dy}, {wd}, {C, 0}, 1};
    mat_linear<T, false, true>(down, M, F, part, false, MlpSavedGrad<T>{{}, rows, gate, gate + F, 2 * F}, s);
  } else if constexpr (sizeof(T) == 2) {
    const MlpGatedGrad<T> gated = {{}, rows};
    const int size = mat_tile_size(M, 2 * F, 1, false, 256);
    if (size >= 128) mlp_gated_grad_tiles<T, 128, 64, MatWaves<2, 2>>(in, wd, C, M, F, gated, s);
    else mlp_gated_grad_tiles<T, 64, 64, MatWaves<2, 2>>(in, wd, C, M, F, gated, s);
  }
  const char* dgate = reinterpret_cast<const char*>(grad);
  if (a->dx) {
    const MatSegments both = {{MatOperand{dgate, 2 * Fp * es, M}, MatOperand{dgate + Fp * es, 2 * Fp * es, M}},
                              {columns(in.wg, C, es), columns(in.wu, C, es)}, {F, F}, 2};
    mat_linear<T, false, true>(both, M, C, part, false, MlpLinear<T>{{}, static_cast<T*>(a->dx), C, nullptr, 0}, s);
  }
  if (a->dw_gate) {
    const MatSegments up = {{MatOperand{dgate, 2 * Fp * es, 2 * Fp}}, {columns(in.x, C, es)}, {M, 0}, 1};
    mat_linear<T, true, true>(up, Fp + F, C, part, true, MlpTwoRows<T>{{}, {static_cast<T*>(a->dw_gate), static_cast<T*>(a->dw_up)}, F, Fp, C}, s);
  }
  if (a->dw_down) {
    const MatSegments down = {{columns(in.dy, C, es)}, {MatOperand{reinterpret_cast<char*>(h), Fp * es, Fp}}, {M, 0}, 1};
    mat_linear<T, true, true>(down, C, F, part, true, MlpLinear<T>{{}, static_cast<T*>(a->dw_down), F, nullptr, 0}, s);
  }
}

// The partial sums of the backward's products, one after the other.
template <typename T> static int64_t mlp_bwd_part(const fovi_gated_mlp_args* a) {
  const int64_t M = a->rows, C = a->dim, F = a->hidden;
  const int64_t parts[4] = {mlp_keeps(a) ? mat_part_bytes<T>(M, F, C, false) : 0, mat_part_bytes<T>(M, C, F, false),
                            mat_part_bytes<T>(wide(F) + F, C, M, true), mat_part_bytes<T>(C, F, M, true)};
  int64_t most = 0;
  for (int64_t n : parts)
    if (n > most) most = n;
  return most;
}

}  // namespace fovi

using namespace fovi;

extern "C" int64_t fovi_gated_mlp_saved_bytes(int64_t rows, int64_t dim, int64_t hidden, int32_t dtype) {
  return mlp_keeps(dim, dtype) && rows > 0 && hidden > 0 ? rows * 2 * hidden * (dtype == FOVI_F32 ? 4 : 2) : 0;
}

extern "C" int64_t fovi_gated_mlp_fwd_workspace_bytes(const fovi_gated_mlp_args* a) {
  if (!a || a->rows < 1 || a->dim < 1 || a->hidden < 1) return 0;
  const int64_t h = aligned(a->rows * wide(a->hidden) * mlp_element(a));
  if (mlp_few(a)) return h;
  return MlpInputs(a, nullptr, false).in.used() + h +
         (a->dtype == FOVI_F32 ? mat_part_bytes<float>(a->rows, a->dim, a->hidden, false) : mat_part_bytes<uint16_t>(a->rows, a->dim, a->hidden, false));
}

extern "C" int64_t fovi_gated_mlp_bwd_workspace_bytes(const fovi_gated_mlp_args* a) {
  if (!a || a->rows < 1 || a->dim < 1 || a->hidden < 1) return 0;
  const int64_t es = mlp_element(a), rows = a->rows, Fp = wide(a->hidden);
  return MlpInputs(a, nullptr, true).in.used() + aligned(rows * 2 * Fp * es) + aligned(rows * Fp * es) +
         (a->dtype == FOVI_F32 ? mlp_bwd_part<float>(a) : mlp_bwd_part<uint16_t>(a));
}

extern "C" int fovi_gated_mlp_fwd(const fovi_gated_mlp_args* a, void* stream) {
  clear_error();
  if (mlp_check(a, "fovi_gated_mlp_fwd")) return 1;
  if (a->rows == 0) return 0;
  const int64_t need = fovi_gated_mlp_fwd_workspace_bytes(a);
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
  const int64_t need = fovi_gated_mlp_bwd_workspace_bytes(a);
  if (!a->workspace || a->workspace_bytes < need) {
    set_error("fovi_gated_mlp_bwd: workspace of %lld bytes needed", static_cast<long long>(need));
    return 1;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == FOVI_BF16) mlp_bwd<uint16_t>(a, s);
  else mlp_bwd<float>(a, s);
  return check_launch("fovi_gated_mlp_bwd");
}
