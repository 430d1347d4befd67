// Rotary positions on several axes: pair j of every head of a token turns by positions[axis(j)] * freqs[j].
//
// Memory bound: every element is read and written once. The angles belong to the token, not to the
// head, so a workgroup computes the cosines and sines of its tokens once into LDS and turns all
// heads from there. The product of two floats is exact in fp64; reduced to [-pi, pi] there, the
// angle reaches the sine with fp32 accuracy at any position (an fp32 product at position 10000 is
// already wrong by 5e-4). 131072 tokens of 6 bf16 heads of 64: 46 us (201 MB, 4.4 TB/s).
#include "common.h"

namespace fovi {

struct RotaryParams {
  const void* x; void* y;
  const float* pos; const float* freqs;
  int64_t B, L;
  int H, D, P, n_axes, adjacent, inverse;
  int end[FOVI_ROTARY_MAX_AXES];
  int64_t xs[3], ys[3], ps[2];
  int tokens;                 // a workgroup's
};

constexpr int kRotaryTable = 2048;   // (cos, sin) pairs of a workgroup: 16 KB

__device__ __forceinline__ float2 rotary_angle(const RotaryParams& p, int64_t token, int j) {
  int axis = 0;
  while (axis + 1 < p.n_axes && j >= p.end[axis]) ++axis;
  const int64_t b = token / p.L, l = token - b * p.L;
  const double angle = static_cast<double>(p.pos[b * p.ps[0] + l * p.ps[1] + axis]) * static_cast<double>(p.freqs[j]);
  const double turns = angle * 0.15915494309189533577;
  const float r = static_cast<float>((turns - rint(turns)) * 6.28318530717958647693);
  float s, c;
  sincosf(r, &s, &c);
  return make_float2(c, p.inverse ? -s : s);
}

// Runs of 16 bytes (N elements, any alignment): whole, or with SHORT the first n elements.
template <typename T, int N, bool SHORT>
__device__ __forceinline__ void load_run(const T* p, int n, T (&e)[N]) {
  u32x4 u = {0, 0, 0, 0};
  if (!SHORT || n >= N) __builtin_memcpy(&u, p, 16);
  __builtin_memcpy(e, &u, 16);
  if (SHORT && n < N) {
#pragma unroll
    for (int i = 0; i < N - 1; ++i)
      if (i < n) e[i] = p[i];
  }
}
template <typename T, int N, bool SHORT>
__device__ __forceinline__ void save_run(T* p, int n, const T (&e)[N]) {
  if (!SHORT || n >= N) {
    u32x4 u;
    __builtin_memcpy(&u, e, 16);
    __builtin_memcpy(p, &u, 16);
  } else {
#pragma unroll
    for (int i = 0; i < N - 1; ++i)
      if (i < n) p[i] = e[i];
  }
}

// Half pairing: a unit is VEC pairs (j .. j + VEC, and n_pairs further on), then come units of VEC copied
// elements. Adjacent pairing: a unit is VEC elements, VEC / 2 pairs, turned or copied. A thread keeps its
// unit of a token's row and goes from token to token. ODD: the units do not divide those runs; the last one
// of a run starts VEC before its end, beside elements that the unit before writes as well (the same values),
// or is short where the run is, or where an odd head would split its pairs.
template <typename T, bool ADJACENT, bool ODD>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ __attribute__((aligned(16))) float2 table[kRotaryTable];
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tokens, all = p.B * p.L;
  const int n = static_cast<int>(all - t0 < p.tokens ? all - t0 : p.tokens);
  for (int i = threadIdx.x; i < n * p.P; i += 256) table[i] = rotary_angle(p, t0 + i / p.P, i % p.P);
  __syncthreads();
  const int turned = (p.P + VEC - 1) / VEC, rest = p.D - 2 * p.P;
  const int per = ADJACENT ? (p.D + VEC - 1) / VEC : turned + (rest + VEC - 1) / VEC, units = p.H * per;
  const int at_once = units < 256 ? 256 / units : 1;
  const int64_t b0 = t0 / p.L, l0 = t0 - b0 * p.L;
  for (int t = threadIdx.x / units; t < n; t += at_once) {
    if (units < 256 && threadIdx.x >= static_cast<unsigned>(units * at_once)) break;
    int64_t b = b0, l = l0 + t;
    if (l >= p.L) { b += l / p.L; l %= p.L; }
    const T* xt = static_cast<const T*>(p.x) + b * p.xs[0] + l * p.xs[1];
    T* yt = static_cast<T*>(p.y) + b * p.ys[0] + l * p.ys[1];
    const float2* turn = table + t * p.P;
    for (int u = units < 256 ? threadIdx.x % units : threadIdx.x; u < units; u += 256) {
      const int h = u / per, r = u - h * per;
      int j = r * VEC;
      if (ADJACENT) {
        if (ODD && j + VEC > p.D && p.D >= VEC && p.D % 2 == 0) j = p.D - VEC;
        const T* x = xt + h * p.xs[2] + j;
        T* y = yt + h * p.ys[2] + j;
        T a[VEC], o[VEC];
        load_run<T, VEC, ODD>(x, p.D - j, a);
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
          o[i] = a[i];
          o[i + 1] = a[i + 1];
          if (j + i < 2 * p.P) {
            const float2 cs = turn[(j + i) / 2];
            const float u0 = Elem<T>::load(&a[i]), v0 = Elem<T>::load(&a[i + 1]);
            Elem<T>::store(&o[i], u0 * cs.x - v0 * cs.y);
            Elem<T>::store(&o[i + 1], v0 * cs.x + u0 * cs.y);
          }
        }
        save_run<T, VEC, ODD>(y, p.D - j, o);
        continue;
      }
      const bool copied = r >= turned;
      if (ODD) {
        if (copied) j -= turned * VEC - p.P;
        const int run = copied ? rest : p.P, end = copied ? p.D - p.P : p.P;
        if (j + VEC > end && run >= VEC) j = end - VEC;
      }
      const T* x = xt + h * p.xs[2] + j;
      T* y = yt + h * p.ys[2] + j;
      if (copied) {
        T c[VEC];
        load_run<T, VEC, ODD>(x + p.P, p.D - p.P - j, c);
        save_run<T, VEC, ODD>(y + p.P, p.D - p.P - j, c);
      } else {
        T a[VEC], c[VEC], ao[VEC], co[VEC];
        load_run<T, VEC, ODD>(x, p.P - j, a);
        load_run<T, VEC, ODD>(x + p.P, p.P - j, c);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float2 cs = turn[!ODD || j + i < p.P ? j + i : p.P - 1];
          const float u0 = Elem<T>::load(&a[i]), v0 = Elem<T>::load(&c[i]);
          Elem<T>::store(&ao[i], u0 * cs.x - v0 * cs.y);
          Elem<T>::store(&co[i], v0 * cs.x + u0 * cs.y);
        }
        save_run<T, VEC, ODD>(y, p.P - j, ao);
        save_run<T, VEC, ODD>(y + p.P, p.P - j, co);
      }
    }
  }
}

template <typename T>
static void rotary_launch(const RotaryParams& p, unsigned grid, hipStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  if (p.adjacent) {
    if (p.D % VEC) rotary_kernel<T, true, true><<<grid, 256, 0, s>>>(p);
    else rotary_kernel<T, true, false><<<grid, 256, 0, s>>>(p);
  } else {
    if (p.P % VEC || p.D % VEC) rotary_kernel<T, false, true><<<grid, 256, 0, s>>>(p);
    else rotary_kernel<T, false, false><<<grid, 256, 0, s>>>(p);
  }
}

}  // namespace fovi

using namespace fovi;

extern "C" int fovi_rotary(const fovi_rotary_args* a, void* stream) {
  clear_error();
  if (!a || !a->x || !a->y || !a->positions || !a->freqs) { set_error("fovi_rotary: null pointer"); return 1; }
  if (a->dtype != FOVI_F32 && a->dtype != FOVI_BF16) { set_error("fovi_rotary: dtype must be F32 or BF16"); return 1; }
  if (a->pairing != FOVI_PAIR_HALF && a->pairing != FOVI_PAIR_ADJACENT) { set_error("fovi_rotary: unknown pairing"); return 1; }
  if (a->n_axes < 1 || a->n_axes > FOVI_ROTARY_MAX_AXES) {
    set_error("fovi_rotary: 1 to %d axes", FOVI_ROTARY_MAX_AXES);
    return 1;
  }
  int last = 0;
  for (int i = 0; i < a->n_axes; ++i) {
    if (a->section_end[i] < last) { set_error("fovi_rotary: section_end must not decrease"); return 1; }
    last = a->section_end[i];
  }
  if (a->batch < 0 || a->length < 0 || a->heads < 0 || a->head_dim < 1 || last < 1 || 2 * static_cast<int64_t>(last) > a->head_dim) {
    set_error("fovi_rotary: bad sizes (1 <= pairs <= head_dim / 2)");
    return 1;
  }
  if (last > kRotaryTable || a->heads * a->head_dim > (1 << 28)) { set_error("fovi_rotary: heads too large"); return 1; }
  const int64_t tokens = a->batch * a->length;
  if (tokens == 0 || a->heads == 0) return 0;
  RotaryParams p;
  p.x = a->x; p.y = a->y; p.pos = a->positions; p.freqs = a->freqs;
  p.B = a->batch; p.L = a->length; p.H = static_cast<int>(a->heads); p.D = static_cast<int>(a->head_dim);
  p.P = last; p.n_axes = a->n_axes; p.adjacent = a->pairing == FOVI_PAIR_ADJACENT; p.inverse = a->inverse != 0;
  for (int i = 0; i < FOVI_ROTARY_MAX_AXES; ++i) p.end[i] = i < a->n_axes ? a->section_end[i] : last;
  for (int i = 0; i < 3; ++i) { p.xs[i] = a->x_stride[i]; p.ys[i] = a->y_stride[i]; }
  p.ps[0] = a->pos_stride[0]; p.ps[1] = a->pos_stride[1];
  // enough tokens for 16 elements a thread, but no fewer than 512 workgroups
  int64_t per = (4096 + a->heads * a->head_dim - 1) / (a->heads * a->head_dim);
  if (per > tokens / 512) per = tokens / 512;
  if (per > kRotaryTable / p.P) per = kRotaryTable / p.P;
  if (per < 1) per = 1;
  p.tokens = static_cast<int>(per);
  const int64_t grid = (tokens + per - 1) / per;
  if (grid > 0x7fffffff) { set_error("fovi_rotary: too many tokens"); return 1; }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == FOVI_BF16) rotary_launch<uint16_t>(p, static_cast<unsigned>(grid), s);
  else rotary_launch<float>(p, static_cast<unsigned>(grid), s);
  return check_launch("fovi_rotary");
}
