// Rotary positions on several axes: pair j of every head of a token turns by positions[axis(j)] * freqs[j].
//
// Memory bound: every element is read and written once. The angles belong to the token, not to the
// head, so a workgroup computes the cosines and sines of its tokens once into LDS and turns all
// heads from there. The product of two floats is exact in fp64; reduced to [-pi, pi] there, the
// angle reaches the sine with fp32 accuracy at any position (an fp32 product at position 10000 is
// already wrong by 5e-4).
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

// N adjacent elements in one access (N * sizeof(T) is 2 to 16 bytes, aligned).
template <typename T, int N> struct alignas(N * sizeof(T)) Run { T e[N]; };

// VEC: elements of an access. Half pairing: a unit is VEC pairs (j .. j + VEC, and n_pairs further on),
// then come units of VEC copied elements; VEC divides n_pairs and head_dim. Adjacent pairing: a unit
// is VEC elements, VEC / 2 pairs, turned or copied; VEC divides head_dim. A thread keeps its unit of a
// token's row and goes from token to token.
template <typename T, int VEC, bool ADJACENT>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p) {
  __shared__ __attribute__((aligned(16))) float2 table[kRotaryTable];
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tokens, all = p.B * p.L;
  const int n = static_cast<int>(all - t0 < p.tokens ? all - t0 : p.tokens);
  for (int i = threadIdx.x; i < n * p.P; i += 256) table[i] = rotary_angle(p, t0 + i / p.P, i % p.P);
  __syncthreads();
  const int per = ADJACENT ? p.D / VEC : (p.D - p.P) / VEC, units = p.H * per, at_once = units < 256 ? 256 / units : 1;
  const int64_t b0 = t0 / p.L, l0 = t0 - b0 * p.L;
  for (int t = threadIdx.x / units; t < n; t += at_once) {
    if (units < 256 && threadIdx.x >= static_cast<unsigned>(units * at_once)) break;
    int64_t b = b0, l = l0 + t;
    if (l >= p.L) { b += l / p.L; l %= p.L; }
    const T* xt = static_cast<const T*>(p.x) + b * p.xs[0] + l * p.xs[1];
    T* yt = static_cast<T*>(p.y) + b * p.ys[0] + l * p.ys[1];
    const float2* turn = table + t * p.P;
    for (int u = units < 256 ? threadIdx.x % units : threadIdx.x; u < units; u += 256) {
      const int h = u / per, j = (u - h * per) * VEC;
      const T* x = xt + h * p.xs[2] + j;
      T* y = yt + h * p.ys[2] + j;
      if (ADJACENT) {
        const Run<T, VEC> a = *reinterpret_cast<const Run<T, VEC>*>(x);
        Run<T, VEC> o = a;
#pragma unroll
        for (int i = 0; i + 1 < VEC; i += 2)
          if (j + i < 2 * p.P) {
            const float2 cs = turn[(j + i) / 2];
            const float u0 = Elem<T>::load(&a.e[i]), v0 = Elem<T>::load(&a.e[i + 1]);
            Elem<T>::store(&o.e[i], u0 * cs.x - v0 * cs.y);
            Elem<T>::store(&o.e[i + 1], v0 * cs.x + u0 * cs.y);
          }
        *reinterpret_cast<Run<T, VEC>*>(y) = o;
      } else if (j >= p.P) {
        *reinterpret_cast<Run<T, VEC>*>(y + p.P) = *reinterpret_cast<const Run<T, VEC>*>(x + p.P);
      } else {
        const Run<T, VEC> a = *reinterpret_cast<const Run<T, VEC>*>(x), c = *reinterpret_cast<const Run<T, VEC>*>(x + p.P);
        Run<T, VEC> ao, co;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float2 cs = turn[j + i];
          const float u0 = Elem<T>::load(&a.e[i]), v0 = Elem<T>::load(&c.e[i]);
          Elem<T>::store(&ao.e[i], u0 * cs.x - v0 * cs.y);
          Elem<T>::store(&co.e[i], v0 * cs.x + u0 * cs.y);
        }
        *reinterpret_cast<Run<T, VEC>*>(y) = ao;
        *reinterpret_cast<Run<T, VEC>*>(y + p.P) = co;
      }
    }
  }
}

// Adjacent pairs of heads of an odd size, or at odd addresses: element by element.
template <typename T>
__global__ __launch_bounds__(256) void rotary_pairs_kernel(RotaryParams p) {
  __shared__ float2 table[kRotaryTable];
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tokens, all = p.B * p.L;
  const int n = static_cast<int>(all - t0 < p.tokens ? all - t0 : p.tokens);
  for (int i = threadIdx.x; i < n * p.P; i += 256) table[i] = rotary_angle(p, t0 + i / p.P, i % p.P);
  __syncthreads();
  const int per = p.D - p.P;                            // a head's pairs, then its copied elements
  for (int i = threadIdx.x; i < n * p.H * per; i += 256) {
    const int t = i / (p.H * per), r = i - t * p.H * per, h = r / per, j = r - h * per;
    const int64_t b = (t0 + t) / p.L, l = t0 + t - b * p.L;
    const T* x = static_cast<const T*>(p.x) + b * p.xs[0] + l * p.xs[1] + h * p.xs[2];
    T* y = static_cast<T*>(p.y) + b * p.ys[0] + l * p.ys[1] + h * p.ys[2];
    if (j >= p.P) {
      y[p.P + j] = x[p.P + j];
      continue;
    }
    const float2 cs = table[t * p.P + j];
    const float u = Elem<T>::load(x + 2 * j), v = Elem<T>::load(x + 2 * j + 1);
    Elem<T>::store(y + 2 * j, u * cs.x - v * cs.y);
    Elem<T>::store(y + 2 * j + 1, v * cs.x + u * cs.y);
  }
}

// Largest access of 2^k elements, up to 16 bytes, that sizes, strides and addresses allow.
static int rotary_vec(const RotaryParams& p, int es) {
  int64_t all = p.D * es;
  if (!p.adjacent) all |= p.P * es;
  for (int i = 0; i < 3; ++i) all |= p.xs[i] * es | p.ys[i] * es;
  all |= static_cast<int64_t>(reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.y));
  int bytes = 16;
  while (all % bytes) bytes /= 2;
  return bytes / es;
}

template <typename T>
static void rotary_launch(const RotaryParams& p, unsigned grid, hipStream_t s) {
  const int vec = rotary_vec(p, sizeof(T));
  if (p.adjacent) {
    if constexpr (sizeof(T) == 2)
      if (vec == 8) { rotary_kernel<T, 8, true><<<grid, 256, 0, s>>>(p); return; }
    if (vec >= 4) rotary_kernel<T, 4, true><<<grid, 256, 0, s>>>(p);
    else if (vec == 2) rotary_kernel<T, 2, true><<<grid, 256, 0, s>>>(p);
    else rotary_pairs_kernel<T><<<grid, 256, 0, s>>>(p);
  } else {
    if constexpr (sizeof(T) == 2)
      if (vec == 8) { rotary_kernel<T, 8, false><<<grid, 256, 0, s>>>(p); return; }
    if (vec >= 4) rotary_kernel<T, 4, false><<<grid, 256, 0, s>>>(p);
    else if (vec == 2) rotary_kernel<T, 2, false><<<grid, 256, 0, s>>>(p);
    else rotary_kernel<T, 1, false><<<grid, 256, 0, s>>>(p);
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
