// Products of a few rows with large weights: serving steps. What counts is the weights' way from memory.
//
// A wave multiplies 16 rows of w (NB matrices, or RB neighbouring blocks of one) by up to TB blocks of 16 rows of x, over its
// share of k, with the 16 x 16 matrix instructions (lane l holds row l % 16, the pieces l / 16 of 64 bytes of k). The waves of
// a workgroup, up to 16, share k; their sums meet in LDS, and the workgroup's threads add them up in order and run
// the epilogue. There are two ways of the operands: rows of whole 16-byte pieces go by 128 bytes a row into a ring of three
// stages in LDS that each wave has for itself (no barriers, whole cache lines); others straight into the instructions'
// registers, several steps of loads at a time, at any start and stride (the last, partial piece of a row is put
// together with care). A register load touches half a line of 16 rows and costs as much as whole ones: 32 x 2048 by 2 x 5504
// in bf16 takes 13.0 us the first way (45 MB, 3.5 TB/s) and took 20.6 the second, 48 x 4096 by 11008 in int8 12.7 (45 MB) and 22.4;
// rows that start an element off whole pieces, which only the second takes, 53 and 72.
#pragma once

#include <type_traits>

#include "matmul.h"

namespace fovi {

typedef int32_t i32x4s __attribute__((ext_vector_type(4)));

template <typename T> struct Few;
template <> struct Few<uint16_t> { typedef f32x4 Acc; };
template <> struct Few<float> { typedef f32x4 Acc; };
template <> struct Few<int8_t> { typedef i32x4s Acc; };

__device__ __forceinline__ f32x4 few_step(uint16_t, u32x4 w, u32x4 x, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 few_step(float, u32x4 w, u32x4 x, f32x4 c) {
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.x), __uint_as_float(x.x), c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.y), __uint_as_float(x.y), c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.z), __uint_as_float(x.z), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.w), __uint_as_float(x.w), c, 0, 0, 0);
}
__device__ __forceinline__ i32x4s few_step(int8_t, u32x4 w, u32x4 x, i32x4s c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, w), __builtin_bit_cast(i32x4, x), c, 0, 0, 0);
}

// acc += the products of COUNT steps. fp32 sums are taken by such groups (of up to 128 products) and added up, as the tiles take
// them by stages. In one chain for a wave's share of k, outputs of 32 x 2048 by 5504 were 7.8e-7 off (the norm of the difference
// over the norm), 2.5e-7 so, at the same speed within 1 %.
template <typename T, int COUNT, int NW, int TB>
__device__ __forceinline__ void few_multiply(const u32x4 (&w)[COUNT][NW], const u32x4 (&x)[COUNT][TB], typename Few<T>::Acc (&acc)[NW][TB]) {
  typedef typename Few<T>::Acc Acc;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      Acc part[TB];
#pragma unroll
      for (int t = 0; t < TB; ++t) part[t] = Acc{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < COUNT; ++s)
#pragma unroll
        for (int t = 0; t < TB; ++t) part[t] = few_step(T(), w[s][i], x[s][t], part[t]);
#pragma unroll
      for (int t = 0; t < TB; ++t) acc[i][t] += part[t];
    }
  } else {
#pragma unroll
    for (int s = 0; s < COUNT; ++s)
#pragma unroll
      for (int i = 0; i < NW; ++i)
#pragma unroll
        for (int t = 0; t < TB; ++t) acc[i][t] = few_step(T(), w[s][i], x[s][t], acc[i][t]);
  }
}

constexpr int kFewRow = 20;                            // words of a row of 16 sums in LDS: rows begin in different banks
template <int NB, int RB, int TB> constexpr int few_lds(int waves) { return waves * NB * RB * TB * 16 * kFewRow * 4; }

// The waves' sums added up, through the epilogue.
template <typename T, int NB, int RB, int TB, typename Epilogue>
__device__ __forceinline__ void few_finish(char* memory, const typename Few<T>::Acc (&acc)[NB * RB][TB], int m0, int64_t n0, int M, int64_t N,
                                           const Epilogue& epilogue) {
  typedef typename Few<T>::Acc Acc;
  typedef typename Mat<T>::Sum Sum;
  constexpr int NW = NB * RB;
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6, l = threadIdx.x & 63;
  Sum* sums = reinterpret_cast<Sum*>(memory);
#pragma unroll
  for (int i = 0; i < NW; ++i)
#pragma unroll
    for (int t = 0; t < TB; ++t)
      *reinterpret_cast<Acc*>(sums + ((wave * NW + i) * TB * 16 + 16 * t + (l & 15)) * kFewRow + 4 * (l >> 4)) = acc[i][t];
  __syncthreads();
  for (int id = threadIdx.x; id < TB * 32 * RB; id += blockDim.x) {
    const int m = id / (2 * RB), r = id % (2 * RB);
    const int64_t n = n0 + 8 * r;
    if (m0 + m >= M || n >= N) continue;
    const int count = static_cast<int>(N - n < 8 ? N - n : 8);
    const typename Epilogue::Column column = epilogue.column(n, count);
    const typename Epilogue::Extra extra = epilogue.load(m0 + m, n, count);
    Sum v[NB][8];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[b][e] = 0;
      for (int z = 0; z < waves; ++z) {
        const Sum* p = sums + ((z * NW + b * RB + r / 2) * TB * 16 + m) * kFewRow + 8 * (r & 1);
        const Acc lo = *reinterpret_cast<const Acc*>(p), hi = *reinterpret_cast<const Acc*>(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[b][e] += lo[e]; v[b][4 + e] += hi[e]; }
      }
    }
    epilogue(m0 + m, n, count, v, column, extra);
  }
}

template <typename T, int NB, int RB, int TB, typename Epilogue>
__global__ __launch_bounds__(1024) void few_kernel(MatOperand x, MatOperand w0, MatOperand w1, int64_t K, int M, int64_t N, Epilogue epilogue) {
  typedef typename Few<T>::Acc Acc;
  typedef typename Mat<T>::Sum Sum;
  constexpr int NW = NB * RB, U = NW + TB <= 3 ? 8 : NW + TB <= 4 ? 6 : 4;
  extern __shared__ __attribute__((aligned(16))) char few_memory[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, l = threadIdx.x & 63;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * RB), bytes = K * static_cast<int64_t>(sizeof(T));
  const int m0 = blockIdx.y * (16 * TB);
  const char* pw[NW];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      const int64_t n = n0 + 16 * r + (l & 15);
      const MatOperand& w = b ? w1 : w0;
      pw[b * RB + r] = w.p + (n < N ? n : N - 1) * w.stride;
    }
  const char* px[TB];
#pragma unroll
  for (int t = 0; t < TB; ++t) {
    const int m = m0 + 16 * t + (l & 15);
    px[t] = x.p + (m < M ? m : M - 1) * x.stride;
  }
  Acc acc[NW][TB];
#pragma unroll
  for (int i = 0; i < NW; ++i)
#pragma unroll
    for (int t = 0; t < TB; ++t) acc[i][t] = Acc{0, 0, 0, 0};
  auto steps = [&](int64_t at, auto n, const auto& load) __attribute__((always_inline)) {
    constexpr int COUNT = decltype(n)::value;
    u32x4 fw[COUNT][NW], fx[COUNT][TB];
#pragma unroll
    for (int s = 0; s < COUNT; ++s) {
#pragma unroll
      for (int i = 0; i < NW; ++i) fw[s][i] = load(pw[i], at + 64 * s + 16 * (l >> 4));
#pragma unroll
      for (int t = 0; t < TB; ++t) fx[s][t] = load(px[t], at + 64 * s + 16 * (l >> 4));
    }
    few_multiply<T>(fw, fx, acc);
  };
  auto whole = [](const char* p, int64_t at) __attribute__((always_inline)) {
    u32x4 u;
    __builtin_memcpy(&u, p + at, 16);
    return u;
  };
  // whole steps of 64 bytes in equal shares, the partial one behind them for the last wave
  const int64_t all = bytes / 64, from = all * wave / waves, to = all * (wave + 1) / waves;
  int64_t s = from;
  for (; s + U <= to; s += U) steps(s * 64, std::integral_constant<int, U>(), whole);
  for (; s + 2 <= to; s += 2) steps(s * 64, std::integral_constant<int, 2>(), whole);
  if (s < to) steps(s * 64, std::integral_constant<int, 1>(), whole);
  if (wave == waves - 1 && all * 64 < bytes)
    steps(all * 64, std::integral_constant<int, 1>(), [&](const char* p, int64_t at) __attribute__((always_inline)) { return mat_piece(p, at, bytes); });

  few_finish<T, NB, RB, TB>(few_memory, acc, m0, n0, M, N, epilogue);
}

// The same by way of LDS.
template <typename T, int NB, int RB, int TB> struct FewRing {
  typedef MatLoader<T, 16 * RB, false, 1> LW;
  typedef MatLoader<T, 16 * TB, false, 1> LX;
  static constexpr int W = 16 * RB * 128, X = 16 * TB * 128, BYTES = NB * W + X, LOADS = BYTES / 1024, LDS = 3 * BYTES;
};
template <typename T, int NB, int RB, int TB, typename Epilogue>
__global__ __launch_bounds__(1024) void few_ring_kernel(MatOperand x, MatOperand w0, MatOperand w1, int64_t K, int M, int64_t N,
                                                        Epilogue epilogue) {
  typedef typename Few<T>::Acc Acc;
  typedef FewRing<T, NB, RB, TB> Ring;
  constexpr int NW = NB * RB, BK = mat_bk<T>(), LOADS = Ring::LOADS;
  extern __shared__ __attribute__((aligned(1024))) char few_ring_memory[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, l = threadIdx.x & 63;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * RB);
  const int m0 = blockIdx.y * (16 * TB);
  char* mine = few_ring_memory + wave * Ring::LDS;
  Acc acc[NW][TB];
#pragma unroll
  for (int i = 0; i < NW; ++i)
#pragma unroll
    for (int t = 0; t < TB; ++t) acc[i][t] = Acc{0, 0, 0, 0};
  const int64_t all = (K + BK - 1) / BK, from = all * wave / waves, to = all * (wave + 1) / waves;
  typename Ring::LW lw[NB];
  typename Ring::LX lx;
  lw[0].open(w0, n0, from * BK);
  if (NB == 2) lw[NB - 1].open(w1, n0, from * BK);
  lx.open(x, m0, from * BK);
  int64_t started = from;
  auto start = [&](int slot) __attribute__((always_inline)) {
    const uint32_t at = lds_address(mine) + slot * Ring::BYTES;
    const int64_t left = K - started * BK;
#pragma unroll
    for (int b = 0; b < NB; ++b) lw[b].start(at + b * Ring::W, left);
    lx.start(at + NB * Ring::W, left);
    ++started;
  };
  for (int i = 0; i < 3; ++i)
    if (started < to) start(i);
  int slot = 0;
  for (int64_t t = from; t < to; ++t) {
    // the stage's loads have landed when no more than those of the stages behind it are outstanding
    const int64_t behind = started - t - 1;
    if (behind == 2) asm volatile("s_waitcnt vmcnt(%0)" :: "n"(2 * LOADS) : "memory");
    else if (behind == 1) asm volatile("s_waitcnt vmcnt(%0)" :: "n"(LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const char* now = mine + slot * Ring::BYTES;
    u32x4 fw[2][NW], fx[2][TB];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < NW; ++i)
        fw[s][i] = *reinterpret_cast<const u32x4*>(now + (i / RB) * Ring::W + Ring::LW::Tile::at((i % RB) * 16 + (l & 15), 4 * s + (l >> 4)));
#pragma unroll
      for (int k = 0; k < TB; ++k) fx[s][k] = *reinterpret_cast<const u32x4*>(now + NB * Ring::W + Ring::LX::Tile::at(16 * k + (l & 15), 4 * s + (l >> 4)));
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");           // read: the place is free
    __builtin_amdgcn_sched_barrier(0);
    if (started < to) start(slot);
    slot = slot == 2 ? 0 : slot + 1;
    few_multiply<T>(fw, fx, acc);
  }
  __syncthreads();                                               // the sums take the stages' place
  few_finish<T, NB, RB, TB>(few_ring_memory, acc, m0, n0, M, N, epilogue);
}

// Up to 64 rows go here, and up to 256 where tiles of 64 x 64 would leave compute units without work: fewer tiles than compute
// units, or half as many where a tile has more to do (fp32, two products in int8). Here and by tiles, us: int8 4096 x 1024,
// 128 rows 5.1 and 10.3, 256 rows 6.5 and 11.5; int8 1024 x 4096, 128 rows 4.7 and 6.6, 192 rows two products 10.6 and 7.6;
// the block of 384 x 1024, 128 rows, bf16 7.7 and 15.1, fp32 12.7 and 32.6, of 2048 x 5504, bf16 33.9 and 40.1, fp32 151 and
// 128; int8 4096 x 11008 (344 tiles), 128 rows, 23.8 and 20.8.
inline bool few_rows_best(int64_t M, int64_t N, bool heavy) {
  return M <= 64 || (M <= 256 && (M + 63) / 64 * ((N + 63) / 64) <= (heavy ? 128 : 255));
}

// Waves of a workgroup: four steps of 64 bytes for each, but no more than give the card 4096 waves (as many as are resident
// at a time), nor fewer than four.
inline int few_waves(int64_t groups, int64_t bytes) {
  int64_t waves = (bytes + 255) / 256;
  const int64_t most = 4096 / groups > 4 ? 4096 / groups : 4;
  if (waves > most) waves = most;
  return static_cast<int>(waves < 1 ? 1 : waves > 16 ? 16 : waves);
}

template <typename T, int NB, int RB, int TB, typename Epilogue>
static void few_launch(const MatOperand& x, const MatOperand& w0, const MatOperand& w1, int64_t K, int64_t M, int64_t N,
                       const Epilogue& epilogue, hipStream_t s) {
  const int64_t across = (N + 16 * RB - 1) / (16 * RB);
  const dim3 groups(static_cast<unsigned>(across), static_cast<unsigned>((M + 16 * TB - 1) / (16 * TB)));
  const int64_t all = across * groups.y;
  if (mat_whole<T>(x, K) && mat_whole<T>(w0, K) && mat_whole<T>(w1, K)) {
    // as many waves as LDS holds (two workgroups a compute unit where there are that many), each with two stages or more
    constexpr int each = FewRing<T, NB, RB, TB>::LDS > few_lds<NB, RB, TB>(1) ? FewRing<T, NB, RB, TB>::LDS : few_lds<NB, RB, TB>(1);
    const int64_t most = (all > 256 ? 81920 : 163840) / each, want = (K + 2 * mat_bk<T>() - 1) / (2 * mat_bk<T>());
    const int w = static_cast<int>(want < most ? want : most < 16 ? most : 16);
    if (!launch_fits(across, 64 * w)) return;
    mat_launch(few_ring_kernel<T, NB, RB, TB, Epilogue>, groups, 64 * w, w * each, s, x, w0, w1, K, static_cast<int>(M), N, epilogue);
    return;
  }
  const int most = 65536 / few_lds<NB, RB, TB>(1), waves = few_waves(all, K * static_cast<int64_t>(sizeof(T)));
  const int w = waves < most ? waves : most;
  if (!launch_fits(across, 64 * w)) return;
  few_kernel<T, NB, RB, TB, Epilogue><<<groups, 64 * w, few_lds<NB, RB, TB>(w), s>>>(x, w0, w1, K, static_cast<int>(M), N, epilogue);
}

// The blocks of w and of x of a workgroup: those with which a compute unit reads least in its rounds of workgroups; on a tie
// fewer parts of x, since each reads w again. (32 rows of 5504 by 2048 in bf16: 128 workgroups take 8.7 us, and 7.7 with the rows
// in two parts.)
template <typename T, int NB, int RB, typename Epilogue>
static void few_rows(int tb, const MatOperand& x, const MatOperand& w0, const MatOperand& w1, int64_t K, int64_t M, int64_t N,
                     const Epilogue& epilogue, hipStream_t s) {
  if (tb == 1) few_launch<T, NB, RB, 1>(x, w0, w1, K, M, N, epilogue, s);
  else if (tb == 2) few_launch<T, NB, RB, 2>(x, w0, w1, K, M, N, epilogue, s);
  else if (tb == 3) few_launch<T, NB, RB, 3>(x, w0, w1, K, M, N, epilogue, s);
  else few_launch<T, NB, RB, 4>(x, w0, w1, K, M, N, epilogue, s);
}
template <typename T, int NB, typename Epilogue>
static void few_product(const MatOperand& x, const MatOperand& w0, const MatOperand& w1, int64_t K, int64_t M, int64_t N,
                        const Epilogue& epilogue, hipStream_t s) {
  const int blocks = static_cast<int>((M + 15) / 16);
  int64_t best = 0;
  int best_rb = 0, best_tb = 0;
  for (int rb = 1; rb <= 3 - NB; ++rb)
    for (int parts = (blocks + 3) / 4; parts <= blocks; ++parts) {
      const int tb = (blocks + parts - 1) / parts;
      const int64_t rounds = ((N + 16 * rb - 1) / (16 * rb) * parts + 255) / 256, cost = rounds * (rb * NB + tb);
      if (!best_rb || cost < best) { best = cost; best_rb = rb; best_tb = tb; }
    }
  if (best_rb == 2) few_rows<T, NB, 3 - NB>(best_tb, x, w0, w1, K, M, N, epilogue, s);
  else few_rows<T, NB, 1>(best_tb, x, w0, w1, K, M, N, epilogue, s);
}

}  // namespace fovi
