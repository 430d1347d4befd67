// Matrix products on the matrix unit for the feed-forward operators: fp32, bf16 and int8, with either operand's
// reduction axis contiguous ("rows") or strided ("columns"), several products of the same left operand at once, and
// the caller's own work on the sums (an epilogue) before they are written.
//
// out[m, n] = sum_k x[m, k] w[n, k]. A workgroup of four waves owns a tile of BM x BN and walks k in steps of 128 bytes a row
// (64 bf16, 128 int8, 32 fp32 elements). Tiles lie in LDS in 16-byte pieces that are swapped within a row
// (XOR) so that the lanes of a read spread over the banks. The matrix instruction takes w as its first operand:
// a lane then holds one row m and runs of four adjacent n of its sums, which are written as they are.
#pragma once

#include "common.h"

namespace fovi {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// One operand: element (r, k) at p + r * stride + k * size where k is contiguous, else p + k * stride + r * size.
// stride in bytes; `extent` rows r.
struct MatOperand {
  const char* p;
  int64_t stride, extent;
};

template <typename T> struct Mat;
template <> struct Mat<uint16_t> { typedef f32x16 Acc; typedef float Sum; static constexpr int BK = 64; };
template <> struct Mat<float> { typedef f32x16 Acc; typedef float Sum; static constexpr int BK = 32; };
template <> struct Mat<int8_t> { typedef i32x16 Acc; typedef int32_t Sum; static constexpr int BK = 128; };

// One step of a product: 16 bytes of 32 rows of either operand; lanes 0 .. 31 hold one piece of k, 32 .. 63 the next.
__device__ __forceinline__ f32x16 mat_step(uint16_t, u32x4 w, u32x4 x, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mat_step(float, u32x4 w, u32x4 x, f32x16 c) {
  c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(w.x), __uint_as_float(x.x), c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(w.y), __uint_as_float(x.y), c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(w.z), __uint_as_float(x.z), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(w.w), __uint_as_float(x.w), c, 0, 0, 0);
}
__device__ __forceinline__ i32x16 mat_step(int8_t, u32x4 w, u32x4 x, i32x16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, w), __builtin_bit_cast(i32x4, x), c, 0, 0, 0);
}

// 16 bytes of a run of `len` bytes from `at` on, at any alignment, zeros from its end on.
__device__ __forceinline__ u32x4 mat_piece(const char* run, int64_t at, int64_t len) {
  u32x4 u = {0, 0, 0, 0};
  if (at + 16 <= len) {
    __builtin_memcpy(&u, run + at, 16);
  } else if (at < len && len >= 16) {                  // the run's last 16 bytes, shifted down
    uint64_t w[2];
    __builtin_memcpy(w, run + len - 16, 16);
    const int over = static_cast<int>(at + 16 - len) * 8, bits = over & 63;
    if (over >= 64) { w[0] = w[1]; w[1] = 0; }
    w[0] = (w[0] >> bits) | (w[1] << 1 << (63 - bits));
    w[1] >>= bits;
    __builtin_memcpy(&u, w, 16);
  } else if (at < len) {                               // a run of fewer than 16 bytes: at is 0
    uint64_t w[2] = {0, 0};
    for (int64_t i = 0; i < len; ++i) w[i >> 3] |= static_cast<uint64_t>(static_cast<uint8_t>(run[i])) << ((i & 7) * 8);
    __builtin_memcpy(&u, w, 16);
  }
  return u;
}

// The tile of an operand in LDS: NR rows of 128 bytes of k, or (COL) BK rows of NR elements.
template <typename T, int NR, bool COL> struct MatTile {
  static constexpr int ES = sizeof(T);
  static constexpr int BYTES = NR * 128;
  static constexpr int PIECES = COL ? NR * ES / 16 : 8;          // 16-byte pieces of an LDS row
  static constexpr int PER = NR * 8 / 256;                       // pieces a thread loads

  static __device__ __forceinline__ int at(int r, int piece) {
    int s;
    if (!COL) s = (r >> 1) & 7;
    else s = (ES == 2 ? (r & 3) << 2 : ((r >> 2) & 1) << 3) & (PIECES - 1);
    return r * PIECES * 16 + ((piece ^ s) << 4);
  }

  u32x4 v[PER];
  // The tile of rows r0 .., elements k0 .. of k; rows behind the last are the last row again (their sums are not
  // written), elements behind k_end zeros.
  __device__ __forceinline__ void load(const MatOperand& o, int64_t r0, int64_t k0, int64_t k_end) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int id = threadIdx.x + 256 * i, a = id / PIECES, b = id % PIECES;
      if (!COL) {
        const int64_t r = r0 + a < o.extent ? r0 + a : o.extent - 1;
        v[i] = mat_piece(o.p + r * o.stride, k0 * ES + b * 16, k_end * ES);
      } else {
        const int64_t k = k0 + a;
        v[i] = k < k_end ? mat_piece(o.p + k * o.stride, r0 * ES + b * 16, o.extent * ES) : u32x4{0, 0, 0, 0};
      }
    }
  }
  __device__ __forceinline__ void put(char* lds) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int id = threadIdx.x + 256 * i;
      *reinterpret_cast<u32x4*>(lds + at(id / PIECES, id % PIECES)) = v[i];
    }
  }
  // Step s (of 4) of the 32 rows from r on.
  static __device__ __forceinline__ u32x4 read(const char* lds, int r, int s) {
    const int l = threadIdx.x & 63;
    if (!COL) return *reinterpret_cast<const u32x4*>(lds + at(r + (l & 31), 2 * s + (l >> 5)));
    if (ES == 2) {
      // Within 16 lanes, lane j addresses four elements of k row j / 4; lane i receives element i of the four rows.
      const int k = 16 * s + 8 * (l >> 5) + ((l & 15) >> 2), c = (r >> 3) + 2 * ((l >> 4) & 1) + ((l & 3) >> 1);
      const char* p = lds + (l & 1) * 8;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + at(k, c)));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + at(k + 4, c)));
      return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    u32x4 u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = 4 * (2 * s + (l >> 5)) + i, c = r + (l & 31);
      u[i] = *reinterpret_cast<const uint32_t*>(lds + at(k, c >> 2) + (c & 3) * 4);
    }
    return u;
  }
};

// acc[b] += the products over k_begin .. k_end of the tile's rows of x and of w[b], b < NB. Every wave holds BM / 64 x
// BN / 64 blocks of 32 x 32 of each.
template <typename T, int BM, int BN, int NB, bool CX, bool CW>
struct MatCore {
  typedef typename Mat<T>::Acc Acc;
  typedef MatTile<T, BM, CX> TX;
  typedef MatTile<T, BN, CW> TW;
  static constexpr int MB = BM / 64, NN = BN / 64, BK = Mat<T>::BK;
  static constexpr int LDS = TX::BYTES + NB * TW::BYTES;

  template <int NA>
  static __device__ __forceinline__ void run(const MatOperand& x, const MatOperand* w, int64_t m0, int64_t n0, int64_t k_begin,
                                             int64_t k_end, char* lds, Acc (&acc)[NA][MB][NN], int first = 0) {
    const int wave = threadIdx.x >> 6, wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
    TX tx;
    TW tw[NB];
    auto load = [&](int64_t k) {
      tx.load(x, m0, k, k_end);
#pragma unroll
      for (int b = 0; b < NB; ++b) tw[b].load(w[b], n0, k, k_end);
    };
    load(k_begin);
    for (int64_t k = k_begin; k < k_end; k += BK) {
      __syncthreads();
      tx.put(lds);
#pragma unroll
      for (int b = 0; b < NB; ++b) tw[b].put(lds + TX::BYTES + b * TW::BYTES);
      __syncthreads();
      if (k + BK < k_end) load(k + BK);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        u32x4 fx[MB], fw[NB][NN];
#pragma unroll
        for (int i = 0; i < MB; ++i) fx[i] = TX::read(lds, wm + 32 * i, s);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int j = 0; j < NN; ++j) fw[b][j] = TW::read(lds + TX::BYTES + b * TW::BYTES, wn + 32 * j, s);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NN; ++j) acc[first + b][i][j] = mat_step(T(), fw[b][j], fx[i], acc[first + b][i][j]);
      }
    }
  }
};

template <typename Acc, int NA, int MB, int NN>
__device__ __forceinline__ void mat_clear(Acc (&acc)[NA][MB][NN]) {
#pragma unroll
  for (int b = 0; b < NA; ++b)
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[b][i][j][r] = 0;
}

// epilogue(m, n, count, v): the sums v[b][0 .. count) of row m from column n on, in runs of four.
template <int BM, int BN, typename Sum, typename Acc, int NA, int MB, int NN, typename Epilogue>
__device__ __forceinline__ void mat_finish(const Acc (&acc)[NA][MB][NN], int64_t m0, int64_t n0, int64_t M, int64_t N,
                                           const Epilogue& epilogue) {
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int64_t m = m0 + (wave >> 1) * (BM / 2) + 32 * i + (l & 31);
    if (m >= M) continue;
#pragma unroll
    for (int j = 0; j < NN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t n = n0 + (wave & 1) * (BN / 2) + 32 * j + 8 * q + 4 * (l >> 5);
        if (n >= N) continue;
        Sum v[NA][4];
#pragma unroll
        for (int b = 0; b < NA; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[b][e] = acc[b][i][j][4 * q + e];
        epilogue(m, n, static_cast<int>(N - n < 4 ? N - n : 4), v);
      }
  }
}

// Four (or `count`) adjacent elements as floats, and back.
template <typename T> __device__ __forceinline__ void load_four(const T* p, int count, float (&v)[4]) {
  T e[4];
  if (count == 4) {
    __builtin_memcpy(e, p, sizeof(e));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = i < count ? p[i] : T(0);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = Elem<T>::load(e + i);
}
template <typename T> __device__ __forceinline__ void store_four(T* p, int count, const float (&v)[4]) {
  T e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) Elem<T>::store(e + i, v[i]);
  if (count == 4) {
    __builtin_memcpy(p, e, sizeof(e));
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < count) p[i] = e[i];
  }
}

// Activations and their derivatives. EXACT: the library's exponential and division, for fp32 operands.
template <bool EXACT> __device__ __forceinline__ float mat_sigmoid(float z) {
  if (EXACT) return 1.0f / (1.0f + expf(-z));
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896340736f));
}
template <bool EXACT> __device__ __forceinline__ float mat_act(float z, int act) {
  if (act == FOVI_GATE_SILU) return EXACT ? z / (1.0f + expf(-z)) : z * mat_sigmoid<false>(z);
  return 0.5f * z * (1.0f + erff(z * 0.70710678118654752440f));
}
template <bool EXACT> __device__ __forceinline__ void mat_act_grad(float z, int act, float& value, float& slope) {
  if (act == FOVI_GATE_SILU) {
    const float s = mat_sigmoid<EXACT>(z);
    value = EXACT ? mat_act<true>(z, act) : z * s;
    slope = s * (1.0f + z * (1.0f - s));
  } else {
    const float half = 0.5f * (1.0f + erff(z * 0.70710678118654752440f));
    value = z * half;
    slope = half + z * expf(-0.5f * z * z) * 0.39894228040143267794f;
  }
}

// Tile number of a workgroup: an XCD works on one range of tiles, the tiles of a row of tiles one after another, so
// that they share x in its L2. false: none is left.
__device__ __forceinline__ bool mat_tile(int64_t tiles_m, int64_t tiles_n, int64_t& tm, int64_t& tn) {
  const int64_t tile = xcd_tile(blockIdx.x, gridDim.x);
  if (tile >= tiles_m * tiles_n) return false;
  tm = tile / tiles_n;
  tn = tile - tm * tiles_n;
  return true;
}
inline unsigned mat_grid(int64_t tiles) { return static_cast<unsigned>((tiles + 7) / 8 * 8); }

}  // namespace fovi
