// Matrix products on the matrix unit for the feed-forward operators: fp32, bf16 and int8, with either operand's
// reduction axis contiguous ("rows") or strided ("columns"), several products of the same left operand at once, and
// the caller's own work on the sums (an epilogue) before they are written.
//
// out[m, n] = sum_k x[m, k] w[n, k]. A workgroup of four waves (eight for tiles of 256 rows) takes tiles of BM x BN one after another and walks k
// in stages of 128 bytes a row (64 bf16, 128 int8, 32 fp32 elements): whole cache lines, since parts of one cost as much
// (loads from L2 into LDS reach 34 TB/s by 128 bytes and 17 by 64). Loads go straight into LDS, a stage ahead of the
// products and past the end of a tile into the next one, so that a tile's first loads run beside the epilogue of the one
// before. The matrix instructions of a step run on registers that were read during the step before. There is one
// barrier a stage, in front of its last step: by then the stage has been read whole (its place is free for the
// loads of the stage after the next) and the next stage has landed, whose first step is read beside the last products.
// Within a row of LDS 16-byte pieces are swapped (XOR) so that the lanes of a read spread over the banks. The
// matrix instruction takes w as its first operand: a lane then holds one row m of the sums and runs of adjacent n.
#pragma once

#include "common.h"

namespace fovi {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// One operand: element (r, k) at p + r * stride + k * size where k is contiguous, else p + k * stride + r * size.
// stride in bytes; `extent` rows r. Starts, strides and contiguous runs are multiples of 16 bytes.
struct MatOperand {
  const char* p;
  int64_t stride, extent;
};

template <typename T> struct Mat;
template <> struct Mat<uint16_t> { typedef f32x16 Acc; typedef float Sum; };
template <> struct Mat<float> { typedef f32x16 Acc; typedef float Sum; };
template <> struct Mat<int8_t> { typedef i32x16 Acc; typedef int32_t Sum; };
template <typename T> constexpr int mat_bk() { return 128 / sizeof(T); }

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

// A stage of an operand in LDS: NR rows of 128 bytes of k, or (COL) k rows of NR elements.
template <typename T, int NR, bool COL, int WAVES> struct MatTile {
  static constexpr int ES = sizeof(T), BK = mat_bk<T>();
  static constexpr int BYTES = NR * 128;
  static constexpr int PIECES = COL ? NR * ES / 16 : 8;          // 16-byte pieces of an LDS row
  static constexpr int LOADS = BYTES / 1024 / WAVES;             // loads a wave makes for a stage

  static __device__ __forceinline__ int at(int r, int piece) {
    int s;
    if (!COL) s = (r >> 1) & 7;
    else if (ES == 4) s = ((r >> 2) & 1) << 3;
    else s = PIECES == 24 ? ((r >> 1) & 1) << 2 : ((r & 3) << 2) & (PIECES - 1);
    return r * PIECES * 16 + ((piece ^ s) << 4);
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

// The loads of an operand's stages. A wave's load writes 64 consecutive pieces of LDS, so the swap of pieces within a row
// is in the address that each lane reads. Rows behind the last are the last row again (their sums are not written). Pieces
// behind the last element of k, or behind the rows of an operand by columns, are read behind the buffer's end, where
// loads give zeros.
template <typename T, int NR, bool COL, int WAVES> struct MatLoader {
  typedef MatTile<T, NR, COL, WAVES> Tile;
  static constexpr int ES = sizeof(T), BK = mat_bk<T>(), LOADS = Tile::LOADS;
  static constexpr uint32_t END = 0x7fffff00u, OUTSIDE = 0x7fffff80u;
  uint64_t base;                                       // all of it uniform: the addresses are formed at each load, since
  int64_t step;                                        // registers are what the largest tiles lack
  int stride, limit;                                   // limit: the last row of the tile, or (COL) bytes of a k row

  __device__ __forceinline__ MatLoader() {}
  // (WAVES 1: every wave loads stages of its own.)
  static __device__ __forceinline__ int load(int i) { return (WAVES == 1 ? 0 : threadIdx.x >> 6) * LOADS + i; }
  __device__ __forceinline__ void open(const MatOperand& o, int64_t r0, int64_t k0) {
    stride = static_cast<int>(o.stride);
    limit = COL ? static_cast<int>(o.extent - r0 < NR ? (o.extent - r0) * ES : NR * ES)
                : static_cast<int>(o.extent - 1 - r0 < NR ? o.extent - 1 - r0 : NR);
    base = reinterpret_cast<uint64_t>(o.p) + (COL ? k0 * o.stride + r0 * ES : r0 * o.stride + k0 * ES);
    step = COL ? BK * o.stride : 128;
  }
  // Starts the loads of the stage whose k has `left` elements, and goes on to the next stage.
  __device__ __forceinline__ void start(uint32_t lds, int64_t left) {
    const i32x4 rsrc = {__builtin_amdgcn_readfirstlane(static_cast<int>(base)), __builtin_amdgcn_readfirstlane(static_cast<int>(base >> 32)),
                        static_cast<int>(END), 0x20000};
    const bool whole = left >= BK;
    const int end = static_cast<int>(COL ? left : left * ES);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int id = load(i) * 64 + (threadIdx.x & 63), r = id / Tile::PIECES;
      const int b = Tile::at(r, id % Tile::PIECES) - r * Tile::PIECES * 16;    // the swap is its own inverse
      uint32_t from = static_cast<uint32_t>(__mul24(COL || r < limit ? r : limit, stride) + b);
      if (COL && b >= limit) from = OUTSIDE;
      if (!whole && (COL ? r : b) >= end) from = OUTSIDE;
      // m0, the place in LDS, is read by the load: one wait state behind its writing
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                   :: "s"(__builtin_amdgcn_readfirstlane(lds + load(i) * 1024)), "v"(from), "s"(rsrc) : "memory");
    }
    base += step;
  }
};

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)p));
}

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

// The waves of a workgroup, WM by WN over its tile.
template <int WM, int WN> struct MatWaves {
  static constexpr int M = WM, N = WN, ALL = M * N, THREADS = 64 * ALL;
  static __device__ __forceinline__ int m() { return (threadIdx.x >> 6) / N; }
  static __device__ __forceinline__ int n() { return (threadIdx.x >> 6) % N; }
};

// Two by two; two by four for tiles of 256 rows, or four by two with 192 columns.
template <int BM, int BN> using MatUsual = MatWaves<(BM == 256 && BN == 192 ? 4 : 2), (BM == 256 && BN != 192 ? 4 : 2)>;

// A run of stages: NB products of the tile's rows of x.
template <typename T, int BM, int BN, int NB, bool CX, bool CW, typename W = MatUsual<BM, BN>>
struct MatPhase {
  typedef typename Mat<T>::Acc Acc;
  typedef W Waves;
  typedef MatTile<T, BM, CX, Waves::ALL> TX;
  typedef MatTile<T, BN, CW, Waves::ALL> TW;
  static constexpr int MB = BM / 32 / Waves::M, NN = BN / 32 / Waves::N, BK = mat_bk<T>();
  static constexpr int BYTES = TX::BYTES + NB * TW::BYTES, LOADS = TX::LOADS + NB * TW::LOADS;

  MatLoader<T, BM, CX, Waves::ALL> lx;
  MatLoader<T, BN, CW, Waves::ALL> lw[NB];

  __device__ __forceinline__ void open(const MatOperand& x, const MatOperand (&w)[NB], int64_t m0, int64_t n0, int64_t k0) {
    lx.open(x, m0, k0);
#pragma unroll
    for (int b = 0; b < NB; ++b) lw[b].open(w[b], n0, k0);
  }
  __device__ __forceinline__ void start(uint32_t lds, int64_t left) {
    lx.start(lds, left);
#pragma unroll
    for (int b = 0; b < NB; ++b) lw[b].start(lds + TX::BYTES + b * TW::BYTES, left);
  }
  // The operands of a step in registers. Every wave holds MB x NN blocks of 32 x 32 of each product.
  struct Step {
    u32x4 x[MB], w[NB][NN];
    __device__ __forceinline__ void read(const char* lds, int s) {
      const int wm = Waves::m() * (BM / Waves::M), wn = Waves::n() * (BN / Waves::N);
#pragma unroll
      for (int i = 0; i < MB; ++i) x[i] = TX::read(lds, wm + 32 * i, s);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < NN; ++j) w[b][j] = TW::read(lds + TX::BYTES + b * TW::BYTES, wn + 32 * j, s);
    }
    // acc[first + b] += the products.
    template <int NA>
    __device__ __forceinline__ void multiply(Acc (&acc)[NA][MB][NN], int first) const {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int j = 0; j < NN; ++j) acc[first + b][i][j] = mat_step(T(), w[b][j], x[i], acc[first + b][i][j]);
    }
  };
  // fp32 sums are taken by stages and added up: a chain of 32 products and one of the stages, instead of one of all
  // (2571 x 387, hidden 1031: outputs and gradients 9.8e-7 off in a row, the norm of the difference over the norm, 2.3e-7 so).
  static constexpr bool STAGED = sizeof(T) == 4;
  // The products of `stages` stages. step[0] holds the first step of the first one; first_step(lds) reads that of the
  // stage behind the last one, if there is one.
  template <int NA, typename Ring, typename Produce, typename FirstStep>
  static __device__ __forceinline__ void run(Ring& ring, int64_t stages, Step (&step)[2], Acc (&acc)[NA][MB][NN], int first,
                                             const Produce& produce, const FirstStep& first_step) {
    for (int64_t t = stages; t > 0; --t) {
      const char* now = ring.now();
      Acc part[NB][MB][NN];
      if (STAGED) mat_clear(part);
#pragma unroll
      for (int s = 0; s < 3; ++s) {
        step[(s + 1) & 1].read(now, s + 1);
        __builtin_amdgcn_sched_barrier(0);
        if (STAGED) step[s & 1].multiply(part, 0);
        else step[s & 1].multiply(acc, first);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (ring.advance(produce)) {
        if (t > 1) step[0].read(ring.now(), 0);
        else first_step(ring.now());
        __builtin_amdgcn_sched_barrier(0);
      }
      if (STAGED) {
        step[1].multiply(part, 0);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NN; ++j) acc[first + b][i][j] += part[b][i][j];
      } else {
        step[1].multiply(acc, first);
      }
    }
  }
  // The same where the sums leave registers for one step only: its reads are waited for, beside another wave's products.
  template <int NA, typename Ring, typename Produce>
  static __device__ __forceinline__ void run_lean(Ring& ring, int64_t stages, Acc (&acc)[NA][MB][NN], int first, const Produce& produce) {
    Step step;
    for (int64_t t = stages; t > 0; --t) {
      const char* now = ring.now();
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        step.read(now, s);
        if (s == 3) ring.advance(produce);
        __builtin_amdgcn_sched_barrier(0);
        step.multiply(acc, first);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
};

// The stages of a workgroup, two in LDS. produce(lds) starts the loads of the next stage; false: there is none left.
// Loads and stores of a wave end in the order of their issue, so that a stage has landed when no more is outstanding than was
// issued behind it: the STORES of an epilogue that was run since (at least so many).
template <int BYTES, int STORES> struct MatRing {
  static constexpr int LDS = 2 * BYTES;
  static_assert(STORES < 64, "more than the counter holds");
  const char* lds;
  int at;                                              // the stage being multiplied is in this half
  bool more;                                           // whether the next one was started
  bool stored;                                         // whether an epilogue has run since then
  template <typename Produce> __device__ __forceinline__ MatRing(const char* memory, const Produce& produce)
      : lds(memory), at(0), stored(false) {
    produce(lds_address(lds));
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    more = produce(lds_address(lds) + BYTES);
  }
  __device__ __forceinline__ const char* now() const { return lds + at * BYTES; }
  // On to the next stage (false: none), when every wave has read this one and everybody's loads of the next have landed.
  template <typename Produce> __device__ __forceinline__ bool advance(const Produce& produce) {
    if (!more) return false;
    if (stored) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(STORES) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    stored = false;
    more = produce(lds_address(lds) + at * BYTES);
    at ^= 1;
    return true;
  }
};

// epilogue(m, n, count, v, column, extra): the sums v[b][0 .. count) of row m from column n on, in runs of eight; what
// epilogue.column(n, count) gave for the columns, and epilogue.load(m, n, count) for the run. These are read a column ahead,
// and for all runs at once (where the sums and they are too many for the registers, for a column and its runs), not run by
// run behind the stores of the run before. A lane's block holds four adjacent columns of every eight, the lane 32
// further on the other four: the two swap halves of two such runs.
template <typename Waves, int BM, int BN, typename Sum, bool WHOLE, typename Acc, int NA, int MB, int NN, typename Epilogue>
__device__ __forceinline__ void mat_runs(const Acc (&acc)[NA][MB][NN], int64_t m0, int64_t n0, int64_t M, int64_t N, const Epilogue& epilogue) {
  constexpr bool FULL = NA * MB * NN * 16 + 2 * NN * MB * static_cast<int>(sizeof(typename Epilogue::Extra)) / 4 > 140;
  const int l = threadIdx.x & 63;
  const int64_t mw = m0 + Waves::m() * (BM / Waves::M) + (l & 31), nw = n0 + Waves::n() * (BN / Waves::N) + 8 * (l >> 5);
  typename Epilogue::Extra extra[FULL ? 1 : 2 * NN][MB];
  auto load = [&](int c, typename Epilogue::Extra (&to)[MB]) __attribute__((always_inline)) {
    const int64_t n = nw + 16 * c;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      if (WHOLE) to[i] = epilogue.load(mw + 32 * i, n, 8);
      else if (mw + 32 * i < M && n < N) to[i] = epilogue.load(mw + 32 * i, n, static_cast<int>(N - n < 8 ? N - n : 8));
    }
  };
  if (!FULL) {
#pragma unroll
    for (int c = 0; c < 2 * NN; ++c) load(c, extra[FULL ? 0 : c]);
  }
  typename Epilogue::Column column[FULL ? 1 : 2];
  auto load_column = [&](int c) __attribute__((always_inline)) {
    const int64_t n = nw + 16 * c;
    if (WHOLE) column[FULL ? 0 : c & 1] = epilogue.column(n, 8);
    else if (n < N) column[FULL ? 0 : c & 1] = epilogue.column(n, static_cast<int>(N - n < 8 ? N - n : 8));
  };
  if (!FULL) load_column(0);
#pragma unroll
  for (int c = 0; c < 2 * NN; ++c) {                   // columns of 16
    if (FULL) { load_column(c); load(c, extra[0]); }
    else if (c + 1 < 2 * NN) load_column(c + 1);
    const int j = c / 2, q = c % 2 * 2;
    const int64_t n = nw + 16 * c;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      const int64_t m = mw + 32 * i;
      Sum v[NA][8];
#pragma unroll
      for (int b = 0; b < NA; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const auto t = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, static_cast<Sum>(acc[b][i][j][4 * q + e])),
                                                          __builtin_bit_cast(uint32_t, static_cast<Sum>(acc[b][i][j][4 * q + 4 + e])), false, false);
          const uint32_t t0 = t[0], t1 = t[1];         // (a bit cast of t[1] itself takes t[0])
          v[b][e] = __builtin_bit_cast(Sum, t0);
          v[b][4 + e] = __builtin_bit_cast(Sum, t1);
        }
      if (WHOLE) epilogue(m, n, 8, v, column[FULL ? 0 : c & 1], extra[FULL ? 0 : c][i]);
      else if (m < M && n < N) epilogue(m, n, static_cast<int>(N - n < 8 ? N - n : 8), v, column[FULL ? 0 : c & 1], extra[FULL ? 0 : c][i]);
      if (FULL) __builtin_amdgcn_sched_barrier(0);     // (mixed, the runs take more registers than there are)
    }
  }
}
template <typename Waves, int BM, int BN, typename Sum, typename Acc, int NA, int MB, int NN, typename Epilogue>
__device__ __forceinline__ bool mat_finish(const Acc (&acc)[NA][MB][NN], int64_t m0, int64_t n0, int64_t M, int64_t N,
                                           const Epilogue& epilogue) {
  const bool whole = m0 + BM <= M && n0 + BN <= N;     // every lane stores every run
  if (whole) mat_runs<Waves, BM, BN, Sum, true>(acc, m0, n0, M, N, epilogue);
  else mat_runs<Waves, BM, BN, Sum, false>(acc, m0, n0, M, N, epilogue);
  return whole;
}

// Eight (or `count`) adjacent elements, in registers as they are in memory, and as floats.
template <typename T> struct Run {
  T e[8];
  __device__ __forceinline__ void load(const T* p, int count) {
    if (count == 8) {
      __builtin_memcpy(e, p, sizeof(e));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = i < count ? p[i] : T(0);
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return Elem<T>::load(e + i); }
};
struct NoExtra {};
struct NoColumn {
  typedef NoExtra Column;
  __device__ __forceinline__ Column column(int64_t, int) const { return Column(); }
};
struct Plain : NoColumn {                              // an epilogue that reads nothing else
  typedef NoExtra Extra;
  __device__ __forceinline__ Extra load(int64_t, int64_t, int) const { return Extra(); }
};
template <typename T> __device__ __forceinline__ void store_run(T* p, int count, const float (&v)[8]) {
  T e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) Elem<T>::store(e + i, v[i]);
  if (count == 8) {
    __builtin_memcpy(p, e, sizeof(e));
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < count) p[i] = e[i];
  }
}

// Activations and their derivatives. EXACT: the library's exponential and division, for fp32 results
// (with the hardware's, silu is 8e-7 off at gates of -10 to -20 and 1.7e-6 at -40).
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

// The tiles of a launch: `tiles` for each share of k, `items` in all. An XCD works on one range of them, its
// workgroups on neighbours. Tiles follow one another along n, in bands of `band` rows of tiles that are walked
// column by column, so that the 32 tiles that an XCD works on at a time form a block of 8 x 4 or so: the rows of x and w
// that they share come from its L2.
struct MatWork {
  uint32_t tiles_m, tiles_n, tiles, items, band;
};
struct MatItem {
  uint32_t i, end, step;
  __device__ __forceinline__ explicit MatItem(const MatWork& w) {
    const uint32_t per = (w.items + 7) >> 3, xcd = blockIdx.x & 7;
    i = xcd * per + (blockIdx.x >> 3);
    end = (xcd + 1) * per < w.items ? (xcd + 1) * per : w.items;
    step = gridDim.x >> 3;
  }
  __device__ __forceinline__ bool live() const { return i < end; }
  __device__ __forceinline__ void next() { i += step; }
  __device__ __forceinline__ int64_t share(const MatWork& w) const { return i / w.tiles; }
  __device__ __forceinline__ void place(const MatWork& w, int64_t& m, int64_t& n) const {
    const uint32_t t = i % w.tiles, band = w.band * w.tiles_n, g = t / band, r = t - g * band;
    const uint32_t rows = w.tiles_m - g * w.band < w.band ? w.tiles_m - g * w.band : w.band;
    m = g * w.band + r % rows;
    n = r / rows;
  }
};
inline int64_t mat_tiles(int64_t M, int64_t N, int bm, int bn) { return (M + bm - 1) / bm * ((N + bn - 1) / bn); }
inline MatWork mat_work(int64_t M, int64_t N, int bm, int bn, int64_t shares) {
  const uint32_t tm = static_cast<uint32_t>((M + bm - 1) / bm), tn = static_cast<uint32_t>((N + bn - 1) / bn);
  return MatWork{tm, tn, tm * tn, static_cast<uint32_t>(tm * tn * shares), tn <= 8 ? 4u : 8u};
}
// Workgroups: `each` on each of 256 compute units, a multiple of the 8 XCDs.
inline unsigned mat_grid(const MatWork& w, int each) {
  const unsigned n = (w.items + 7) / 8 * 8;
  return n < 256u * each ? n : 256u * each;
}

// Columns of a tile of 256 rows: 192 where that leaves less of the last one empty.
inline int mat_columns(int64_t N) { return (N + 191) / 192 * 192 < (N + 255) / 256 * 256 ? 192 : 256; }

// The tile of a product of M x N sums (`shares` times): of 256, 128 or 64 rows, whichever ends first by the time that a
// compute unit takes for a stage of its workgroups, one, two or four of them. A stage of 64 K sums is taken as 1, 1.13
// and 1.6 in tiles of these sizes (131072 x 1024 by 384, bf16: 123, 131 and 203 us, in short runs 129, 147 and 208; 131072 x
// 384 by 2 x 1024: 277, 285 and 406, in short runs 300, 344 and 432): small ones read more bytes a product from L2 and LDS. fp32 products are slow enough for tiles of 64 to keep up and, with more
// waves, to be ahead (2571 x 387 by 2 x 1031: 58 us, and 70 in tiles of 128); tiles of 256 rows are not built for them.
inline int mat_tile_size(int64_t M, int64_t N, int64_t shares, bool fp32, int columns) {
  const int64_t l = (mat_tiles(M, N, 256, columns) * shares + 255) / 256 * (fp32 ? 1 << 20 : columns);
  const int64_t m = (mat_tiles(M, N, 128, 128) * shares + 511) / 512 * 145;
  const int64_t s = (mat_tiles(M, N, 64, 64) * shares + 1023) / 1024 * (fp32 ? 61 : 102);
  return l <= m && l <= s ? 256 : m <= s ? 128 : 64;
}

template <typename Kernel, typename... Args>
inline void mat_launch(Kernel kernel, dim3 grid, int threads, size_t lds, hipStream_t stream, Args... args) {
  if (lds > 65536 && reserve_dynamic_lds(reinterpret_cast<const void*>(kernel), lds) != hipSuccess) return;
  kernel<<<grid, threads, lds, stream>>>(args...);
}

// Whether the loads take an operand by rows as it is.
template <typename T> inline bool mat_whole(const MatOperand& o, int64_t k) {
  return (reinterpret_cast<uintptr_t>(o.p) | o.stride | k * static_cast<int64_t>(sizeof(T))) % 16 == 0 && o.stride < (1 << 22);
}

// out = x w^T through the epilogue, k in up to two segments of other operands each. With more than one share, every
// segment is split into shares of `share`, whose sums go to `part` and are added up by a second launch.
struct MatSegments {
  MatOperand x[2], w[2];
  int64_t k[2];
  int n;
};

template <typename Sum> struct MatPartial : Plain {             // the sums of a share
  static constexpr int STORES = 2;                      // of 16 bytes for a run of eight
  Sum* part; int64_t M, N;
  __device__ __forceinline__ void operator()(int64_t m, int64_t n, int count, const Sum (&v)[1][8], const NoExtra&, const NoExtra&) const {
    Sum* p = part + m * N + n;
    if (count == 8) {
      __builtin_memcpy(p, v[0], 32);
    } else {
#pragma unroll
      for (int i = 0; i < 7; ++i)
        if (i < count) p[i] = v[0][i];
    }
  }
};

template <typename T, int BM, int BN, bool CX, bool CW, typename Epilogue> struct MatLinearTile {
  typedef MatPhase<T, BM, BN, 1, CX, CW> Phase;
  typedef MatRing<Phase::BYTES, 2 * Phase::MB * Phase::NN * Epilogue::STORES> Ring;
};
template <typename T, int BM, int BN, bool CX, bool CW, typename Epilogue>
__global__ __launch_bounds__((MatUsual<BM, BN>::THREADS), 2) void mat_linear_kernel(MatSegments s, int64_t M, int64_t N, MatWork work,
                                                                                   int64_t share, Epilogue epilogue) {
  typedef typename MatLinearTile<T, BM, BN, CX, CW, Epilogue>::Phase Phase;
  typedef typename MatLinearTile<T, BM, BN, CX, CW, Epilogue>::Ring Ring;
  typedef typename Mat<T>::Sum Sum;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  MatItem item(work), ahead(work);
  if (!item.live()) return;
  auto part = [&](const MatItem& at, int i, int64_t& from) __attribute__((always_inline)) {
    const int64_t k = i ? s.k[1] : s.k[0];
    from = at.share(work) * share;
    return (from + share < k ? from + share : k) - from;
  };
  Phase phase;
  int segment = -1;
  int64_t left = 0;
  auto produce = [&](uint32_t to) __attribute__((always_inline)) {
    while (left <= 0) {
      if (++segment == s.n) { segment = 0; ahead.next(); }
      if (!ahead.live()) return false;
      int64_t from;
      left = part(ahead, segment, from);
      const MatOperand w[1] = {segment ? s.w[1] : s.w[0]};
      int64_t tm, tn;
      ahead.place(work, tm, tn);
      phase.open(segment ? s.x[1] : s.x[0], w, tm * BM, tn * BN, from);
    }
    phase.start(to, left);
    left -= Phase::BK;
    return true;
  };
  Ring ring(lds, produce);
  typename Phase::Step step[2];
  auto first_step = [&](const char* now) __attribute__((always_inline)) { step[0].read(now, 0); };
  first_step(ring.now());
  for (; item.live(); item.next()) {
    typename Phase::Acc acc[1][Phase::MB][Phase::NN];
    mat_clear(acc);
    int64_t stages = 0, from;
    for (int i = 0; i < s.n; ++i) {
      const int64_t n = part(item, i, from);
      stages += n > 0 ? (n + Phase::BK - 1) / Phase::BK : 0;
    }
    Phase::run(ring, stages, step, acc, 0, produce, first_step);
    int64_t tm, tn;
    item.place(work, tm, tn);
    if constexpr (__is_same(Epilogue, MatPartial<Sum>)) {
      MatPartial<Sum> mine = epilogue;
      mine.part += item.share(work) * M * N;
      ring.stored = mat_finish<typename Phase::Waves, BM, BN, Sum>(acc, tm * BM, tn * BN, M, N, mine);
    } else {
      ring.stored = mat_finish<typename Phase::Waves, BM, BN, Sum>(acc, tm * BM, tn * BN, M, N, epilogue);
    }
  }
}

// The shares' sums added up in order, through the epilogue.
template <typename Sum, typename Epilogue>
__global__ __launch_bounds__(256) void mat_join_kernel(const Sum* part, int64_t shares, int64_t M, int64_t N, Epilogue epilogue) {
  const int64_t per = (N + 7) / 8, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= M * per) return;
  const int64_t m = i / per, n = (i - m * per) * 8;
  const int count = static_cast<int>(N - n < 8 ? N - n : 8);
  Sum v[1][8] = {};
  for (int64_t z = 0; z < shares; ++z) {
    const Sum* p = part + (z * M + m) * N + n;
    Sum t[8] = {};
    if (count == 8) {
      __builtin_memcpy(t, p, 32);
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e) t[e] = e < count ? p[e] : 0;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[0][e] += t[e];
  }
  epilogue(m, n, count, v, epilogue.column(n, count), epilogue.load(m, n, count));
}

// Shares of k. Over the tokens (long: k in the ten thousands, few sums) as many as give every compute unit a tile of
// 256 x 256, of 512 tokens or more; else, where even tiles of 64 x 64 leave half of the card without work, as many as
// fill it, of eight stages or more.
template <typename T> inline int64_t mat_shares(int64_t M, int64_t N, int64_t k, bool tokens) {
  const int64_t small = mat_tiles(M, N, 64, 64), most = tokens ? (k + 511) / 512 : k / (8 * mat_bk<T>());
  int64_t shares = 1;
  if (tokens) {
    shares = (256 + mat_tiles(M, N, 256, 256) - 1) / mat_tiles(M, N, 256, 256);
    if (shares > most) shares = (1024 + small - 1) / small;
  } else if (small <= 512) {
    shares = 1024 / small;
  }
  if (shares > most) shares = most;
  return shares < 1 ? 1 : shares;
}
template <typename T> inline int64_t mat_part_bytes(int64_t M, int64_t N, int64_t k, bool tokens) {
  const int64_t shares = mat_shares<T>(M, N, k, tokens);
  return shares > 1 ? shares * M * N * 4 : 0;
}

template <typename T, int BM, int BN, bool CX, bool CW, typename Epilogue>
inline void mat_linear_tiles(const MatSegments& s, int64_t M, int64_t N, int64_t share, int64_t shares, const Epilogue& epilogue,
                             hipStream_t stream) {
  const MatWork work = mat_work(M, N, BM, BN, shares);
  mat_launch(mat_linear_kernel<T, BM, BN, CX, CW, Epilogue>, mat_grid(work, 256 / BM), (MatUsual<BM, BN>::THREADS),
             MatLinearTile<T, BM, BN, CX, CW, Epilogue>::Ring::LDS, stream, s, M, N, work, share, epilogue);
}
// Tiles of 256 rows have 128 columns for an epilogue that reads much beside the sums: more of it is then read at once
// (131072 x 1024 by 384, bf16, with gate and up read and three results written: 551 us, and 763 with 256 columns). Its tiles
// of 256 and 128 rows still take more than the 256 registers there are: 37 and 35 of a lane's go through scratch memory.
template <typename Epilogue> constexpr bool mat_narrow = false;
template <typename T, bool CX, bool CW, typename Epilogue>
inline void mat_linear_shares(const MatSegments& s, int64_t M, int64_t N, int64_t share, int64_t shares, const Epilogue& epilogue,
                              hipStream_t stream) {
  const int size = mat_tile_size(M, N, shares, sizeof(T) == 4, mat_narrow<Epilogue> ? 128 : mat_columns(N));
  if constexpr (sizeof(T) < 4 && mat_narrow<Epilogue>) {
    if (size == 256) {
      mat_linear_tiles<T, 256, 128, CX, CW>(s, M, N, share, shares, epilogue, stream);
      return;
    }
  } else if constexpr (sizeof(T) < 4) {
    if (size == 256) {
      if (mat_columns(N) == 192) mat_linear_tiles<T, 256, 192, CX, CW>(s, M, N, share, shares, epilogue, stream);
      else mat_linear_tiles<T, 256, 256, CX, CW>(s, M, N, share, shares, epilogue, stream);
      return;
    }
  }
  if (size == 128) mat_linear_tiles<T, 128, 128, CX, CW>(s, M, N, share, shares, epilogue, stream);
  else mat_linear_tiles<T, 64, 64, CX, CW>(s, M, N, share, shares, epilogue, stream);
}
// part: mat_part_bytes of M, N and the longest segment.
template <typename T, bool CX, bool CW, typename Epilogue>
inline void mat_linear(const MatSegments& s, int64_t M, int64_t N, void* part, bool tokens, const Epilogue& epilogue, hipStream_t stream) {
  typedef typename Mat<T>::Sum Sum;
  const int64_t k = s.n == 2 && s.k[1] > s.k[0] ? s.k[1] : s.k[0], shares = mat_shares<T>(M, N, k, tokens);
  if (shares == 1) {
    mat_linear_shares<T, CX, CW>(s, M, N, k, 1, epilogue, stream);
    return;
  }
  const int64_t bk = mat_bk<T>(), share = ((k + shares - 1) / shares + bk - 1) / bk * bk, used = (k + share - 1) / share;
  Sum* sums = static_cast<Sum*>(part);
  mat_linear_shares<T, CX, CW>(s, M, N, share, used, MatPartial<Sum>{{}, sums, M, N}, stream);
  mat_join_kernel<Sum, Epilogue><<<static_cast<unsigned>((M * ((N + 7) / 8) + 255) / 256), 256, 0, stream>>>(sums, used, M, N, epilogue);
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

// Matrices that the loads do not take as they are (rows of other lengths, starts or strides than whole 16-byte pieces)
// are copied in front of a product, their rows filled up with zeros: one launch for all of a call.
struct MatCopies {
  static constexpr int MOST = 5;
  struct { const char* from; char* to; int64_t stride, len; } m[MOST];
  int64_t first[MOST + 1];                             // of each matrix's pieces, in one sequence
  int n;
};
__global__ void mat_copy_kernel(MatCopies c);

// A call's operands: take() gives the matrix that the kernels read, which is the caller's or a copy in the workspace.
class MatInputs {
 public:
  explicit MatInputs(void* workspace) : at_(static_cast<char*>(workspace)), start_(at_) { copies_.n = 0; copies_.first[0] = 0; }
  // rows x cols elements of `es` bytes, `stride` elements apart; the result's stride is in bytes.
  MatOperand take(const void* p, int64_t stride, int64_t rows, int64_t cols, int64_t es) {
    const int64_t bytes = cols * es;
    const MatOperand as_is = {static_cast<const char*>(p), stride * es, rows};
    if (mat_whole<char>(as_is, bytes)) return as_is;
    const int64_t wide = (bytes + 15) / 16 * 16;
    auto& m = copies_.m[copies_.n];
    m.from = static_cast<const char*>(p); m.to = at_; m.stride = stride * es; m.len = bytes;
    copies_.first[copies_.n + 1] = copies_.first[copies_.n] + rows * (wide / 16);
    ++copies_.n;
    const MatOperand o = {at_, wide, rows};
    at_ += (rows * wide + 255) / 256 * 256;
    return o;
  }
  int64_t used() const { return at_ - start_; }
  char* rest() const { return at_; }
  void copy(hipStream_t s) const;

 private:
  MatCopies copies_;
  char* at_;
  char* start_;
};

}  // namespace fovi
