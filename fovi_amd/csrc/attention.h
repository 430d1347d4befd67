// Shared parts of the attention kernels (forward, single-token forward, backward): parameters, the LDS
// tile layout and the two kinds of 32 x 32 MFMA product.
//
// Every kernel works on 32 x 32 blocks of the score matrix in the C layout of the 32x32 MFMA: lane l
// holds column l % 32 and the rows 8 (i / 4) + 4 (l / 32) + i % 4, i = 0..15. The columns are what the
// wave owns (its query rows in the forward and in dq, its states in dk and dv), so softmax
// statistics and sums over the other axis stay in a lane but for one swap of halves. The block
// then is the B operand of the second product (out^T = V^T P^T and its like) as it lies in the
// registers: the k order of an MFMA is free as long as A agrees, so A is read from LDS in the order
// that the C layout has (bf16: transposing 64-bit reads; fp32: plain 32-bit reads). No probability
// moves between lanes.
#pragma once

#include "common.h"

namespace fovi {

constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;

struct AttnParams {
  const void* q; const void* k; const void* v; const void* mask; const int32_t* lens;
  void* o; float* stats; void* rest;
  const void* dout; void* dq; void* dk; void* dv;
  float* part;                // partial results of split work
  float* part_k;              // backward: those of dk and dv (part: dq)
  float* delta;               // backward: dout . out of each row
  int64_t B, Lq, Lk;
  int H, Hk, G, D, kind;
  int64_t qs[3], ks[3], vs[3], os[3], ms[4], dos[3], dqs[3], dks[3], dvs[3];
  float scale, c;             // c = scale * log2(e)
  int64_t R;                  // query rows of a key head: G * Lq, row r = head r / Lq of the group, query r % Lq
  int splits;                 // of the summed axis
  int64_t chunk;              // its length per split
  int64_t tiles;              // workgroups along the owned axis
  int k_splits;               // backward: of dk and dv, for the join
};

__device__ __forceinline__ int64_t attn_len(const AttnParams& p, int64_t b) {
  if (!p.lens) return p.Lk;
  const int64_t n = p.lens[b];
  return n < 0 ? 0 : n < p.Lk ? n : p.Lk;
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <typename T> struct Chunk { static constexpr int N = 16 / sizeof(T); };   // elements of 16 bytes

// 16 bytes of a row from element c * N on; zeros beyond the D elements of a head (a multiple of N).
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* row, int c, int D) {
  return c * Chunk<T>::N < D ? *reinterpret_cast<const u32x4*>(row + c * Chunk<T>::N) : u32x4{0, 0, 0, 0};
}

// Whether any of the chunk's values is infinite or NaN.
template <typename T> __device__ __forceinline__ bool chunk_bad(u32x4 u);
template <> __device__ __forceinline__ bool chunk_bad<float>(u32x4 u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (w[i] & 0x7f800000u) == 0x7f800000u;
  return bad;
}
template <> __device__ __forceinline__ bool chunk_bad<uint16_t>(u32x4 u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (w[i] & 0x7f80u) == 0x7f80u || (w[i] & 0x7f800000u) == 0x7f800000u;
  return bad;
}

// An LDS tile has rows of LP elements (a power of two) in 16-byte chunks; chunk c of row r lies at
// place c ^ swizzle(r). 16 rows of one chunk (operand reads by rows) then fall on different banks,
// and so do the four rows of four chunks that a transposing read takes (fp32: rows r and r + 4).
template <typename T, int LP> __device__ __forceinline__ int swizzle(int r) {
  constexpr int NC = LP / Chunk<T>::N;
  if (sizeof(T) == 2) {
    if (NC == 4) return (r >> 2) & 3;
    if (NC == 8) return ((r >> 1) & 1) << 2 | ((r >> 2) & 1) << 1 | ((r >> 3) & 1);
    return (r & 3) << 2 | ((r >> 2) & 3);
  }
  if (NC == 8) return (r >> 1) & 7;
  return ((r >> 2) & 1) << 3 | (r & 3) << 1 | ((r >> 3) & 1);
}

template <typename T, int LP> __device__ __forceinline__ int tile_at(int r, int c) {
  return r * static_cast<int>(LP * sizeof(T)) + ((c ^ swizzle<T, LP>(r)) << 4);
}

// One step of a product over the head elements: both operands hold the chunk 2 t + l / 32 of their row.
__device__ __forceinline__ f32x16 mma_step(uint16_t, u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma_step(float, u32x4 a, u32x4 b, f32x16 c) {
  c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
}

// A score block as the B operand of the second product. bf16 rounds it (to nearest even): the matrix
// unit takes both operands in one type, and a value in [0, 1] (or its product with a difference)
// loses at most 2^-9 of itself, which the sums then average. sum() adds up what the product will see,
// so that probabilities and their sum agree (a row of equal values comes out exact) and dout . out
// cancels against dout . v in the backward as it should.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
template <typename T> struct Block;
template <> struct Block<uint16_t> {
  bf16x8 b[2];
  __device__ __forceinline__ Block() {}
  __device__ __forceinline__ explicit Block(const f32x16& s) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 8; ++i) b[t][i] = static_cast<__bf16>(s[8 * t + i]);
  }
  __device__ __forceinline__ float sum(float start) const {
    const bf16x2 one = {static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)};
    float even = start, odd = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      even = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{b[0][i], b[0][i + 1]}, one, even, false);
      odd = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{b[0][i + 2], b[0][i + 3]}, one, odd, false);
      even = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{b[1][i], b[1][i + 1]}, one, even, false);
      odd = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{b[1][i + 2], b[1][i + 3]}, one, odd, false);
    }
    return even + odd;
  }
};
template <> struct Block<float> {
  f32x16 b;
  __device__ __forceinline__ Block() {}
  __device__ __forceinline__ explicit Block(const f32x16& s) : b(s) {}
  __device__ __forceinline__ float sum(float start) const {
    float part[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) part[i & 3] += b[i];
    return start + ((part[0] + part[1]) + (part[2] + part[3]));
  }
};

__device__ __forceinline__ s16x4 read_tr(const char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p));
}

// The A operand of tile[base .. base + 31, 32 head elements dt * 32 ..]^T, in the order of a block, and
// acc += it * block. Reads and products are apart so that the reads of several operands can be in
// flight together: left to itself the compiler saves registers and waits for every one.
template <typename T, int LP> struct Turned;
template <int LP> struct Turned<uint16_t, LP> {
  bf16x8 a[2];
  __device__ __forceinline__ void read(const char* tile, int base, int dt) {
    const int l = threadIdx.x & 63;
    const int r = 4 * (l >> 5) + ((l & 15) >> 2), c = dt * 4 + 2 * ((l >> 4) & 1) + ((l & 3) >> 1);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char* at = tile + (base + 16 * t) * LP * 2 + (l & 1) * 8;
      const s16x4 lo = read_tr(at + tile_at<uint16_t, LP>(r, c)), hi = read_tr(at + tile_at<uint16_t, LP>(r + 8, c));
      a[t] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
  __device__ __forceinline__ f32x16 mma(const Block<uint16_t>& s, f32x16 acc) const {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], s.b[0], acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], s.b[1], acc, 0, 0, 0);
  }
};
template <int LP> struct Turned<float, LP> {
  float a[16];
  __device__ __forceinline__ void read(const char* tile, int base, int dt) {
    const int l = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = 8 * (i / 4) + 4 * (l >> 5) + i % 4, d = dt * 32 + (l & 31);
      a[i] = *reinterpret_cast<const float*>(tile + base * LP * 4 + tile_at<float, LP>(r, d >> 2) + (d & 3) * 4);
    }
  }
  __device__ __forceinline__ f32x16 mma(const Block<float>& s, f32x16 acc) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], s.b[i], acc, 0, 0, 0);
    return acc;
  }
};

// Reads stay above, products below.
__device__ __forceinline__ void reads_done() { __builtin_amdgcn_sched_barrier(0); }

// s (and s2) += the 32 rows of `tile` (`tile2`) times the columns b (b2), over the head elements, G pieces
// of each read ahead.
template <typename T, int LP, int STEPS>
__device__ __forceinline__ void row_product(const char* tile, const u32x4 (&b)[STEPS], f32x16& s) {
  constexpr int G = STEPS < 4 ? STEPS : 4;
  const int l = threadIdx.x & 63;
#pragma unroll
  for (int t = 0; t < STEPS; t += G) {
    u32x4 a[G];
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (t + g < STEPS) a[g] = *reinterpret_cast<const u32x4*>(tile + tile_at<T, LP>(l & 31, 2 * (t + g) + (l >> 5)));
    reads_done();
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (t + g < STEPS) s = mma_step(T(), a[g], b[t + g], s);
  }
}
template <typename T, int LP, int G, bool BATCH, int STEPS>
__device__ __forceinline__ void row_products(const char* tile, const char* tile2, const u32x4 (&b)[STEPS], const u32x4 (&b2)[STEPS],
                                             f32x16& s, f32x16& s2) {
  const int l = threadIdx.x & 63;
#pragma unroll
  for (int t = 0; t < STEPS; t += G) {
    u32x4 a[G], a2[G];
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (t + g < STEPS) {
        const int at = tile_at<T, LP>(l & 31, 2 * (t + g) + (l >> 5));
        a[g] = *reinterpret_cast<const u32x4*>(tile + at);
        a2[g] = *reinterpret_cast<const u32x4*>(tile2 + at);
      }
    if (BATCH) reads_done();
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (t + g < STEPS) {
        s = mma_step(T(), a[g], b[t + g], s);
        s2 = mma_step(T(), a2[g], b2[t + g], s2);
      }
  }
}

// The same product pair by pair, leaving out the pairs whose block value is kLeftOut: for tiles that
// hold infinities or NaN under a mask, where 0 * value would not be 0.
constexpr float kLeftOut = -0.0f;
__device__ __forceinline__ bool left_out(float v) { return __float_as_uint(v) == 0x80000000u; }

template <typename T, int LP, int DT>
__device__ __forceinline__ void slow_second(const char* tile, int base, const f32x16& s, f32x16 (&acc)[DT]) {
  const int h = (threadIdx.x & 63) >> 5;
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = s[i];
#pragma unroll 1
  for (int i = 0; i < 32; ++i) {
    const float other = __shfl_xor(v[i >> 1], 32), sv = i & 1 ? other : v[i >> 1];
    if (left_out(sv)) continue;
    const int r = 8 * (i >> 3) + 4 * (h ^ (i & 1)) + ((i >> 1) & 3);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int d = dt * 32 + 8 * (e / 4) + 4 * h + e % 4;
        const T* at = reinterpret_cast<const T*>(tile + base * static_cast<int>(LP * sizeof(T)) +
                                                 tile_at<T, LP>(r, d / Chunk<T>::N)) + d % Chunk<T>::N;
        acc[dt][e] = fmaf(sv, Elem<T>::load(at), acc[dt][e]);
      }
  }
}

// A tile of ROWS rows on its way from memory to LDS through the registers of THREADS threads. A thread
// keeps its 16-byte column; its place in the tile is a 32-bit offset from the tile's (uniform) address, so
// that a full tile's loads take no vector arithmetic: on this machine matrix and vector instructions of
// a SIMD hardly overlap, and every vector instruction of the loop adds to its time. Loads are never
// predicated (that would wait for earlier ones): rows behind the last are the last row again, which the products
// meet with probability 0. Where an infinity in it would turn that into NaN, clear_tail() makes them zeros: without
// a mask, for what probabilities are multiplied with (under a mask a tile with infinities leaves pairs out one by
// one; of keys and queries an infinity is in the scores already).
constexpr int64_t kMostPitch = int64_t(1) << 26;       // bytes between rows: 64 of them stay below 2^32

template <typename T, int LP, int ROWS, int THREADS>
struct Staged {
  static constexpr int NC = LP / Chunk<T>::N, STEP = THREADS / NC, N = (ROWS + STEP - 1) / STEP;
  u32x4 r[N];
  uint32_t off, pitch, col;   // bytes
  int row, c, last;           // last: of the rows that the tile has
  __device__ __forceinline__ void init(int64_t stride, int D, int thread) {
    row = thread / NC < ROWS ? thread / NC : ROWS - 1;
    c = thread % NC;
    col = c * Chunk<T>::N < D ? c * 16 : 0;
    pitch = static_cast<uint32_t>(stride * static_cast<int64_t>(sizeof(T)));
    off = row * pitch + col;
  }
  // rows [0, n) of `base`, n > 0
  __device__ __forceinline__ void load(const T* base, int64_t n) {
    const bool full = n >= ROWS;
    last = full ? ROWS - 1 : static_cast<int>(n) - 1;
    const char* at = reinterpret_cast<const char*>(base);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint32_t o = off + i * STEP * pitch;
      if (!full) [[unlikely]] o = (row + i * STEP < last ? row + i * STEP : last) * pitch + col;
      r[i] = *reinterpret_cast<const u32x4*>(at + o);
    }
  }
  // Columns behind the D head elements are zero in LDS from the start (clear) and stay so.
  __device__ __forceinline__ bool in(int D) const { return c * Chunk<T>::N < D; }
  __device__ __forceinline__ void clear(char* tile, int D) const {
    if (in(D)) return;
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<u32x4*>(tile + tile_at<T, LP>(row + i * STEP, c)) = u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void clear_tail() {
    if (last < ROWS - 1) [[unlikely]] {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (row + i * STEP > last) r[i] = u32x4{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ void store(char* tile, int D) const {
    if (!in(D)) return;
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<u32x4*>(tile + tile_at<T, LP>(row + i * STEP, c)) = r[i];
  }
  __device__ __forceinline__ bool bad() const {
    bool b = false;
#pragma unroll
    for (int i = 0; i < N; ++i) b |= chunk_bad<T>(r[i]);
    return b;
  }
};

// The other half's value (lane l and l ^ 32), by a swap of register halves: no trip through LDS.
__device__ __forceinline__ float other_half(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// Waits for every load so far. In front of the loops: without it the compiler does not know that the
// operands loaded once have arrived, and waits for them inside the loop, and with them for the next
// tile's loads.
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// KIND of a kernel: 0 no mask, 1 bits of states to keep, 2 a bias. A masked score is -inf where a pair is left
// out; else it is in units of log2 under KIND 1, so that exponentials take it as it is, and in those of the bias
// under KIND 2: biases up to the type's limits are numbers there, and differences among them count (times
// log2(e) they would overflow). unit<KIND>(p) is what a difference of such scores (KIND 0: of products q.k) is
// multiplied with for exp2.
template <int KIND> __device__ __forceinline__ float unit(const AttnParams& p) { return KIND == 0 ? p.c : KIND == 1 ? 1.0f : kLog2e; }

// exp2((s - top) unit), top finite. Under a bias the difference comes first: top * unit may pass the type's limits.
template <int KIND> __device__ __forceinline__ float exp2_below(float s, float top, float c) {
  return exp2_fast(KIND == 2 ? (s - top) * c : fmaf(s, c, -top * c));
}

// Where a block's columns are query rows, a lane has the word of its row and the block's 32 states; the
// pairs are its bits 8 (i / 4) + 4 half + i % 4.
__device__ __forceinline__ void keep_block(const AttnParams& p, uint32_t word, f32x16& s) {
  const uint32_t w = word >> (4 * ((threadIdx.x & 63) >> 5));
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = w & (1u << (8 * (i / 4) + i % 4)) ? s[i] * p.c : kNegInf;
}

__device__ __forceinline__ float biased(const AttnParams& p, float bias, float s) {
  return bias == kNegInf ? kNegInf : fmaf(s, p.scale, bias);
}

// A bias over a lane's 16 pairs: states j0 + 8 (i / 4) + i % 4 of its row (j0 holds the half; n states in all)...
__device__ __forceinline__ void bias_block(const AttnParams& p, const float* row, int64_t j0, int64_t n, f32x16& s) {
  const float* m = row + j0 * p.ms[3];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int at = 8 * (i / 4) + i % 4;
    s[i] = biased(p, j0 + at < n ? m[at * p.ms[3]] : kNegInf, s[i]);
  }
}
// ... or rows i0 + 8 (i / 4) + i % 4 (n in all) of one state, `col` its place in row 0.
__device__ __forceinline__ void bias_column(const AttnParams& p, const float* col, int64_t i0, int64_t n, f32x16& s) {
  const float* m = col + i0 * p.ms[2];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int at = 8 * (i / 4) + i % 4;
    s[i] = biased(p, i0 + at < n ? m[at * p.ms[2]] : kNegInf, s[i]);
  }
}
// A row of the mask: its words, or its biases (both of four bytes).
__device__ __forceinline__ const uint32_t* mask_row(const AttnParams& p, int64_t b, int64_t h, int64_t i) {
  return static_cast<const uint32_t*>(p.mask) + b * p.ms[0] + h * p.ms[1] + i * p.ms[2];
}

// Four adjacent head elements from d on, to memory.
__device__ __forceinline__ void store_run(uint16_t* row, int d, int D, float a, float b, float c, float e) {
  if (d >= D) return;
  uint2 w;
  w.x = static_cast<uint32_t>(f32_to_bf16_bits(a)) | static_cast<uint32_t>(f32_to_bf16_bits(b)) << 16;
  w.y = static_cast<uint32_t>(f32_to_bf16_bits(c)) | static_cast<uint32_t>(f32_to_bf16_bits(e)) << 16;
  *reinterpret_cast<uint2*>(row + d) = w;
}
__device__ __forceinline__ void store_run(float* row, int d, int D, float a, float b, float c, float e) {
  if (d < D) *reinterpret_cast<f32x4*>(row + d) = f32x4{a, b, c, e};
}

// Host side (attention_fwd.hip, attention_bwd.hip).
int attn_fwd_launch(AttnParams& p, int dtype, hipStream_t s);
int64_t attn_fwd_workspace(int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hk, int64_t D, int dtype);
int attn_pack_launch(const void* keep, const int64_t* stride, int64_t n0, int64_t n1, int64_t n2, int64_t states, uint32_t* words,
                     hipStream_t s);
int attn_bwd_launch(AttnParams& p, int dtype, hipStream_t s);
int64_t attn_bwd_workspace(int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hk, int64_t D, int dtype);

}  // namespace fovi
