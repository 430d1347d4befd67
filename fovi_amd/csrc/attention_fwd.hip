// Attention forward: out = softmax(scale q k^T + mask) v, one pass over the states with the running
// maximum and sum of every row (see attention.h for the block layout).
//
//  * tile kernel: a workgroup owns 128 query rows of one key head (the rows of the query heads that share
//    it, in one sequence) and walks the states in tiles that all four waves read from LDS; the next tile is
//    on its way in registers meanwhile.
//  * few-row kernel (fp32, or under a mask): up to 32 rows in all. Every wave of the workgroup has all the rows and its own
//    states: keys straight from memory as matrix operands, values through an LDS tile of the
//    wave's own (only the transposing read needs it), no barrier until the four waves' results join.
//
// Where rows are few, the states are split over workgroups too; a second launch joins the partial
// results in a fixed order.
#include "attention.h"

namespace fovi {

template <typename T, int DP>
struct RowState {
  static constexpr int DT = DP / 32, STEPS = DP / (2 * Chunk<T>::N);
  u32x4 q[STEPS];
  f32x16 o[DT];
  float m, l;                 // the row's maximum so far, or a little less; the lane's share of the sum
  const uint32_t* mrow;
  uint32_t word[2];           // KIND 1: the next blocks' bits
};

// The rows r0 + lane of key head (b, hk): queries as B operands, statistics cleared.
template <typename T, int DP>
__device__ __forceinline__ void init_rows(const AttnParams& p, RowState<T, DP>& st, int64_t b, int hk, int64_t r0) {
  const int l = threadIdx.x & 63;
  const int64_t r = r0 + (l & 31), g = r < p.R ? r / p.Lq : 0, i = r < p.R ? r - g * p.Lq : 0, h = hk * p.G + g;
  const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + i * p.qs[1] + h * p.qs[2];
#pragma unroll
  for (int s = 0; s < RowState<T, DP>::STEPS; ++s) st.q[s] = r < p.R ? load_chunk<T>(q, 2 * s + (l >> 5), p.D) : u32x4{0, 0, 0, 0};
  st.m = kNegInf;
  st.l = 0;
  st.mrow = p.kind ? mask_row(p, b, h, i) : nullptr;
#pragma unroll
  for (int d = 0; d < RowState<T, DP>::DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) st.o[d][e] = 0;
}

// Scores of KB blocks of 32 states (j .. n valid) into probabilities; the running statistics of
// the rows and the outputs' scale follow. Under a mask, pairs that are left out become kLeftOut.
template <typename T, int DP, int KIND, int KB>
__device__ __forceinline__ void softmax_blocks(const AttnParams& p, RowState<T, DP>& st, f32x16 (&s)[KB], Block<T> (&e)[KB],
                                               const uint32_t (&word)[2], int64_t j, int64_t n) {
  const int h = (threadIdx.x & 63) >> 5;
  const float c = unit<KIND>(p);
  const int left = static_cast<int>(n - j < 32 * KB ? n - j : 32 * KB);
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    if (KIND == 1) keep_block(p, word[kb], s[kb]);
    if (KIND == 2) bias_block(p, reinterpret_cast<const float*>(st.mrow), j + kb * 32 + 4 * h, n, s[kb]);
    if (KIND < 2 && left < kb * 32 + 32) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (kb * 32 + 8 * (i / 4) + 4 * h + i % 4 >= left) s[kb][i] = kNegInf;
    }
  }
  float top = st.m;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kb][i]);
  top = fmaxf(top, other_half(top));
  // m is the maximum of the tile that last moved it. It follows only where a row's maximum has grown by
  // more than 8 (in log2), which leaves probabilities up to 256 (no loss in floating point) and saves
  // scaling the outputs after most tiles, where some row's maximum still grows a little.
  if (__any((top - st.m) * c > 8.0f)) {
    const float at = top == kNegInf ? 0.0f : top, keep = exp2_fast((st.m - at) * c);
    st.l *= keep;
#pragma unroll
    for (int d = 0; d < RowState<T, DP>::DT; ++d) st.o[d] *= keep;
    st.m = top;
  }
  const float m = st.m == kNegInf ? 0.0f : st.m;
  float sum = 0;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float x = exp2_below<KIND>(s[kb][i], m, c);
      s[kb][i] = KIND && s[kb][i] == kNegInf ? kLeftOut : x;
    }
    e[kb] = Block<T>(s[kb]);
    sum = e[kb].sum(sum);
  }
  st.l += sum;
}

// Partial results: unscaled outputs [split][key head][row][D], then (maximum, sum) of each.
__device__ __forceinline__ float2* part_stats(const AttnParams& p) {
  return reinterpret_cast<float2*>(p.part + static_cast<int64_t>(p.splits) * p.B * p.Hk * p.R * p.D);
}

__device__ __forceinline__ int64_t stat_at(const AttnParams& p, int64_t b, int hk, int64_t r) {
  return (b * p.H + static_cast<int64_t>(hk) * p.G) * p.Lq + r;      // row (b, head, query) of the statistics
}

// Waves a SIMD shall hold: two (256 registers each) wherever a kernel fits without spilling much; a lone
// wave waits out every latency (bf16, heads of 64, 1024 x 4096 x 192 heads: 602 us with one, 390 with two).
template <typename T> constexpr int tile_waves(int DP, int KIND) {
  return sizeof(T) == 2 ? (KIND ? (DP >= 96 ? 1 : 2) : DP <= 64 ? 3 : 2) : (DP == 128 || (KIND && DP == 96) ? 1 : 2);
}
template <typename T> constexpr int few_waves(int DP, int KIND) {
  return sizeof(T) == 2 ? (DP >= 96 ? 1 : 2) : (DP >= 96 || (KIND && DP == 64) ? 1 : 2);
}

// Bound by the matrix and the vector instructions of a SIMD, which hardly overlap here: of 1024
// rows x 4096 states x 192 bf16 heads of 64 (319 us, 646 TFLOP/s) the matrix unit is busy 35 % of the cycles
// and the vector unit 58 % (an exponential takes as long as two or three other instructions). A loop of the same
// instructions on registers alone takes 250 us; staging the tiles costs most of the rest. Two row blocks a
// wave would stage and read half as much, but leave two waves a SIMD instead of three: 359 us where one
// block takes 347 (52 and 63 us for 384 x 768 x 384). Asynchronous loads into LDS were no way out either: every
// LDS read then waits for all of them. Few rows are bound by memory: 4 rows of 16 heads over 131072 states of 4
// key heads of 128 take 43 us (268 MB, 6.2 TB/s), one row of 128 images over 256 to 5120 states, 6 heads of 64,
// 116 us (528 MB, 4.6 TB/s; a copy of this size reaches 4.9).
template <typename T, int DP, int KIND>
__global__ __launch_bounds__(256, tile_waves<T>(DP, KIND)) void attn_fwd_tile_kernel(AttnParams p) {
  constexpr int LP = DP == 96 ? 128 : DP, KB = sizeof(T) == 2 ? 2 : 1, KT = 32 * KB, DT = DP / 32;
  constexpr int STEPS = RowState<T, DP>::STEPS;
  __shared__ __attribute__((aligned(16))) char tiles[2][2][KT * LP * sizeof(T)];
  __shared__ int bad_tile[2];
  const int64_t all = p.tiles * p.splits * p.B * p.Hk, id = xcd_tile(blockIdx.x, gridDim.x);
  if (id >= all) return;
  const int64_t group = id / p.tiles, bh = group / p.splits, b = bh / p.Hk;
  const int hk = static_cast<int>(bh - b * p.Hk), split = static_cast<int>(group - bh * p.splits);
  const int64_t len = attn_len(p, b), j0 = split * p.chunk, n = len < j0 + p.chunk ? len : j0 + p.chunk;
  if (split && n <= j0) return;                        // (split 0 writes the rows of images without states)
  const int64_t r0 = (id - group * p.tiles) * 128 + (threadIdx.x >> 6) * 32;
  RowState<T, DP> st;
  init_rows<T, DP>(p, st, b, hk, r0);
  const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
  const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];
  Staged<T, LP, KT, 256> kr, vr;
  kr.init(p.ks[1], p.D, threadIdx.x);
  vr.init(p.vs[1], p.D, threadIdx.x);
#pragma unroll
  for (int i = 0; i < 4; ++i) kr.clear(tiles[i >> 1][i & 1], p.D);
  if (KIND && threadIdx.x < 2) bad_tile[threadIdx.x] = -1;
  if (KIND) __syncthreads();
  int at = 0;
  uint32_t word[2] = {0, 0};
  auto words = [&](int64_t j) {                        // (words of whole blocks: bits behind the states are 0)
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) st.word[kb] = j + 32 * kb < n && r0 + (threadIdx.x & 31) < p.R ? st.mrow[j / 32 + kb] : 0;
  };
  auto put = [&](int buf, int tile) {
    kr.store(tiles[buf][0], p.D);
    if (!KIND) vr.clear_tail();
    vr.store(tiles[buf][1], p.D);
    if (KIND && vr.bad()) bad_tile[buf] = tile;
  };
  if (j0 < n) {
    kr.load(k + j0 * p.ks[1], n - j0);
    vr.load(v + j0 * p.vs[1], n - j0);
    if (KIND == 1) words(j0);
    put(0, 0);
  }
  wait_loads();
  for (int64_t j = j0; j < n; j += KT, ++at) {
    const int64_t next = j + KT;
    if (KIND == 1) {
      word[0] = st.word[0];
      word[1] = st.word[1];
      if (next < n) words(next);
    }
    if (next < n) {
      kr.load(k + next * p.ks[1], n - next);
      vr.load(v + next * p.vs[1], n - next);
    }
    __syncthreads();                                   // tile `at` is in LDS, tile at - 1 is done with
    const char* kt = tiles[at & 1][0];
    const char* vt = tiles[at & 1][1];
    // (the last workgroup's waves may have no rows, and no row may read this tile)
    if (r0 < p.R && (KIND != 1 || __any((word[0] | (KB > 1 ? word[1] : 0)) != 0))) {
      f32x16 s[KB] = {};
      Block<T> e[KB];
      Turned<T, LP> va[2][DT];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) row_product<T, LP>(kt + kb * 32 * LP * sizeof(T), st.q, s[kb]);
#pragma unroll
      for (int d = 0; d < DT; ++d) va[0][d].read(vt, 0, d);
      reads_done();
      softmax_blocks<T, DP, KIND, KB>(p, st, s, e, word, j, n);
      if (KIND && bad_tile[at & 1] == at) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) slow_second<T, LP, DT>(vt, kb * 32, s[kb], st.o);
      } else {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          if (kb + 1 < KB) {
#pragma unroll
            for (int d = 0; d < DT; ++d) va[(kb + 1) & 1][d].read(vt, (kb + 1) * 32, d);
            reads_done();
          }
#pragma unroll
          for (int d = 0; d < DT; ++d) st.o[d] = va[kb & 1][d].mma(e[kb], st.o[d]);
        }
      }
    }
    if (next < n) put((at + 1) & 1, at + 1);
  }
  const int lane = threadIdx.x & 63;
  const int64_t r = r0 + (lane & 31);
  const float sum = st.l + other_half(st.l), m = KIND ? st.m : st.m * p.c;
  if (r >= p.R) return;
  if (p.splits > 1) {
    const int64_t row = (split * p.B * p.Hk + bh) * p.R + r;
    if (lane < 32) part_stats(p)[row] = make_float2(m, sum);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        store_run(p.part + row * p.D, d * 32 + 2 * e + 4 * (lane >> 5), p.D, st.o[d][e], st.o[d][e + 1], st.o[d][e + 2],
                  st.o[d][e + 3]);
    return;
  }
  const int64_t g = r / p.Lq, i = r - g * p.Lq, off = b * p.os[0] + i * p.os[1] + (hk * p.G + g) * p.os[2];
  T* out = static_cast<T*>(p.o) + off;
  const float inv = sum == 0 ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int at_d = d * 32 + 2 * e + 4 * (lane >> 5);
      float y[4], rest[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        y[x] = st.o[d][e + x] * inv;
        rest[x] = y[x] - bf16_bits_to_f32(f32_to_bf16_bits(y[x]));
      }
      store_run(out, at_d, p.D, y[0], y[1], y[2], y[3]);
      if (p.rest) store_run(static_cast<T*>(p.rest) + off, at_d, p.D, rest[0], rest[1], rest[2], rest[3]);
    }
  if (p.stats && lane < 32) {
    const int64_t w = stat_at(p, b, hk, r);
    p.stats[w] = m;
    p.stats[p.B * p.H * p.Lq + w] = sum;
  }
}

// Element d of row r (key head (b, hk)) from its sum, maximum and unscaled value.
template <typename T>
__device__ __forceinline__ void put_row(const AttnParams& p, int64_t b, int hk, int64_t r, int d, float value, float m, float sum) {
  const int64_t g = r / p.Lq, i = r - g * p.Lq, off = b * p.os[0] + i * p.os[1] + (hk * p.G + g) * p.os[2] + d;
  const float y = sum == 0 ? 0.0f : value / sum;
  Elem<T>::store(static_cast<T*>(p.o) + off, y);
  if (p.rest) Elem<T>::store(static_cast<T*>(p.rest) + off, y - Elem<T>::load(static_cast<const T*>(p.o) + off));
  if (p.stats && d == 0) {
    const int64_t w = stat_at(p, b, hk, r);
    p.stats[w] = m;
    p.stats[p.B * p.H * p.Lq + w] = sum;
  }
}

// Every key and value is read once, for all rows of its key head. 64 images, 2048 states, 6 heads of 64: 403 MB
// of fp32 in 104 us, 3.9 TB/s, with the products of a whole block of rows however few there are.
template <typename T, int DP, int KIND>
__global__ __launch_bounds__(256, few_waves<T>(DP, KIND)) void attn_fwd_few_kernel(AttnParams p) {
  constexpr int LP = DP == 96 ? 128 : DP, DT = DP / 32, STEPS = RowState<T, DP>::STEPS;
  constexpr int TILE = 32 * LP * static_cast<int>(sizeof(T)), JOIN = 32 * (DP + 1) * 4;
  __shared__ __attribute__((aligned(16))) char lds[4 * (TILE > JOIN ? TILE : JOIN)];
  __shared__ float wm[4][32], wl[4][32];
  const int64_t bh = blockIdx.x, b = bh / p.Hk;
  const int hk = static_cast<int>(bh - b * p.Hk), split = blockIdx.y, l = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t len = attn_len(p, b), j0 = split * p.chunk, n = len < j0 + p.chunk ? len : j0 + p.chunk;
  if (split && n <= j0) return;
  RowState<T, DP> st;
  init_rows<T, DP>(p, st, b, hk, 0);
  const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
  const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];
  char* vt = lds + w * TILE;
  u32x4 ka[STEPS];
  Staged<T, LP, 32, 64> vr;
  vr.init(p.vs[1], p.D, l);
  vr.clear(vt, p.D);
  uint32_t word[2] = {};
  auto fetch = [&](int64_t j) {
    if (KIND == 1) st.word[0] = (l & 31) < p.R ? st.mrow[j / 32] : 0;
    const T* row = k + (j + (l & 31)) * p.ks[1];
#pragma unroll
    for (int t = 0; t < STEPS; ++t)
      ka[t] = j + (l & 31) < n ? load_chunk<T>(row, 2 * t + (l >> 5), p.D) : u32x4{0, 0, 0, 0};
    vr.load(v + j * p.vs[1], n - j);
  };
  wait_loads();
  if (j0 + 32 * w < n) fetch(j0 + 32 * w);
  for (int64_t j = j0 + 32 * w; j < n; j += 128) {
    f32x16 s[1] = {};
    Block<T> e[1];
    Turned<T, LP> va[DT];
#pragma unroll
    for (int t = 0; t < STEPS; ++t) s[0] = mma_step(T(), ka[t], st.q[t], s[0]);
    if (!KIND) vr.clear_tail();
    vr.store(vt, p.D);                     // the wave's own tile: LDS serves a wave's accesses in order
    __builtin_amdgcn_wave_barrier();
    const bool bad = KIND && __any(vr.bad());
    if (KIND == 1) word[0] = st.word[0];
    if (j + 128 < n) fetch(j + 128);
#pragma unroll
    for (int d = 0; d < DT; ++d) va[d].read(vt, 0, d);
    reads_done();
    softmax_blocks<T, DP, KIND, 1>(p, st, s, e, word, j, n);
    if (bad) {
      slow_second<T, LP, DT>(vt, 0, s[0], st.o);
    } else {
#pragma unroll
      for (int d = 0; d < DT; ++d) st.o[d] = va[d].mma(e[0], st.o[d]);
    }
    __builtin_amdgcn_wave_barrier();
  }
  float* join = reinterpret_cast<float*>(lds) + w * (JOIN / 4);
  __syncthreads();
  const float sum = st.l + other_half(st.l);
  if (l < 32) { wm[w][l] = KIND ? st.m : st.m * p.c; wl[w][l] = sum; }
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) join[(l & 31) * (DP + 1) + d * 32 + 8 * (e / 4) + 4 * (l >> 5) + e % 4] = st.o[d][e];
  __syncthreads();
  const int rows = static_cast<int>(p.R);
  for (int x = threadIdx.x; x < rows * p.D; x += 256) {
    const int r = x / p.D, d = x - r * p.D;
    const float m = fmaxf(fmaxf(wm[0][r], wm[1][r]), fmaxf(wm[2][r], wm[3][r])), at = m == kNegInf ? 0.0f : m;
    float value = 0, total = 0;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const float f = exp2_fast((wm[y][r] - at) * (KIND == 2 ? kLog2e : 1.0f));
      total = fmaf(wl[y][r], f, total);
      value = fmaf(reinterpret_cast<const float*>(lds)[y * (JOIN / 4) + r * (DP + 1) + d], f, value);
    }
    const int64_t row = r;
    if (p.splits > 1) {
      const int64_t at_row = (split * p.B * p.Hk + bh) * p.R + row;
      p.part[at_row * p.D + d] = value;
      if (d == 0) part_stats(p)[at_row] = make_float2(m, total);
    } else {
      put_row<T>(p, b, hk, row, d, value, m, total);
    }
  }
}

// The partial results of a row's splits added up in a fixed order: 32 lanes a row and group, four
// elements each; GROUPS 8 (one row a workgroup) where there are many splits, whose loads would
// otherwise follow one another (256 splits of 16 x 4 rows: 191 us by one wave a row).
template <typename T, int GROUPS>
__global__ __launch_bounds__(256) void attn_fwd_join_kernel(AttnParams p) {
  __shared__ float sh[GROUPS][32][6];
  const int64_t rows = p.B * p.Hk * p.R, x = static_cast<int64_t>(blockIdx.x) * (8 / GROUPS) + (GROUPS == 1 ? threadIdx.x >> 5 : 0);
  if (x >= rows) return;
  const int d = (threadIdx.x & 31) * 4, group = GROUPS == 1 ? 0 : threadIdx.x >> 5;
  const int64_t bh = x / p.R, b = bh / p.Hk, len = attn_len(p, b);
  int used = static_cast<int>((len + p.chunk - 1) / p.chunk);
  if (used < 1) used = 1;
  const float2* stats = part_stats(p) + x;
  const float c = p.kind == FOVI_MASK_BIAS ? kLog2e : 1.0f;      // the maxima's unit
  float m = kNegInf, sum = 0;
  f32x4 y = {};
#pragma unroll 4
  for (int s = group; s < used; s += GROUPS) {
    const float2 ml = stats[s * rows];
    const f32x4 v = d < p.D ? *reinterpret_cast<const f32x4*>(p.part + (s * rows + x) * p.D + d) : f32x4{};
    const float top = fmaxf(m, ml.x), at = top == kNegInf ? 0.0f : top, old = exp2_fast((m - at) * c), f = exp2_fast((ml.x - at) * c);
    sum = fmaf(sum, old, ml.y * f);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = fmaf(y[e], old, v[e] * f);
    m = top;
  }
  if (GROUPS > 1) {
    float* mine = sh[group][threadIdx.x & 31];
    mine[0] = m; mine[1] = sum;
#pragma unroll
    for (int e = 0; e < 4; ++e) mine[2 + e] = y[e];
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int g = 1; g < GROUPS; ++g) {
      const float* o = sh[g][threadIdx.x & 31];
      const float top = fmaxf(m, o[0]), at = top == kNegInf ? 0.0f : top, old = exp2_fast((m - at) * c), f = exp2_fast((o[0] - at) * c);
      sum = fmaf(sum, old, o[1] * f);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = fmaf(y[e], old, o[2 + e] * f);
      m = top;
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (d + e < p.D) put_row<T>(p, b, static_cast<int>(bh - b * p.Hk), x - bh * p.R, d + e, y[e], m, sum);
}

// Bytes of a mask into bits, a word a thread.
__global__ __launch_bounds__(256) void attn_pack_kernel(const uint8_t* keep, int64_t s0, int64_t s1, int64_t s2, int64_t s3, int64_t n1,
                                                        int64_t n2, int64_t states, int64_t per, int64_t all, uint32_t* words) {
  const int64_t x = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (x >= all) return;
  const int64_t row = x / per, w = x - row * per, i2 = row % n2, i1 = row / n2 % n1, i0 = row / n2 / n1;
  const uint8_t* m = keep + i0 * s0 + i1 * s1 + i2 * s2 + w * 32 * s3;
  const int n = static_cast<int>(states - w * 32 < 32 ? states - w * 32 : 32);
  uint32_t bits = 0;
  if (s3 == 1 && n == 32) {
    uint32_t b[8];
    __builtin_memcpy(b, m, 32);
#pragma unroll
    for (int i = 0; i < 32; ++i) bits |= ((b[i >> 2] >> (8 * (i & 3))) & 0xff ? 1u : 0u) << i;
  } else {
    for (int i = 0; i < n; ++i) bits |= (m[i * s3] ? 1u : 0u) << i;
  }
  words[x] = bits;
}

int attn_pack_launch(const void* keep, const int64_t* stride, int64_t n0, int64_t n1, int64_t n2, int64_t states, uint32_t* words,
                     hipStream_t s) {
  const int64_t per = (states + 31) / 32, all = n0 * n1 * n2 * per;
  if (all == 0) return 0;
  attn_pack_kernel<<<static_cast<unsigned>((all + 255) / 256), 256, 0, s>>>(static_cast<const uint8_t*>(keep), stride[0], stride[1],
                                                                           stride[2], stride[3], n1, n2, states, per, all, words);
  return check_launch("fovi_attention_pack_mask");
}

// How a call is laid out. Few rows: every workgroup has them all. Else tiles of 128 rows.
struct FwdPlan {
  bool few;
  int splits;
  int64_t tiles, chunk;
};

// Workgroups of the few-row kernel on a compute unit: its waves a SIMD.
static int few_waves_at(int dtype, int64_t D, bool mask) {
  const int dp = D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128;
  return dtype == FOVI_BF16 ? few_waves<uint16_t>(dp, mask) : few_waves<float>(dp, mask);
}

static FwdPlan fwd_plan(int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hk, int64_t D, int dtype, bool mask) {
  FwdPlan f;
  const int64_t R = H / Hk * Lq;
  // Few rows of fp32, whose products are slow (four waves share them: 64 x 6 heads of 64, one row over 2048
  // states: 104 us and a join of 5, by tiles 168), or under a mask (bf16, the same sizes: 40 + 5, by tiles 61).
  // Plain bf16 rows go by tiles, whose one wave keeps up with memory (128 images, 256 to 5120 states: 117 us, 125 +
  // 5 here; 131072 states, 4 key heads of 128: 44, 51 here).
  f.few = R <= 32 && (dtype == FOVI_F32 || mask);
  f.tiles = f.few ? 1 : (R + 127) / 128;
  // The states are split until the card is full, few rows of 64 key heads and images or more twice, since lengths
  // differ then and a last round of workgroups costs less (32 images of 256 to 5120 states, 6 heads of 64, fp32: 85 us,
  // filled once 122; all of 5120: 115 and 139; but 8 images of 9000 states and 8 heads: 77 and 72). Below that once
  // (4 images of 9000 states, 8 heads of 64, fp32: 44 us, twice 47; 131072 states, 4 heads of 128: 126 and 142). Parts
  // are still worth a workgroup's start and the join: 512 states for few rows (where a
  // wave a SIMD is all there is, 9000 fp32 states and 32 heads of 80: 8 parts 57 us, 4 98), 128 for tiles (515
  // states, 32 groups, fp32 under a mask: parts of 128 14 us, of 256 23; the join 5 each).
  const int waves = f.few ? few_waves_at(dtype, D, mask) : 2;
  const int64_t groups = B * Hk * f.tiles, least = f.few ? 512 : 128, want = f.few ? (groups < 64 ? 256 : 512) * waves : 512;
  int64_t splits = groups > 0 ? want / groups : 1;
  if (splits > (Lk + least - 1) / least) splits = (Lk + least - 1) / least;
  if (splits > 1024) splits = 1024;
  if (splits < 1) splits = 1;
  f.chunk = ((Lk + splits - 1) / splits + 127) / 128 * 128;
  if (f.chunk < 128) f.chunk = 128;
  f.splits = static_cast<int>(Lk ? (Lk + f.chunk - 1) / f.chunk : 1);
  return f;
}

int64_t attn_fwd_workspace(int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hk, int64_t D, int dtype) {
  int64_t most = 0;
  for (const bool mask : {false, true}) {
    const FwdPlan f = fwd_plan(B, Lq, Lk, H, Hk, D, dtype, mask);
    const int64_t need = f.splits > 1 ? f.splits * B * H * Lq * (D + 2) * 4 : 0;
    if (need > most) most = need;
  }
  return most;
}

template <typename T, int DP, int KIND>
static void fwd_launch(const AttnParams& p, const FwdPlan& f, hipStream_t s) {
  const int64_t all = p.B * p.Hk * f.tiles;
  if (!launch_fits(f.few ? all : (all * f.splits + 7) / 8 * 8, 256)) return;
  if (f.few) {
    const dim3 grid(static_cast<unsigned>(all), static_cast<unsigned>(f.splits));
    if constexpr (sizeof(T) == 4 || KIND != 0) attn_fwd_few_kernel<T, DP, KIND><<<grid, 256, 0, s>>>(p);
  } else {
    const unsigned grid = static_cast<unsigned>((all * f.splits + 7) / 8 * 8);
    attn_fwd_tile_kernel<T, DP, KIND><<<grid, 256, 0, s>>>(p);
  }
}

template <typename T, int KIND>
static void fwd_heads(const AttnParams& p, const FwdPlan& f, hipStream_t s) {
  if (p.D <= 32) fwd_launch<T, 32, KIND>(p, f, s);
  else if (p.D <= 64) fwd_launch<T, 64, KIND>(p, f, s);
  else if (p.D <= 96) fwd_launch<T, 96, KIND>(p, f, s);
  else fwd_launch<T, 128, KIND>(p, f, s);
}

template <typename T>
static int fwd_type(AttnParams& p, hipStream_t s) {
  const FwdPlan f = fwd_plan(p.B, p.Lq, p.Lk, p.H, p.Hk, p.D, sizeof(T) == 2 ? FOVI_BF16 : FOVI_F32, p.kind != 0);
  p.splits = f.splits;
  p.chunk = f.chunk;
  p.tiles = f.tiles;
  if (p.kind == FOVI_MASK_NONE) fwd_heads<T, 0>(p, f, s);
  else if (p.kind == FOVI_MASK_KEEP) fwd_heads<T, 1>(p, f, s);
  else fwd_heads<T, 2>(p, f, s);
  if (check_launch("fovi_attention_fwd")) return 1;
  if (f.splits > 1) {
    const int64_t rows = p.B * p.Hk * p.R;
    if (!launch_fits(f.splits >= 16 ? rows : (rows + 7) / 8, 256)) return check_launch("fovi_attention_fwd");
    if (f.splits >= 16) attn_fwd_join_kernel<T, 8><<<static_cast<unsigned>(rows), 256, 0, s>>>(p);
    else attn_fwd_join_kernel<T, 1><<<static_cast<unsigned>((rows + 7) / 8), 256, 0, s>>>(p);
    return check_launch("fovi_attention_fwd");
  }
  return 0;
}

int attn_fwd_launch(AttnParams& p, int dtype, hipStream_t s) {
  return dtype == FOVI_BF16 ? fwd_type<uint16_t>(p, s) : fwd_type<float>(p, s);
}

}  // namespace fovi
