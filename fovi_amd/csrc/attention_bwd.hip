// Attention backward (see attention.h for the block layout).
//
//   p_ij = exp(s_ij - max_i) / sum_i, ds_ij = p_ij (do_i.v_j - delta_i), delta_i = do_i.o_i
//   dq_i = scale sum_j ds_ij k_j, dk_j = scale sum_i ds_ij q_i, dv_j = sum_i p_ij do_i
//
// Two launches: dq, whose workgroups own query rows and walk the states (and leave delta behind); dk
// and dv, whose workgroups own states and walk the query rows of all heads that share the key head.
// The scores are formed twice (7 products instead of 5), and in return every gradient is summed by
// one workgroup in a fixed order, without atomics and without a score matrix in memory. Where the
// owned axis is short, the walked one is split over workgroups and the partial sums join in a third.
#include "attention.h"

namespace fovi {

// What a row's probabilities need: exp2((t - shift) unit) * factor. Without a mask the log of the sum goes
// into the shift (factor 1). A row that keeps nothing has shift +inf: probabilities 0. A row whose sum is NaN (it
// keeps a NaN, or a score of +inf, which is its maximum then) has shift NaN, so that its gradients are NaN as well.
struct RowStat { float shift, factor, delta; };
template <int KIND>
__device__ __forceinline__ RowStat row_stat(float m, float sum, float delta) {
  const float shift = KIND ? m + 0.0f * sum : m + log2f(sum);       // (0 * sum: 0, or NaN)
  return {sum == 0 ? __builtin_inff() : shift, KIND && sum != 0 ? 1.0f / sum : KIND ? 0.0f : 1.0f, delta};
}

// Probability and score gradient of one pair, dp = do.v - delta (the product starts from -delta). Under a mask t is
// the masked score, and left-out pairs become kLeftOut.
template <int KIND>
__device__ __forceinline__ void pair_grad(float t, float c, float shift, float factor, float dp, float& e, float& ds) {
  if (KIND) {
    const bool out = t == kNegInf || shift == __builtin_inff();
    e = exp2_fast(KIND == 2 ? (t - shift) * kLog2e : t - shift) * factor;
    ds = out ? kLeftOut : e * dp;
    e = out ? kLeftOut : e;
  } else {
    e = exp2_fast(fmaf(t, c, -shift));
    ds = e * dp;
  }
}

// Waves a SIMD shall hold: two wherever a kernel fits 256 registers without spilling much.
template <typename T> constexpr int dq_waves(int DP, int KIND) {
  return sizeof(T) == 2 ? (KIND && DP == 128 ? 1 : DP == 64 && !KIND ? 3 : 2) : DP >= 96 ? 1 : 2;
}
template <typename T> constexpr int dkv_waves(int DP, int KIND) {
  return sizeof(T) == 2 ? (DP >= 96 ? 1 : 2) : DP >= 64 ? 1 : 2;
}

// As the forward's tile kernel, with three products a pair: 1024 rows x 4096 states x 192 bf16 heads of 64 in
// 366 us (845 TFLOP/s), matrix unit busy 48 % of the cycles, vector unit 61 % (some of both at once).
template <typename T, int DP, int KIND>
__global__ __launch_bounds__(256, dq_waves<T>(DP, KIND)) void attn_dq_kernel(AttnParams p) {
  constexpr int LP = DP == 96 ? 128 : DP, KB = sizeof(T) == 2 ? 2 : 1, KT = 32 * KB, DT = DP / 32, STEPS = DP / (2 * Chunk<T>::N);
  __shared__ __attribute__((aligned(16))) char tiles[2][2][KT * LP * sizeof(T)];
  __shared__ int bad_tile[2];
  const int64_t all = p.tiles * p.splits * p.B * p.Hk, id = xcd_tile(blockIdx.x, gridDim.x);
  if (id >= all) return;
  const int64_t group = id / p.tiles, bh = group / p.splits, b = bh / p.Hk;
  const int hk = static_cast<int>(bh - b * p.Hk), split = static_cast<int>(group - bh * p.splits), l = threadIdx.x & 63;
  const int64_t len = attn_len(p, b), j0 = split * p.chunk, n = len < j0 + p.chunk ? len : j0 + p.chunk;
  if (split && n <= j0) return;
  const int64_t r0 = (id - group * p.tiles) * 128 + (threadIdx.x >> 6) * 32;
  u32x4 q[STEPS], g[STEPS];
  f32x16 dq[DT] = {};
  constexpr bool START = sizeof(T) == 2 && DP == 32;   // -delta as a block of its own, where registers allow
  // Heads of 96 and 128: operands are read as they are needed. Two waves a SIMD that way (229 us for 8 x 1024 x
  // 2048 and 16 heads of 128) beat one with its reads in batches (300).
  constexpr bool LATE = DP > 64;
  f32x16 start;
  uint32_t word[2] = {}, coming[2] = {};       // KIND 1: the blocks' bits, and the next tile's
  const int64_t r = r0 + (l & 31);
  const int64_t gr = r < p.R ? r / p.Lq : 0, i = r < p.R ? r - gr * p.Lq : 0, h = hk * p.G + gr;
  const T* qr = static_cast<const T*>(p.q) + b * p.qs[0] + i * p.qs[1] + h * p.qs[2];
  const T* gg = static_cast<const T*>(p.dout) + b * p.dos[0] + i * p.dos[1] + h * p.dos[2];
  // delta = do.o, o before its rounding; half of the elements a lane
  const int64_t off = b * p.os[0] + i * p.os[1] + h * p.os[2];
  float delta = 0;
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    q[s] = load_chunk<T>(qr, 2 * s + (l >> 5), r < p.R ? p.D : 0);
    g[s] = load_chunk<T>(gg, 2 * s + (l >> 5), r < p.R ? p.D : 0);
    const u32x4 o = load_chunk<T>(static_cast<const T*>(p.o) + off, 2 * s + (l >> 5), p.D);
    const u32x4 rest = p.rest ? load_chunk<T>(static_cast<const T*>(p.rest) + off, 2 * s + (l >> 5), p.D) : u32x4{0, 0, 0, 0};
    T ge[Chunk<T>::N], oe[Chunk<T>::N], re[Chunk<T>::N];
    __builtin_memcpy(ge, &g[s], 16);
    __builtin_memcpy(oe, &o, 16);
    __builtin_memcpy(re, &rest, 16);
#pragma unroll
    for (int e = 0; e < Chunk<T>::N; ++e) delta = fmaf(Elem<T>::load(ge + e), Elem<T>::load(oe + e) + Elem<T>::load(re + e), delta);
  }
  delta += other_half(delta);
  const int64_t at_row = (b * p.H + h) * p.Lq + i;
  if (split == 0 && l < 32 && r < p.R) p.delta[at_row] = delta;
  const RowStat st = row_stat<KIND>(p.stats[at_row], p.stats[p.B * p.H * p.Lq + at_row], delta);
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (START) start[e] = -st.delta;
  const uint32_t* mrow = KIND ? mask_row(p, b, h, i) : nullptr;
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
  auto words = [&](int64_t j) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) coming[kb] = j + 32 * kb < n && r < p.R ? mrow[j / 32 + kb] : 0;
  };
  auto put = [&](int buf, int tile) {
    kr.store(tiles[buf][0], p.D);
    vr.store(tiles[buf][1], p.D);
    if (KIND && kr.bad()) bad_tile[buf] = tile;
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
      word[0] = coming[0];
      word[1] = coming[1];
      if (next < n) words(next);
    }
    if (next < n) {
      kr.load(k + next * p.ks[1], n - next);
      vr.load(v + next * p.vs[1], n - next);
    }
    __syncthreads();
    const char* kt = tiles[at & 1][0];
    const char* vt = tiles[at & 1][1];
    const int left = static_cast<int>(n - j < KT ? n - j : KT);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      if (KIND == 1 && !__any(word[kb] != 0)) continue;      // no row reads these states
      f32x16 s = {}, dp = {};
      if (START) dp = start;
      row_products<T, LP, (LATE ? 1 : DP == 64 ? 2 : STEPS < 4 ? STEPS : 4), !LATE>(
          kt + kb * 32 * LP * sizeof(T), vt + kb * 32 * LP * sizeof(T), q, g, s, dp);
      Turned<T, LP> ka[DT];
#pragma unroll
      for (int d = 0; d < DT; ++d)
        if (!LATE) ka[d].read(kt, kb * 32, d);
      if (!LATE) reads_done();
      if (KIND == 1) keep_block(p, word[kb], s);
      if (KIND == 2) bias_block(p, reinterpret_cast<const float*>(mrow), j + kb * 32 + 4 * (l >> 5), n, s);
      if (KIND < 2 && left < kb * 32 + 32) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (kb * 32 + 8 * (i / 4) + 4 * (l >> 5) + i % 4 >= left) s[i] = kNegInf;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float e, ds;
        pair_grad<KIND>(s[i], p.c, st.shift, st.factor, START ? dp[i] : dp[i] - st.delta, e, ds);
        s[i] = ds;
      }
      if (KIND && bad_tile[at & 1] == at) {
        slow_second<T, LP, DT>(kt, kb * 32, s, dq);
      } else {
        const Block<T> ds(s);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          if (LATE) ka[d].read(kt, kb * 32, d);
          dq[d] = ka[d].mma(ds, dq[d]);
        }
      }
    }
    if (next < n) put((at + 1) & 1, at + 1);
  }
  if (r >= p.R) return;
  T* out = static_cast<T*>(p.dq) + b * p.dqs[0] + i * p.dqs[1] + (hk * p.G + gr) * p.dqs[2];
  float* part = p.part + ((split * p.B * p.Hk + bh) * p.R + r) * p.D;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int at_d = d * 32 + 2 * e + 4 * (l >> 5);
      const float a = dq[d][e] * p.scale, bb = dq[d][e + 1] * p.scale, c = dq[d][e + 2] * p.scale, f = dq[d][e + 3] * p.scale;
      if (p.splits > 1) store_run(part, at_d, p.D, a, bb, c, f);
      else store_run(out, at_d, p.D, a, bb, c, f);
    }
}

// Blocks of 32 rows in a tile of the dk, dv kernel.
template <typename T> constexpr int dkv_blocks(int DP) { return sizeof(T) == 2 && DP <= 64 ? 2 : 1; }

// Four products a pair: the same sizes in 560 us (736 TFLOP/s), matrix unit busy 40 % of the cycles and vector
// unit 40 %, a fifth of them neither. Keys, values and both gradients of 32 states hold 160 registers a lane for heads of 64, so that only
// two waves share a SIMD and not every latency is hidden (lone waves, for wider heads, hide less).
template <typename T, int DP, int KIND>
__global__ __launch_bounds__(256, dkv_waves<T>(DP, KIND)) void attn_dkv_kernel(AttnParams p) {
  constexpr int LP = DP == 96 ? 128 : DP, DT = DP / 32, STEPS = DP / (2 * Chunk<T>::N), RB = dkv_blocks<T>(DP), RT = 32 * RB;
  __shared__ __attribute__((aligned(16))) char tiles[2][2][RT * LP * sizeof(T)];
  __shared__ __attribute__((aligned(16))) float stats[2][3][RT];
  __shared__ int bad_tile[2][2];
  __shared__ __attribute__((aligned(16))) uint32_t bits[2][4][KIND == 1 ? RT : 4];     // [wave][row]: its 32 states
  const int64_t all = p.tiles * p.splits * p.B * p.Hk, id = xcd_tile(blockIdx.x, gridDim.x);
  if (id >= all) return;
  const int64_t group = id / p.tiles, bh = group / p.splits, b = bh / p.Hk;
  const int hk = static_cast<int>(bh - b * p.Hk), split = static_cast<int>(group - bh * p.splits), l = threadIdx.x & 63;
  const int64_t n = attn_len(p, b), w0 = (id - group * p.tiles) * 128, j = w0 + (threadIdx.x >> 6) * 32 + (l & 31);
  const T* kp = static_cast<const T*>(p.k) + b * p.ks[0] + j * p.ks[1] + hk * p.ks[2];
  const T* vp = static_cast<const T*>(p.v) + b * p.vs[0] + j * p.vs[1] + hk * p.vs[2];
  u32x4 k[STEPS], v[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    k[s] = load_chunk<T>(kp, 2 * s + (l >> 5), j < n ? p.D : 0);
    v[s] = load_chunk<T>(vp, 2 * s + (l >> 5), j < n ? p.D : 0);
  }
  f32x16 dk[DT] = {}, dv[DT] = {};
  // tiles of RT rows, head by head; split s walks tiles s * chunk .. of the p.G * per there are (none without
  // queries: then no row, statistic or mask has an element, and the gradients below are zeros)
  const int per = p.Lq > 0 ? static_cast<int>((p.Lq + RT - 1) / RT) : 1;
  const int64_t first = split * p.chunk, end = static_cast<int64_t>(per) * p.G;
  const int count = w0 >= n || p.Lq == 0 ? 0 : static_cast<int>(end < first + p.chunk ? end - first : p.chunk);
  Staged<T, LP, RT, 256> qr, gr;
  qr.init(p.qs[1], p.D, threadIdx.x);
  gr.init(p.dos[1], p.D, threadIdx.x);
#pragma unroll
  for (int i = 0; i < 4; ++i) qr.clear(tiles[i >> 1][i & 1], p.D);
  float m = 0, sum = 0, delta = 0;                 // raw: nothing waits for them before the tile is stored
  uint32_t word = 0;
  if (KIND && threadIdx.x < 4) bad_tile[threadIdx.x >> 1][threadIdx.x & 1] = -1;
  if (KIND) __syncthreads();
  int h = hk * p.G + static_cast<int>(first / per), i0 = static_cast<int>(first % per) * RT;      // the next tile to fetch
  // the next tile's rows: pointers move along, a new head sets them anew
  const T *qp, *gp;
  const float* sp;
  const int64_t sums = p.B * p.H * p.Lq;
  auto rewind = [&]() {
    qp = static_cast<const T*>(p.q) + b * p.qs[0] + i0 * p.qs[1] + h * p.qs[2];
    gp = static_cast<const T*>(p.dout) + b * p.dos[0] + i0 * p.dos[1] + h * p.dos[2];
    sp = p.stats + (b * p.H + h) * p.Lq + i0;
  };
  auto fetch = [&]() {
    const int left = static_cast<int>(p.Lq - i0 < RT ? p.Lq - i0 : RT);
    qr.load(qp, left);
    gr.load(gp, left);
    if (threadIdx.x < RT) {
      const bool in = static_cast<int>(threadIdx.x) < left;
      const float* at = sp + (in ? threadIdx.x : 0);
      m = at[0];
      sum = in ? at[sums] : 0.0f;
      delta = p.delta[at - p.stats];
    }
    if (KIND == 1) {
      const int r = threadIdx.x % RT, w = threadIdx.x / RT;
      word = w < 4 && r < left && w0 + 32 * w < p.Lk ? mask_row(p, b, h, i0 + r)[w0 / 32 + w] : 0;
    }
  };
  auto put = [&](int buf, int tile) {
    qr.store(tiles[buf][0], p.D);
    if (!KIND) gr.clear_tail();
    gr.store(tiles[buf][1], p.D);
    if (threadIdx.x < RT) {
      const RowStat sr = row_stat<KIND>(m, sum, sum == 0 ? 0.0f : delta);
      stats[buf][0][threadIdx.x] = sr.shift;
      if (KIND) stats[buf][1][threadIdx.x] = sr.factor;
      stats[buf][2][threadIdx.x] = -sr.delta;
    }
    if (KIND == 1 && threadIdx.x / RT < 4) bits[buf][threadIdx.x / RT][threadIdx.x % RT] = word;
    if (KIND && qr.bad()) bad_tile[buf][0] = tile;
    if (KIND && gr.bad()) bad_tile[buf][1] = tile;
  };
  rewind();
  if (count > 0) {
    fetch();
    put(0, 0);
  }
  wait_loads();
  for (int at = 0; at < count; ++at) {
    const int h_at = h, i_at = i0;
    i0 += RT;
    qp += RT * p.qs[1];
    gp += RT * p.dos[1];
    sp += RT;
    if (i0 >= p.Lq) {
      i0 = 0;
      ++h;
      rewind();
    }
    if (at + 1 < count) fetch();
    __syncthreads();
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const char* qt = tiles[at & 1][0] + rb * 32 * LP * sizeof(T);
      const char* gt = tiles[at & 1][1] + rb * 32 * LP * sizeof(T);
      uint32_t keep = 0;                  // KIND 1: the lane's 16 pairs
      if (KIND == 1) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(&bits[at & 1][threadIdx.x >> 6][rb * 32 + 2 * i + 4 * (l >> 5)]);
#pragma unroll
          for (int y = 0; y < 4; ++y) keep |= ((w[y] >> (l & 31)) & 1u) << (i + y);
        }
        if (j >= n) keep = 0;
        if (!__any(keep != 0)) continue;  // no pair of the block
      }
      f32x16 s = {}, dp;
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4 start = *reinterpret_cast<const f32x4*>(&stats[at & 1][2][rb * 32 + 2 * i + 4 * (l >> 5)]);
#pragma unroll
        for (int y = 0; y < 4; ++y) dp[i + y] = start[y];
      }
      row_products<T, LP, (STEPS < 4 ? STEPS : 4), true>(qt, gt, k, v, s, dp);
      Turned<T, LP> ga[DT], qa[DT];
#pragma unroll
      for (int d = 0; d < DT; ++d) ga[d].read(gt, 0, d);
      reads_done();
      if (KIND == 1) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = keep & (1u << i) ? s[i] * p.c : kNegInf;
      }
      if (KIND == 2)
        bias_column(p, reinterpret_cast<const float*>(mask_row(p, b, h_at, 0)) + (j < n ? j : 0) * p.ms[3], i_at + rb * 32 + 4 * (l >> 5),
                    j < n ? p.Lq : 0, s);
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int r = rb * 32 + 2 * i + 4 * (l >> 5);
        const f32x4 shift = *reinterpret_cast<const f32x4*>(&stats[at & 1][0][r]);
        f32x4 factor;
        if (KIND) factor = *reinterpret_cast<const f32x4*>(&stats[at & 1][1][r]);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          float e, ds;
          pair_grad<KIND>(s[i + y], p.c, shift[y], KIND ? factor[y] : 1.0f, dp[i + y], e, ds);
          s[i + y] = e;
          dp[i + y] = ds;
        }
      }
      if (KIND && bad_tile[at & 1][1] == at) {
        slow_second<T, LP, DT>(gt, 0, s, dv);
      } else {
        const Block<T> e(s);
#pragma unroll
        for (int d = 0; d < DT; ++d)
          if (!KIND) qa[d].read(qt, 0, d);
        reads_done();
#pragma unroll
        for (int d = 0; d < DT; ++d) dv[d] = ga[d].mma(e, dv[d]);
      }
      if (KIND && bad_tile[at & 1][0] == at) {
        slow_second<T, LP, DT>(qt, 0, dp, dk);
      } else {
        const Block<T> ds(dp);
        if (KIND) {
#pragma unroll
          for (int d = 0; d < DT; ++d) qa[d].read(qt, 0, d);
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) dk[d] = qa[d].mma(ds, dk[d]);
      }
    }
    if (at + 1 < count) put((at + 1) & 1, at + 1);
  }
  if (j >= p.Lk) return;
  T* dko = static_cast<T*>(p.dk) + b * p.dks[0] + j * p.dks[1] + hk * p.dks[2];
  T* dvo = static_cast<T*>(p.dv) + b * p.dvs[0] + j * p.dvs[1] + hk * p.dvs[2];
  float* part = p.part_k + ((split * p.B * p.Hk + bh) * p.Lk + j) * 2 * p.D;
  const float keep = j < n ? 1.0f : 0.0f;          // (columns behind the length never met a value: 0 or NaN)
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int at_d = d * 32 + 2 * e + 4 * (l >> 5);
      float a[4], c[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        a[y] = keep != 0 ? dk[d][e + y] * p.scale : 0.0f;
        c[y] = keep != 0 ? dv[d][e + y] : 0.0f;
      }
      if (p.splits > 1) {
        store_run(part, at_d, p.D, a[0], a[1], a[2], a[3]);
        store_run(part + p.D, at_d, p.D, c[0], c[1], c[2], c[3]);
      } else {
        store_run(dko, at_d, p.D, a[0], a[1], a[2], a[3]);
        store_run(dvo, at_d, p.D, c[0], c[1], c[2], c[3]);
      }
    }
}

// Partial sums added up in the order of the splits, four elements a thread: dq's (where it was split),
// then those of dk and dv. p.splits and p.chunk are dq's.
template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_join_kernel(AttnParams p) {
  const int per = p.D / 4;
  const int64_t q_all = p.splits > 1 ? p.B * p.Hk * p.R * per : 0, k_all = p.k_splits > 1 ? p.B * p.Hk * p.Lk * 2 * per : 0;
  int64_t x = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  f32x4 sum = {};
  if (x < q_all) {
    const int64_t rows = p.B * p.Hk * p.R, row = x / per, d = (x - row * per) * 4, bh = row / p.R, r = row - bh * p.R, b = bh / p.Hk, g = r / p.Lq;
    int64_t used = (attn_len(p, b) + p.chunk - 1) / p.chunk;
    if (used < 1) used = 1;
    for (int64_t s = 0; s < used; ++s) sum += *reinterpret_cast<const f32x4*>(p.part + (s * rows + row) * p.D + d);
    T* out = static_cast<T*>(p.dq) + b * p.dqs[0] + (r - g * p.Lq) * p.dqs[1] + ((bh - b * p.Hk) * p.G + g) * p.dqs[2];
    store_run(out, static_cast<int>(d), p.D, sum[0], sum[1], sum[2], sum[3]);
    return;
  }
  x -= q_all;
  if (x >= k_all) return;
  const int64_t rows = p.B * p.Hk * p.Lk, row = x / (2 * per), y = x - row * 2 * per, d = y % per * 4, bh = row / p.Lk, j = row - bh * p.Lk, b = bh / p.Hk;
  for (int64_t s = 0; s < p.k_splits; ++s) sum += *reinterpret_cast<const f32x4*>(p.part_k + (s * rows + row) * 2 * p.D + y * 4);
  T* out = y >= per ? static_cast<T*>(p.dv) + b * p.dvs[0] + j * p.dvs[1] + (bh - b * p.Hk) * p.dvs[2]
                    : static_cast<T*>(p.dk) + b * p.dks[0] + j * p.dks[1] + (bh - b * p.Hk) * p.dks[2];
  store_run(out, static_cast<int>(d), p.D, sum[0], sum[1], sum[2], sum[3]);
}

struct BwdPlan {
  int q_splits, k_splits;
  int64_t q_tiles, q_chunk, k_tiles, k_chunk;
};

static int64_t dkv_tile(int64_t D, int dtype) { return 32 * (dtype == FOVI_BF16 && D <= 64 ? 2 : 1); }

static BwdPlan bwd_plan(int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hk, int64_t D, int dtype) {
  BwdPlan f;
  const int64_t R = H / Hk * Lq;
  f.q_tiles = (R + 127) / 128;
  f.k_tiles = (Lk + 127) / 128;
  // splits for two workgroups a compute unit, each with at least 128 states or 64 rows to walk (fp32 under a
  // mask, 8 x 77 x 4 rows over 515 states: dq 38 -> 17 us, dk and dv 62 -> 22, the joins 5 each)
  const int64_t gq = B * Hk * f.q_tiles, gk = B * Hk * f.k_tiles, row_tile = dkv_tile(D, dtype),
                row_tiles = H / Hk * ((Lq + row_tile - 1) / row_tile);
  int64_t s = gq > 0 ? 512 / gq : 1;
  if (s > Lk / 64) s = Lk / 64;
  if (s < 1) s = 1;
  f.q_chunk = ((Lk + s - 1) / s + 127) / 128 * 128;
  if (f.q_chunk < 128) f.q_chunk = 128;
  f.q_splits = static_cast<int>(Lk ? (Lk + f.q_chunk - 1) / f.q_chunk : 1);
  s = gk > 0 ? 512 / gk : 1;
  if (s > row_tiles * row_tile / 64) s = row_tiles * row_tile / 64;
  if (s < 1) s = 1;
  f.k_chunk = (row_tiles + s - 1) / s;
  if (f.k_chunk < 1) f.k_chunk = 1;
  f.k_splits = static_cast<int>(row_tiles ? (row_tiles + f.k_chunk - 1) / f.k_chunk : 1);
  return f;
}

static int64_t align16(int64_t n) { return (n + 15) / 16 * 16; }

int64_t attn_bwd_workspace(int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hk, int64_t D, int dtype) {
  const BwdPlan f = bwd_plan(B, Lq, Lk, H, Hk, D, dtype);
  // delta, then the partial sums of dq, then those of dk and dv
  return align16(B * H * Lq * 4) + (f.q_splits > 1 ? f.q_splits * B * H * Lq * D * 4 : 0) +
         (f.k_splits > 1 ? f.k_splits * B * Hk * Lk * 2 * D * 4 : 0);
}

template <typename T, int DP, int KIND>
static void bwd_dq(const AttnParams& p, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>((p.B * p.Hk * p.tiles * p.splits + 7) / 8 * 8);
  attn_dq_kernel<T, DP, KIND><<<grid, 256, 0, s>>>(p);
}

template <typename T, int DP, int KIND>
static void bwd_dkv(const AttnParams& p, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>((p.B * p.Hk * p.tiles * p.splits + 7) / 8 * 8);
  attn_dkv_kernel<T, DP, KIND><<<grid, 256, 0, s>>>(p);
}

template <typename T, int KIND, bool DQ>
static void bwd_heads(const AttnParams& p, hipStream_t s) {
  if constexpr (DQ) {
    if (p.D <= 32) bwd_dq<T, 32, KIND>(p, s);
    else if (p.D <= 64) bwd_dq<T, 64, KIND>(p, s);
    else if (p.D <= 96) bwd_dq<T, 96, KIND>(p, s);
    else bwd_dq<T, 128, KIND>(p, s);
  } else {
    if (p.D <= 32) bwd_dkv<T, 32, KIND>(p, s);
    else if (p.D <= 64) bwd_dkv<T, 64, KIND>(p, s);
    else if (p.D <= 96) bwd_dkv<T, 96, KIND>(p, s);
    else bwd_dkv<T, 128, KIND>(p, s);
  }
}

template <typename T>
static int bwd_type(AttnParams& p, hipStream_t s) {
  const BwdPlan f = bwd_plan(p.B, p.Lq, p.Lk, p.H, p.Hk, p.D, sizeof(T) == 2 ? FOVI_BF16 : FOVI_F32);
  p.delta = p.part;
  p.part = reinterpret_cast<float*>(reinterpret_cast<char*>(p.part) + align16(p.B * p.H * p.Lq * 4));
  const int64_t rows = p.B * p.H * p.Lq;
  p.part_k = p.part + (f.q_splits > 1 ? f.q_splits * rows * p.D : 0);
  p.k_splits = f.k_splits;
  if (rows) {
    p.tiles = f.q_tiles; p.splits = f.q_splits; p.chunk = f.q_chunk;
    if (p.kind == FOVI_MASK_NONE) bwd_heads<T, 0, true>(p, s);
    else if (p.kind == FOVI_MASK_KEEP) bwd_heads<T, 1, true>(p, s);
    else bwd_heads<T, 2, true>(p, s);
    if (check_launch("fovi_attention_bwd")) return 1;
  }
  if (p.Lk == 0 || p.B == 0) return 0;
  p.tiles = f.k_tiles; p.splits = f.k_splits; p.chunk = f.k_chunk;
  if (p.kind == FOVI_MASK_NONE) bwd_heads<T, 0, false>(p, s);
  else if (p.kind == FOVI_MASK_KEEP) bwd_heads<T, 1, false>(p, s);
  else bwd_heads<T, 2, false>(p, s);
  if (check_launch("fovi_attention_bwd")) return 1;
  if (f.q_splits > 1 || f.k_splits > 1) {
    p.splits = f.q_splits;
    p.chunk = f.q_chunk;
    const int64_t n = (f.q_splits > 1 ? rows : 0) * (p.D / 4) + (f.k_splits > 1 ? p.B * p.Hk * p.Lk : 0) * 2 * (p.D / 4);
    attn_bwd_join_kernel<T><<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(p);
    return check_launch("fovi_attention_bwd");
  }
  return 0;
}

int attn_bwd_launch(AttnParams& p, int dtype, hipStream_t s) {
  return dtype == FOVI_BF16 ? bwd_type<uint16_t>(p, s) : bwd_type<float>(p, s);
}

}  // namespace fovi
