// Attention of queries to the states of an encoder: forward, and the gradients of q, k and v.
//
//   s_ij = scale q_i.k_j (+ bias_ij) over the states j that row i keeps, p_i = softmax(s_i), o_i = sum_j p_ij v_j
//   ds_ij = p_ij (do_i.v_j - do_i.o_i), dq_i = scale sum_j ds_ij k_j, dk_j = scale sum_i ds_ij q_i, dv_j = sum_i p_ij do_i
//
// One wave per query row (forward, dq) or per state (dk, dv): each lane scores one of 64 states
// (rows), the wave keeps the running maximum and sum, and then each lane sums its two head elements
// over the 64. Pairs that are left out are skipped, so nothing in their place has an effect.
#include "common.h"

namespace fovi {

constexpr float kNegInf = -__builtin_inff();

struct AttnParams {
  const void* q; const void* k; const void* v; const void* mask; const int32_t* lens;
  void* o; float* stats; void* rest;
  const void* dout; void* dq; void* dk; void* dv;
  int64_t B, Lq, Lk;
  int H, Hk, G, D, kind;
  int64_t qs[3], ks[3], vs[3], os[3], ms[4], dos[3], dqs[3], dks[3], dvs[3];
  float scale;
};

__device__ __forceinline__ int64_t attn_len(const AttnParams& p, int64_t b) {
  if (!p.lens) return p.Lk;
  const int64_t n = p.lens[b];
  return n < 0 ? 0 : n < p.Lk ? n : p.Lk;
}

// The score of pair (i, j), -inf where it is left out.
template <typename T>
__device__ __forceinline__ float attn_score(const AttnParams& p, int64_t b, int h, int64_t i, int64_t j, const float* a,
                                            const T* row) {
  float bias = 0;
  if (p.kind) {
    const int64_t at = b * p.ms[0] + h * p.ms[1] + i * p.ms[2] + j * p.ms[3];
    if (p.kind == FOVI_MASK_KEEP) {
      if (!static_cast<const uint8_t*>(p.mask)[at]) return kNegInf;
    } else {
      bias = static_cast<const float*>(p.mask)[at];
      if (bias == kNegInf) return kNegInf;
    }
  }
  float s = 0;
  for (int d = 0; d < p.D; ++d) s = fmaf(a[d], Elem<T>::load(row + d), s);
  return fmaf(s, p.scale, bias);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

template <typename T>
__global__ __launch_bounds__(64) void attn_fwd_kernel(AttnParams p) {
  __shared__ float q[128];
  const int lane = threadIdx.x;
  const int64_t bh = blockIdx.x / p.Lq, i = blockIdx.x - bh * p.Lq, b = bh / p.H;
  const int h = static_cast<int>(bh - b * p.H), hk = h / p.G;
  const T* qr = static_cast<const T*>(p.q) + b * p.qs[0] + i * p.qs[1] + h * p.qs[2];
  const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
  const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];
  for (int d = lane; d < p.D; d += 64) q[d] = Elem<T>::load(qr + d);
  __syncthreads();
  float m = kNegInf, l = 0, acc[2] = {0, 0};
  const int64_t n = attn_len(p, b);
  for (int64_t j0 = 0; j0 < n; j0 += 64) {
    const int64_t j = j0 + lane;
    const float s = j < n ? attn_score<T>(p, b, h, i, j, q, k + j * p.ks[1]) : kNegInf;
    const float top = fmaxf(m, wave_max(s));
    const float e = s == kNegInf ? 0.0f : expf(s - top);
    const float keep = m == kNegInf ? 0.0f : expf(m - top);
    m = top;
    l = fmaf(l, keep, wave_sum(e));
    acc[0] *= keep;
    acc[1] *= keep;
    for (int t = 0; t < 64 && j0 + t < n; ++t) {
      const float et = __shfl(e, t);
      if (__shfl(s, t) == kNegInf) continue;
      for (int c = 0; c < 2; ++c)
        if (lane + 64 * c < p.D) acc[c] = fmaf(et, Elem<T>::load(v + (j0 + t) * p.vs[1] + lane + 64 * c), acc[c]);
    }
  }
  T* o = static_cast<T*>(p.o) + b * p.os[0] + i * p.os[1] + h * p.os[2];
  T* rest = p.rest ? static_cast<T*>(p.rest) + (o - static_cast<T*>(p.o)) : nullptr;
  for (int c = 0; c < 2; ++c)
    if (lane + 64 * c < p.D) {
      const float r = l == 0 ? 0.0f : acc[c] / l;
      Elem<T>::store(o + lane + 64 * c, r);
      if (rest) Elem<T>::store(rest + lane + 64 * c, r - Elem<T>::load(o + lane + 64 * c));
    }
  if (lane == 0 && p.stats) {
    p.stats[bh * p.Lq + i] = m;
    p.stats[(p.B * p.H + bh) * p.Lq + i] = l;
  }
}

// Element d of the output before its rounding, from the offset of its row.
template <typename T>
__device__ __forceinline__ float attn_out(const AttnParams& p, int64_t at) {
  const float o = Elem<T>::load(static_cast<const T*>(p.o) + at);
  return p.rest ? o + Elem<T>::load(static_cast<const T*>(p.rest) + at) : o;
}

template <typename T>
__global__ __launch_bounds__(64) void attn_dq_kernel(AttnParams p) {
  __shared__ float q[128], g[128];
  const int lane = threadIdx.x;
  const int64_t bh = blockIdx.x / p.Lq, i = blockIdx.x - bh * p.Lq, b = bh / p.H;
  const int h = static_cast<int>(bh - b * p.H), hk = h / p.G;
  const T* qr = static_cast<const T*>(p.q) + b * p.qs[0] + i * p.qs[1] + h * p.qs[2];
  const T* gr = static_cast<const T*>(p.dout) + b * p.dos[0] + i * p.dos[1] + h * p.dos[2];
  const int64_t o = b * p.os[0] + i * p.os[1] + h * p.os[2];
  const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
  const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];
  float delta = 0;
  for (int d = lane; d < p.D; d += 64) {
    q[d] = Elem<T>::load(qr + d);
    g[d] = Elem<T>::load(gr + d);
    delta = fmaf(g[d], attn_out<T>(p, o + d), delta);
  }
  delta = wave_sum(delta);
  __syncthreads();
  const float m = p.stats[bh * p.Lq + i], l = p.stats[(p.B * p.H + bh) * p.Lq + i];
  float acc[2] = {0, 0};
  const int64_t n = l == 0 ? 0 : attn_len(p, b);
  for (int64_t j0 = 0; j0 < n; j0 += 64) {
    const int64_t j = j0 + lane;
    const float s = j < n ? attn_score<T>(p, b, h, i, j, q, k + j * p.ks[1]) : kNegInf;
    float ds = 0;
    if (s != kNegInf) {
      float dp = 0;
      for (int d = 0; d < p.D; ++d) dp = fmaf(g[d], Elem<T>::load(v + j * p.vs[1] + d), dp);
      ds = expf(s - m) / l * (dp - delta);
    }
    for (int t = 0; t < 64 && j0 + t < n; ++t) {
      const float dt = __shfl(ds, t);
      if (__shfl(s, t) == kNegInf) continue;
      for (int c = 0; c < 2; ++c)
        if (lane + 64 * c < p.D) acc[c] = fmaf(dt, Elem<T>::load(k + (j0 + t) * p.ks[1] + lane + 64 * c), acc[c]);
    }
  }
  T* dq = static_cast<T*>(p.dq) + b * p.dqs[0] + i * p.dqs[1] + h * p.dqs[2];
  for (int c = 0; c < 2; ++c)
    if (lane + 64 * c < p.D) Elem<T>::store(dq + lane + 64 * c, acc[c] * p.scale);
}

template <typename T>
__global__ __launch_bounds__(64) void attn_dkv_kernel(AttnParams p) {
  __shared__ float kj[128], vj[128];
  const int lane = threadIdx.x;
  const int64_t bh = blockIdx.x / p.Lk, j = blockIdx.x - bh * p.Lk, b = bh / p.Hk;
  const int hk = static_cast<int>(bh - b * p.Hk);
  for (int d = lane; d < p.D; d += 64) {
    kj[d] = Elem<T>::load(static_cast<const T*>(p.k) + b * p.ks[0] + j * p.ks[1] + hk * p.ks[2] + d);
    vj[d] = Elem<T>::load(static_cast<const T*>(p.v) + b * p.vs[0] + j * p.vs[1] + hk * p.vs[2] + d);
  }
  __syncthreads();
  float dk[2] = {0, 0}, dv[2] = {0, 0};
  if (j < attn_len(p, b))
    for (int h = hk * p.G; h < (hk + 1) * p.G; ++h) {
      const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[2];
      const T* g = static_cast<const T*>(p.dout) + b * p.dos[0] + h * p.dos[2];
      const int64_t o = b * p.os[0] + h * p.os[2];
      for (int64_t i0 = 0; i0 < p.Lq; i0 += 64) {
        const int64_t i = i0 + lane;
        float s = kNegInf, e = 0, ds = 0;
        const int64_t at = (b * p.H + h) * p.Lq + i;
        const float l = i < p.Lq ? p.stats[p.B * p.H * p.Lq + at] : 0.0f;
        if (l != 0) s = attn_score<T>(p, b, h, i, j, kj, q + i * p.qs[1]);
        if (s != kNegInf) {
          float dp = 0, delta = 0;
          for (int d = 0; d < p.D; ++d) {
            const float gd = Elem<T>::load(g + i * p.dos[1] + d);
            dp = fmaf(gd, vj[d], dp);
            delta = fmaf(gd, attn_out<T>(p, o + i * p.os[1] + d), delta);
          }
          e = expf(s - p.stats[at]) / l;
          ds = e * (dp - delta);
        }
        for (int t = 0; t < 64 && i0 + t < p.Lq; ++t) {
          const float et = __shfl(e, t), dt = __shfl(ds, t);
          if (__shfl(s, t) == kNegInf) continue;
          for (int c = 0; c < 2; ++c)
            if (lane + 64 * c < p.D) {
              dk[c] = fmaf(dt, Elem<T>::load(q + (i0 + t) * p.qs[1] + lane + 64 * c), dk[c]);
              dv[c] = fmaf(et, Elem<T>::load(g + (i0 + t) * p.dos[1] + lane + 64 * c), dv[c]);
            }
        }
      }
    }
  T* dkr = static_cast<T*>(p.dk) + b * p.dks[0] + j * p.dks[1] + hk * p.dks[2];
  T* dvr = static_cast<T*>(p.dv) + b * p.dvs[0] + j * p.dvs[1] + hk * p.dvs[2];
  for (int c = 0; c < 2; ++c)
    if (lane + 64 * c < p.D) {
      Elem<T>::store(dkr + lane + 64 * c, dk[c] * p.scale);
      Elem<T>::store(dvr + lane + 64 * c, dv[c]);
    }
}

static int attn_check(const fovi_attention_args* a, const char* what) {
  if (!a || !a->q || !a->out) { set_error("%s: null pointer", what); return 1; }
  if (a->dtype != FOVI_F32 && a->dtype != FOVI_BF16) { set_error("%s: dtype must be F32 or BF16", what); return 1; }
  if (a->batch < 0 || a->q_len < 0 || a->kv_len < 0 || a->heads < 1 || a->kv_heads < 1) { set_error("%s: bad sizes", what); return 1; }
  if (a->heads % a->kv_heads) { set_error("%s: heads must be a multiple of kv_heads", what); return 1; }
  if (a->heads > (1 << 20)) { set_error("%s: more than 2^20 heads", what); return 1; }
  if (a->head_dim < 1 || a->head_dim > 128) { set_error("%s: head_dim must be 1 to 128", what); return 1; }
  if (a->kv_len && (!a->k || !a->v)) { set_error("%s: null pointer", what); return 1; }
  if (!(a->scale > 0) || a->scale > 3.0e38f) { set_error("%s: scale must be positive and finite", what); return 1; }
  if (a->mask_kind < FOVI_MASK_NONE || a->mask_kind > FOVI_MASK_BIAS) { set_error("%s: unknown mask_kind", what); return 1; }
  if (a->mask_kind != FOVI_MASK_NONE && !a->mask) { set_error("%s: null mask", what); return 1; }
  if (a->batch * a->heads * a->q_len > 0x7fffffff || a->batch * a->kv_heads * a->kv_len > 0x7fffffff) {
    set_error("%s: too many rows", what);
    return 1;
  }
  return 0;
}

static AttnParams attn_params(const fovi_attention_args* a) {
  AttnParams p = {};
  p.q = a->q; p.k = a->k; p.v = a->v; p.mask = a->mask; p.lens = a->kv_lengths; p.o = a->out; p.stats = a->stats; p.rest = a->out_rest;
  p.B = a->batch; p.Lq = a->q_len; p.Lk = a->kv_len;
  p.H = static_cast<int>(a->heads); p.Hk = static_cast<int>(a->kv_heads); p.G = p.H / p.Hk;
  p.D = static_cast<int>(a->head_dim); p.kind = a->mask_kind; p.scale = a->scale;
  for (int i = 0; i < 3; ++i) { p.qs[i] = a->q_stride[i]; p.ks[i] = a->k_stride[i]; p.vs[i] = a->v_stride[i]; p.os[i] = a->out_stride[i]; }
  for (int i = 0; i < 4; ++i) p.ms[i] = a->mask_stride[i];
  return p;
}

}  // namespace fovi

using namespace fovi;

extern "C" int64_t fovi_attention_fwd_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int32_t) { return 0; }

extern "C" int fovi_attention_fwd(const fovi_attention_args* a, void* stream) {
  clear_error();
  if (attn_check(a, "fovi_attention_fwd")) return 1;
  const unsigned rows = static_cast<unsigned>(a->batch * a->heads * a->q_len);
  if (rows == 0) return 0;
  const AttnParams p = attn_params(a);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == FOVI_BF16) attn_fwd_kernel<uint16_t><<<rows, 64, 0, s>>>(p);
  else attn_fwd_kernel<float><<<rows, 64, 0, s>>>(p);
  return check_launch("fovi_attention_fwd");
}

extern "C" int64_t fovi_attention_bwd_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int32_t) { return 0; }

extern "C" int fovi_attention_bwd(const fovi_attention_bwd_args* a, void* stream) {
  clear_error();
  if (!a) { set_error("fovi_attention_bwd: null pointer"); return 1; }
  if (attn_check(&a->fwd, "fovi_attention_bwd")) return 1;
  if (!a->fwd.stats || !a->dout || !a->dq || (a->fwd.kv_len && (!a->dk || !a->dv))) {
    set_error("fovi_attention_bwd: null pointer");
    return 1;
  }
  AttnParams p = attn_params(&a->fwd);
  p.dout = a->dout; p.dq = a->dq; p.dk = a->dk; p.dv = a->dv;
  for (int i = 0; i < 3; ++i) {
    p.dos[i] = a->dout_stride[i]; p.dqs[i] = a->dq_stride[i]; p.dks[i] = a->dk_stride[i]; p.dvs[i] = a->dv_stride[i];
  }
  const unsigned rows = static_cast<unsigned>(p.B * p.H * p.Lq), states = static_cast<unsigned>(p.B * p.Hk * p.Lk);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool bf16 = a->fwd.dtype == FOVI_BF16;
  if (rows) {
    if (bf16) attn_dq_kernel<uint16_t><<<rows, 64, 0, s>>>(p);
    else attn_dq_kernel<float><<<rows, 64, 0, s>>>(p);
    if (check_launch("fovi_attention_bwd")) return 1;
  }
  if (states) {
    if (bf16) attn_dkv_kernel<uint16_t><<<states, 64, 0, s>>>(p);
    else attn_dkv_kernel<float><<<states, 64, 0, s>>>(p);
  }
  return check_launch("fovi_attention_bwd");
}
