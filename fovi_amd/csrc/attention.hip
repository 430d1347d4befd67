// Attention of queries to the states of an encoder: the C entries, their checks and the layouts they take.
//
//   s_ij = scale q_i.k_j (+ bias_ij) over the states j that row i keeps, p_i = softmax(s_i), o_i = sum_j p_ij v_j
//
// The kernels are in attention_fwd.hip and attention_bwd.hip, what they share in attention.h.
#include "attention.h"

namespace fovi {

static int attn_check(const fovi_attention_args* a, const char* what) {
  if (!a || !a->q || !a->out) { set_error("%s: null pointer", what); return 1; }
  if (a->dtype != FOVI_F32 && a->dtype != FOVI_BF16) { set_error("%s: dtype must be F32 or BF16", what); return 1; }
  if (a->batch < 0 || a->q_len < 0 || a->kv_len < 0 || a->heads < 1 || a->kv_heads < 1) { set_error("%s: bad sizes", what); return 1; }
  if (a->heads % a->kv_heads) { set_error("%s: heads must be a multiple of kv_heads", what); return 1; }
  if (a->heads > (1 << 20)) { set_error("%s: more than 2^20 heads", what); return 1; }
  if (a->head_dim < 1 || a->head_dim > 128) { set_error("%s: head_dim must be 1 to 128", what); return 1; }
  if (a->kv_len && (!a->k || !a->v)) { set_error("%s: null pointer", what); return 1; }
  if (!(a->scale > 0) || a->scale > 2.0e38f) { set_error("%s: scale must be positive and finite", what); return 1; }
  if (a->mask_kind < FOVI_MASK_NONE || a->mask_kind > FOVI_MASK_BIAS) { set_error("%s: unknown mask_kind", what); return 1; }
  if (a->mask_kind != FOVI_MASK_NONE && a->kv_len && !a->mask) { set_error("%s: null mask", what); return 1; }
  if (a->q_len > 0x7fffffff / a->heads / (a->batch ? a->batch : 1) ||
      a->kv_len > 0x7fffffff / a->kv_heads / (a->batch ? a->batch : 1)) {
    set_error("%s: too many rows or states", what);
    return 1;
  }
  return 0;
}

// Rows of 16-byte pieces: pointers and strides of whole pieces, rows less than kMostPitch apart.
static bool whole(const void* p, const int64_t* stride, int es) {
  if (reinterpret_cast<uintptr_t>(p) % 16 || stride[1] < 0 || stride[1] * es >= kMostPitch) return false;
  for (int i = 0; i < 3; ++i)
    if (stride[i] * es % 16) return false;
  return true;
}

static int attn_check_rows(const fovi_attention_args* a, const char* what) {
  const int es = a->dtype == FOVI_BF16 ? 2 : 4;
  if (a->head_dim * es % 16 || !whole(a->q, a->q_stride, es) || !whole(a->k, a->k_stride, es) || !whole(a->v, a->v_stride, es) ||
      !whole(a->out, a->out_stride, es) || !whole(a->out_rest, a->out_stride, es)) {
    set_error("%s: heads must be whole 16-byte pieces, aligned, and rows less than 64 MiB apart", what);
    return 1;
  }
  return 0;
}

static AttnParams attn_params(const fovi_attention_args* a) {
  AttnParams p = {};
  p.q = a->q; p.k = a->k; p.v = a->v; p.mask = a->mask; p.lens = a->kv_lengths; p.o = a->out; p.stats = a->stats; p.rest = a->out_rest;
  p.B = a->batch; p.Lq = a->q_len; p.Lk = a->kv_len;
  p.H = static_cast<int>(a->heads); p.Hk = static_cast<int>(a->kv_heads); p.G = p.H / p.Hk;
  p.D = static_cast<int>(a->head_dim); p.kind = a->mask_kind; p.scale = a->scale; p.c = a->scale * kLog2e;
  p.R = p.G * p.Lq; p.part = static_cast<float*>(a->workspace);
  for (int i = 0; i < 3; ++i) { p.qs[i] = a->q_stride[i]; p.ks[i] = a->k_stride[i]; p.vs[i] = a->v_stride[i]; p.os[i] = a->out_stride[i]; }
  for (int i = 0; i < 4; ++i) p.ms[i] = a->mask_stride[i];
  return p;
}

}  // namespace fovi

using namespace fovi;

extern "C" int fovi_attention_pack_mask(const void* keep, const int64_t* stride, int64_t n0, int64_t n1, int64_t n2, int64_t kv_len,
                                        uint32_t* words, void* stream) {
  clear_error();
  if (!keep || !stride || !words) { set_error("fovi_attention_pack_mask: null pointer"); return 1; }
  if (n0 < 0 || n1 < 0 || n2 < 0 || kv_len < 0) { set_error("fovi_attention_pack_mask: bad sizes"); return 1; }
  const int64_t per = (kv_len + 31) / 32, most = int64_t(0x7fffffff) * 256;
  if (n0 && n1 && n2 && per && (n0 > most / n1 || n0 * n1 > most / n2 || n0 * n1 * n2 > most / per)) {
    set_error("fovi_attention_pack_mask: mask too large");
    return 1;
  }
  return attn_pack_launch(keep, stride, n0, n1, n2, kv_len, words, static_cast<hipStream_t>(stream));
}

extern "C" int64_t fovi_attention_fwd_workspace_bytes(int64_t batch, int64_t q_len, int64_t kv_len, int64_t heads, int64_t kv_heads,
                                                      int64_t head_dim, int32_t dtype) {
  if (batch < 0 || q_len < 0 || kv_len < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads) return 0;
  return attn_fwd_workspace(batch, q_len, kv_len, heads, kv_heads, head_dim, dtype);
}

static int attn_check_workspace(const fovi_attention_args* a, int64_t need, const char* what) {
  if (need == 0) return 0;
  if (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16) {
    set_error("%s: workspace of %lld bytes needed, 16-byte aligned", what, static_cast<long long>(need));
    return 1;
  }
  return 0;
}

extern "C" int fovi_attention_fwd(const fovi_attention_args* a, void* stream) {
  clear_error();
  if (attn_check(a, "fovi_attention_fwd") || attn_check_rows(a, "fovi_attention_fwd")) return 1;
  if (a->batch == 0 || a->q_len == 0) return 0;
  AttnParams p = attn_params(a);
  if (attn_check_workspace(a, attn_fwd_workspace(p.B, p.Lq, p.Lk, p.H, p.Hk, p.D, a->dtype), "fovi_attention_fwd")) return 1;
  return attn_fwd_launch(p, a->dtype, static_cast<hipStream_t>(stream));
}

extern "C" int64_t fovi_attention_bwd_workspace_bytes(int64_t batch, int64_t q_len, int64_t kv_len, int64_t heads, int64_t kv_heads,
                                                      int64_t head_dim, int32_t dtype) {
  if (batch < 0 || q_len < 0 || kv_len < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads) return 0;
  return attn_bwd_workspace(batch, q_len, kv_len, heads, kv_heads, head_dim, dtype);
}

extern "C" int fovi_attention_bwd(const fovi_attention_bwd_args* a, void* stream) {
  clear_error();
  if (!a) { set_error("fovi_attention_bwd: null pointer"); return 1; }
  const fovi_attention_args* f = &a->fwd;
  if (attn_check(f, "fovi_attention_bwd")) return 1;
  if (!f->stats || !a->dout || !a->dq || (f->kv_len && (!a->dk || !a->dv))) {
    set_error("fovi_attention_bwd: null pointer");
    return 1;
  }
  const int es = f->dtype == FOVI_BF16 ? 2 : 4;
  if (attn_check_rows(f, "fovi_attention_bwd")) return 1;
  if (!whole(a->dout, a->dout_stride, es) || !whole(a->dq, a->dq_stride, es) || !whole(a->dk, a->dk_stride, es) ||
      !whole(a->dv, a->dv_stride, es)) {
    set_error("fovi_attention_bwd: heads must be whole 16-byte pieces, aligned, and rows less than 64 MiB apart");
    return 1;
  }
  AttnParams p = attn_params(f);
  if (attn_check_workspace(f, attn_bwd_workspace(p.B, p.Lq, p.Lk, p.H, p.Hk, p.D, f->dtype), "fovi_attention_bwd")) return 1;
  p.dout = a->dout; p.dq = a->dq; p.dk = a->dk; p.dv = a->dv;
  for (int i = 0; i < 3; ++i) {
    p.dos[i] = a->dout_stride[i]; p.dqs[i] = a->dq_stride[i]; p.dks[i] = a->dk_stride[i]; p.dvs[i] = a->dv_stride[i];
  }
  return attn_bwd_launch(p, f->dtype, static_cast<hipStream_t>(stream));
}
