// pk_ops.cpp -- extern "C" entry points of the drafted-decoding and serving
// operators (include/pk.h): arguments are checked here, before anything is launched.
#include <cuda_runtime.h>

#include <cmath>
#include <string>

#include "pk.h"
#include "pk_cache.h"

namespace pk {
int set_error(int code, const std::string &msg);
int cuda_error(cudaError_t e, const char *what);
}  // namespace pk
using namespace pk;

#define CK(expr)                                         \
  do {                                                   \
    cudaError_t _e = (expr);                             \
    if (_e != cudaSuccess) return cuda_error(_e, #expr); \
  } while (0)

namespace {

int bad(const std::string &msg) { return set_error(PK_ERR_INVALID, msg); }
bool is_float_type(int t) { return t == PK_TYPE_F32 || t == PK_TYPE_F16 || t == PK_TYPE_BF16; }
uintptr_t elem_mask(int t) { return t == PK_TYPE_F32 ? 3 : 1; }

int check_cache(const char *who, const pk_kv_cache *c) {
  const std::string w(who);
  if (!c) return bad(w + ": null cache");
  if (c->type != PK_KV_Q8 && c->type != PK_KV_Q4)
    return set_error(PK_ERR_UNSUPPORTED, w + ": cache type " + std::to_string(c->type) + " is not PK_KV_Q8 or PK_KV_Q4");
  if (c->head_dim != 64 && c->head_dim != 128)
    return set_error(PK_ERR_UNSUPPORTED, w + ": head_dim " + std::to_string(c->head_dim) + " is not 64 or 128");
  if (c->n_pages < 1 || c->n_kv < 1 || c->n_kv > 65536) return bad(w + ": n_pages and n_kv must be positive (n_kv at most 65536)");
  if (c->page_size < 16 || c->page_size > 65536 || (c->page_size & (c->page_size - 1)))
    return bad(w + ": page_size must be a power of two from 16 to 65536");
  if (!c->k || !c->v || !c->ks || !c->vs) return bad(w + ": null cache array");
  if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->ks | (uintptr_t)c->vs) & 15)
    return bad(w + ": cache arrays must be 16-byte aligned");
  return PK_OK;
}

int check_seqs(const char *who, const pk_kv_seqs *s) {
  const std::string w(who);
  if (!s) return bad(w + ": null sequences");
  if (s->n_seq < 0 || s->n_tok < 0 || s->max_new < 0 || s->max_len < 0) return bad(w + ": negative count");
  if (s->n_seq == 0 || s->n_tok == 0 || s->max_new == 0 || s->max_len == 0) return PK_OK;
  if (s->max_pages < 1) return bad(w + ": max_pages must be positive");
  if (s->max_len > (1 << 30) || s->n_tok > (1 << 30)) return bad(w + ": max_len and n_tok are at most 2^30");
  if (!s->start || !s->ctx || !s->pages) return bad(w + ": null sequence array");
  if (((uintptr_t)s->start | (uintptr_t)s->ctx | (uintptr_t)s->pages) & 3) return bad(w + ": misaligned sequence array");
  return PK_OK;
}
// Query rows, and (sequence, kv head) pairs, that a grid can number.
bool fits_grid(const pk_kv_cache *c, const pk_kv_seqs *s, int n_head) {
  return (int64_t)s->n_tok * n_head <= 0x7fffffff && (int64_t)s->n_seq * c->n_kv <= 0x7fffffff;
}
bool nothing(const pk_kv_seqs *s) { return s->n_seq == 0 || s->n_tok == 0 || s->max_new == 0 || s->max_len == 0; }

int check_rows(const char *who, const pk_kv_cache *c, const void *k, const void *v, int type, int64_t ts, int64_t hs) {
  const std::string w(who);
  if (!is_float_type(type)) return set_error(PK_ERR_UNSUPPORTED, w + ": element type " + std::to_string(type) + " is not f32, f16 or bf16");
  if (!k || !v) return bad(w + ": null rows");
  if (((uintptr_t)k | (uintptr_t)v) & elem_mask(type)) return bad(w + ": misaligned rows");
  if (hs < c->head_dim && c->n_kv > 1) return bad(w + ": head_stride is less than head_dim");
  if (ts < 0 || hs < 0 || ts > (1LL << 40) || hs > (1LL << 40)) return bad(w + ": stride out of range");
  return PK_OK;
}

int check_query(const char *who, const pk_kv_cache *c, const pk_kv_seqs *s, const pk_kv_query *q) {
  const std::string w(who);
  if (!q) return bad(w + ": null query");
  if (!is_float_type(q->type)) return set_error(PK_ERR_UNSUPPORTED, w + ": element type " + std::to_string(q->type) + " is not f32, f16 or bf16");
  if (q->n_head < 1 || q->n_head % c->n_kv) return bad(w + ": n_head must be a positive multiple of n_kv");
  if (!(q->scale > 0.0f) || !std::isfinite(q->scale)) return bad(w + ": scale must be positive and finite");
  if (q->mask && (q->mask_words < 1 || q->mask_words > 4096)) return bad(w + ": mask_words must be 1 to 4096 with a mask");
  if (nothing(s)) return PK_OK;
  if (!fits_grid(c, s, q->n_head)) return bad(w + ": n_tok * n_head and n_seq * n_kv are at most 2^31 - 1");
  if (!q->q || !q->out) return bad(w + ": null q or out");
  if (((uintptr_t)q->q | (uintptr_t)q->out) & elem_mask(q->type) || ((uintptr_t)q->mask & 7)) return bad(w + ": misaligned q, out or mask");
  const int64_t st[4] = {q->q_tok_stride, q->q_head_stride, q->out_tok_stride, q->out_head_stride};
  for (int64_t x : st)
    if (x < 0 || x > (1LL << 40)) return bad(w + ": stride out of range");
  if ((q->out_head_stride < c->head_dim && q->n_head > 1) || (q->out_tok_stride < c->head_dim && s->n_tok > 1))
    return bad(w + ": out strides are less than head_dim");
  return PK_OK;
}
int check_shared(const char *who, const pk_kv_seqs *s, const pk_kv_shared *sh) {
  const std::string w(who);
  if (!sh) return bad(w + ": null groups");
  if (sh->n_group < 0 || sh->n_group > s->n_seq || sh->max_tok < 0 || sh->max_len < 0 || sh->max_own < 0)
    return bad(w + ": negative count, or more groups than sequences");
  if (sh->n_group > 0 && (!sh->first || !sh->len || (((uintptr_t)sh->first | (uintptr_t)sh->len) & 3)))
    return bad(w + ": null or misaligned group array");
  return PK_OK;
}
int check_scratch(const char *who, size_t need, const void *scratch, size_t bytes) {
  if (need && (!scratch || bytes < need || ((uintptr_t)scratch & 15)))
    return bad(std::string(who) + ": scratch must be 16-byte aligned and hold " + std::to_string(need) + " bytes");
  return PK_OK;
}

}  // namespace

extern "C" {

int pk_kv_store(const pk_kv_cache *c, const pk_kv_seqs *s, const void *k, const void *v, int type, int64_t tok_stride,
                int64_t head_stride, void *stream) {
  if (int rc = check_cache("pk_kv_store", c)) return rc;
  if (int rc = check_seqs("pk_kv_store", s)) return rc;
  if (!is_float_type(type)) return set_error(PK_ERR_UNSUPPORTED, "pk_kv_store: element type " + std::to_string(type) + " is not f32, f16 or bf16");
  if (nothing(s)) return PK_OK;
  if (int rc = check_rows("pk_kv_store", c, k, v, type, tok_stride, head_stride)) return rc;
  CK(launch_kv_store(*c, *s, k, v, type, (long)tok_stride, (long)head_stride, (cudaStream_t)stream));
  return PK_OK;
}

int pk_kv_load(const pk_kv_cache *c, const pk_kv_seqs *s, void *k, void *v, int type, int64_t tok_stride,
               int64_t head_stride, void *stream) {
  if (int rc = check_cache("pk_kv_load", c)) return rc;
  if (int rc = check_seqs("pk_kv_load", s)) return rc;
  if (!is_float_type(type)) return set_error(PK_ERR_UNSUPPORTED, "pk_kv_load: element type " + std::to_string(type) + " is not f32, f16 or bf16");
  if (nothing(s)) return PK_OK;
  if (int rc = check_rows("pk_kv_load", c, k, v, type, tok_stride, head_stride)) return rc;
  if (tok_stride < (int64_t)c->head_dim && s->n_tok > 1) return bad("pk_kv_load: tok_stride is less than head_dim");
  CK(launch_kv_load(*c, *s, k, v, type, (long)tok_stride, (long)head_stride, (cudaStream_t)stream));
  return PK_OK;
}

int pk_kv_keep(const pk_kv_cache *c, const pk_kv_seqs *s, const int *keep, int keep_stride, const int *n_keep,
               void *stream) {
  if (int rc = check_cache("pk_kv_keep", c)) return rc;
  if (int rc = check_seqs("pk_kv_keep", s)) return rc;
  if (keep_stride < 0) return bad("pk_kv_keep: negative keep_stride");
  if (nothing(s) || keep_stride == 0) return PK_OK;
  if (!keep || !n_keep || (((uintptr_t)keep | (uintptr_t)n_keep) & 3)) return bad("pk_kv_keep: null or misaligned keep");
  CK(launch_kv_keep(*c, *s, keep, keep_stride, n_keep, (cudaStream_t)stream));
  return PK_OK;
}

size_t pk_kv_attn_scratch_bytes(const pk_kv_cache *c, const pk_kv_seqs *s, int n_head, int type) {
  if (check_cache("pk_kv_attn_scratch_bytes", c) || check_seqs("pk_kv_attn_scratch_bytes", s)) return 0;
  if (nothing(s) || n_head < 1 || n_head % c->n_kv || !is_float_type(type) || !fits_grid(c, s, n_head)) return 0;
  return kv_attn_scratch_bytes(*c, *s, n_head, type);
}

int pk_kv_attn(const pk_kv_cache *c, const pk_kv_seqs *s, const pk_kv_query *q, void *scratch, size_t scratch_bytes,
               void *stream) {
  if (int rc = check_cache("pk_kv_attn", c)) return rc;
  if (int rc = check_seqs("pk_kv_attn", s)) return rc;
  if (int rc = check_query("pk_kv_attn", c, s, q)) return rc;
  if (nothing(s)) return PK_OK;
  const size_t need = kv_attn_scratch_bytes(*c, *s, q->n_head, q->type);
  if (int rc = check_scratch("pk_kv_attn", need, scratch, scratch_bytes)) return rc;
  CK(launch_kv_attn(*c, *s, *q, scratch, (cudaStream_t)stream));
  return PK_OK;
}

size_t pk_kv_attn_shared_scratch_bytes(const pk_kv_cache *c, const pk_kv_seqs *s, const pk_kv_shared *sh, int n_head, int type) {
  const char *who = "pk_kv_attn_shared_scratch_bytes";
  if (check_cache(who, c) || check_seqs(who, s) || check_shared(who, s, sh)) return 0;
  if (nothing(s) || n_head < 1 || n_head % c->n_kv || !is_float_type(type) || !fits_grid(c, s, n_head)) return 0;
  return kv_attn_shared_scratch_bytes(*c, *s, *sh, n_head, type);
}

int pk_kv_attn_shared(const pk_kv_cache *c, const pk_kv_seqs *s, const pk_kv_shared *sh, const pk_kv_query *q, void *scratch,
                      size_t scratch_bytes, void *stream) {
  const char *who = "pk_kv_attn_shared";
  if (int rc = check_cache(who, c)) return rc;
  if (int rc = check_seqs(who, s)) return rc;
  if (int rc = check_shared(who, s, sh)) return rc;
  if (int rc = check_query(who, c, s, q)) return rc;
  if (nothing(s)) return PK_OK;
  const size_t need = kv_attn_shared_scratch_bytes(*c, *s, *sh, q->n_head, q->type);
  if (int rc = check_scratch(who, need, scratch, scratch_bytes)) return rc;
  CK(launch_kv_attn_shared(*c, *s, *sh, *q, scratch, (cudaStream_t)stream));
  return PK_OK;
}

int pk_kv_plan(const pk_kv_plan_args *a, void *stream) {
  if (!a) return bad("pk_kv_plan: null argument");
  if (a->n_seq < 0 || a->n_seq > 16384 || a->n_tok < 0 || a->n_tok > (1 << 30) || a->max_pages < 0 || a->free_cap < 0)
    return bad("pk_kv_plan: count out of range (n_seq at most 16384, n_tok 2^30)");
  if ((int64_t)a->n_seq * a->max_pages > 0x7fffffff) return bad("pk_kv_plan: n_seq * max_pages is at most 2^31 - 1");
  if (a->page_size < 16 || a->page_size > 65536 || (a->page_size & (a->page_size - 1)))
    return bad("pk_kv_plan: page_size must be a power of two from 16 to 65536");
  const bool seqs = a->n_seq > 0, tables = seqs && a->max_pages > 0;
  if ((seqs && (!a->ctx || !a->n_new || !a->held || !a->held_out)) || (tables && (!a->pages || !a->pages_out)) ||
      (a->free_cap > 0 && (!a->free || !a->free_out)) || !a->n_free || !a->n_free_out || !a->start || !a->lacking)
    return bad("pk_kv_plan: null array");
  const uintptr_t all = (uintptr_t)a->ctx | (uintptr_t)a->n_new | (uintptr_t)a->pages | (uintptr_t)a->held | (uintptr_t)a->free |
                        (uintptr_t)a->n_free | (uintptr_t)a->done | (uintptr_t)a->shared | (uintptr_t)a->pages_out |
                        (uintptr_t)a->held_out | (uintptr_t)a->free_out | (uintptr_t)a->n_free_out | (uintptr_t)a->start |
                        (uintptr_t)a->lacking | (uintptr_t)a->pos | (uintptr_t)a->seq;
  if ((all & 3) || ((uintptr_t)a->slot & 7)) return bad("pk_kv_plan: misaligned array");
  // in place: all of what is there
  const bool in_place = a->n_free_out == a->n_free;
  if ((seqs && (a->held_out == a->held) != in_place) || (tables && (a->pages_out == a->pages) != in_place) ||
      (a->free_cap > 0 && (a->free_out == a->free) != in_place))
    return bad("pk_kv_plan: pages, held, free and n_free are all updated in place or none is");
  CK(launch_kv_plan(*a, in_place, (cudaStream_t)stream));
  return PK_OK;
}

int pk_sample_rows(const void *logits, int type, int rows, int n, int64_t stride, const pk_sample_args *a, void *stream) {
  if (!is_float_type(type)) return set_error(PK_ERR_UNSUPPORTED, "pk_sample_rows: element type " + std::to_string(type) + " is not f32, f16 or bf16");
  if (!a) return bad("pk_sample_rows: null arguments");
  if (rows < 0 || rows > (1 << 24) || n < 1 || n > (1 << 30)) return bad("pk_sample_rows: rows must be 0 to 2^24 and n 1 to 2^30");
  if (rows == 0) return PK_OK;
  if (!logits || !a->u || !a->tok) return bad("pk_sample_rows: null logits, u or tok");
  if ((uintptr_t)logits & elem_mask(type)) return bad("pk_sample_rows: misaligned logits");
  if (((uintptr_t)a->u | (uintptr_t)a->temp | (uintptr_t)a->top_k | (uintptr_t)a->top_p | (uintptr_t)a->min_p | (uintptr_t)a->tok |
       (uintptr_t)a->prob | (uintptr_t)a->kept) & 3)
    return bad("pk_sample_rows: misaligned array");
  if (stride < 0 || stride > (1LL << 40)) return bad("pk_sample_rows: row stride out of range");
  CK(launch_sample(logits, type, rows, n, (long)stride, *a, (cudaStream_t)stream));
  return PK_OK;
}

int pk_rope_turns(const pk_rope_spec *p, double *turns, float *gain) {
  if (!p || !turns || !gain) return bad("pk_rope_turns: null argument");
  if (p->n_rot < 2 || p->n_rot % 2 || p->n_rot > 4096) return bad("pk_rope_turns: n_rot must be even, 2 to 4096");
  if (!(p->theta > 0.0) || !std::isfinite(p->theta)) return bad("pk_rope_turns: theta must be positive");
  if (p->scaling < PK_ROPE_NONE || p->scaling > PK_ROPE_YARN) return bad("pk_rope_turns: unknown scaling");
  if (p->scaling != PK_ROPE_NONE && (!(p->factor > 0.0) || !std::isfinite(p->factor))) return bad("pk_rope_turns: factor must be positive");
  if (p->scaling == PK_ROPE_YARN && (!(p->n_ctx_train > 0.0) || !(p->high > p->low) || !(p->low >= 0.0)))
    return bad("pk_rope_turns: n_ctx_train must be positive and high > low >= 0");
  if (!(p->gain >= 0.0) || !std::isfinite(p->gain)) return bad("pk_rope_turns: gain must be 0 or positive");
  const int n = p->n_rot;
  double theta = p->theta, g = 1.0;
  if (p->scaling == PK_ROPE_NTK && n > 2) theta *= std::pow(p->factor, (double)n / (n - 2));
  if (p->scaling == PK_ROPE_YARN && p->factor > 1.0) g = 0.1 * std::log(p->factor) + 1.0;
  for (int i = 0; i < n / 2; i++) {
    double f = std::pow(theta, -2.0 * i / n) / 6.283185307179586476925286766559;
    if (p->factors) {
      if (!(p->factors[i] > 0.0f) || !std::isfinite(p->factors[i])) return bad("pk_rope_turns: factors must be positive");
      f /= (double)p->factors[i];
    }
    if (p->scaling == PK_ROPE_LINEAR) f /= p->factor;
    if (p->scaling == PK_ROPE_YARN) {
      double keep = (f * p->n_ctx_train - p->low) / (p->high - p->low);
      keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
      f = f / p->factor * (1.0 - keep) + f * keep;
    }
    turns[i] = f;
  }
  *gain = (float)(p->gain > 0.0 ? p->gain : g);
  return PK_OK;
}

int pk_rope(const pk_rope_args *a, void *stream) {
  if (!a) return bad("pk_rope: null argument");
  if (!is_float_type(a->type)) return set_error(PK_ERR_UNSUPPORTED, "pk_rope: element type " + std::to_string(a->type) + " is not f32, f16 or bf16");
  if (a->layout != PK_ROPE_INTERLEAVED && a->layout != PK_ROPE_HALF) return bad("pk_rope: unknown layout");
  if (a->head_dim < 2 || a->n_rot < 2 || a->n_rot % 2 || a->n_rot > a->head_dim || a->n_rot > 4096)
    return bad("pk_rope: n_rot must be even, 2 to head_dim (at most 4096)");
  if (a->n_tok < 0 || a->n_head < 0 || a->n_kv < 0 || a->n_head > 65536 || a->n_kv > 65536 || a->head_dim > 8192)
    return bad("pk_rope: count out of range");
  if (a->n_tok == 0 || (a->n_head == 0 && a->n_kv == 0)) return PK_OK;  // (no rows: their pointers may be null)
  if (!a->q && !a->k) return bad("pk_rope: neither q nor k");
  if ((!a->q || a->n_head == 0) && (!a->k || a->n_kv == 0)) return PK_OK;
  if (!a->pos || !a->turns || ((uintptr_t)a->pos & 3) || ((uintptr_t)a->turns & 7)) return bad("pk_rope: null or misaligned pos or turns");
  if ((a->q && !a->q_out) || (a->k && !a->k_out)) return bad("pk_rope: null output");
  const uintptr_t m = elem_mask(a->type);
  if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)(a->q ? a->q_out : nullptr) | (uintptr_t)(a->k ? a->k_out : nullptr)) & m)
    return bad("pk_rope: misaligned rows");
  const int64_t st[8] = {a->q_tok_stride, a->q_head_stride, a->k_tok_stride, a->k_head_stride,
                         a->qo_tok_stride, a->qo_head_stride, a->ko_tok_stride, a->ko_head_stride};
  for (int i = 0; i < 8; i++) {
    const bool k = (i & 2) != 0, head = (i & 1) != 0;
    if (!(k ? a->k : a->q)) continue;
    if (st[i] < 0 || st[i] > (1LL << 40)) return bad("pk_rope: stride out of range");
    if (i >= 4 && st[i] < a->head_dim && (head ? (k ? a->n_kv : a->n_head) : a->n_tok) > 1)
      return bad("pk_rope: output strides are less than head_dim");
  }
  CK(launch_rope(*a, (cudaStream_t)stream));
  return PK_OK;
}

int pk_apply_logit_rules(const void *logits, void *out, int type, int rows, int n, int64_t in_stride,
                         int64_t out_stride, const pk_logit_rules *r, void *stream) {
  if (!is_float_type(type)) return set_error(PK_ERR_UNSUPPORTED, "pk_apply_logit_rules: element type " + std::to_string(type) + " is not f32, f16 or bf16");
  if (!r) return bad("pk_apply_logit_rules: null rules");
  if (rows < 0 || n < 0 || n > (1 << 30)) return bad("pk_apply_logit_rules: rows is negative or n not within 0 .. 2^30");
  if (rows == 0 || n == 0) return PK_OK;
  if (!logits || !out || (((uintptr_t)logits | (uintptr_t)out) & elem_mask(type))) return bad("pk_apply_logit_rules: null or misaligned logits");
  if (in_stride < 0 || in_stride > (1LL << 40) || out_stride > (1LL << 40) || (rows > 1 && out_stride < n) || out_stride < 0)
    return bad("pk_apply_logit_rules: row stride out of range");
  if (logits == out && rows > 1 && in_stride != out_stride) return bad("pk_apply_logit_rules: in place with two row strides");
  if (r->n_hist_max < 0 || r->n_bias < 0) return bad("pk_apply_logit_rules: negative count");
  const int64_t st[3] = {r->hist ? r->hist_stride : 0, r->bias_id ? r->bias_stride : 0, r->allow ? r->allow_stride : 0};
  for (int64_t x : st)
    if (x < 0 || x > (1LL << 40)) return bad("pk_apply_logit_rules: list stride out of range");
  if ((r->bias_id != nullptr) != (r->bias != nullptr)) return bad("pk_apply_logit_rules: bias ids and biases come together");
  if (((uintptr_t)r->repeat | (uintptr_t)r->freq | (uintptr_t)r->presence | (uintptr_t)r->hist | (uintptr_t)r->n_hist |
       (uintptr_t)r->bias_id | (uintptr_t)r->bias | (uintptr_t)r->allow) & 3)
    return bad("pk_apply_logit_rules: misaligned rule array");
  CK(launch_logit_rules(logits, out, type, rows, n, (long)in_stride, (long)out_stride, *r, (cudaStream_t)stream));
  return PK_OK;
}

}  // extern "C"
