// pk_cache.h -- host-side view of the quantised paged K/V cache's kernels
// (pk_cache.cu), of the attention that reads it (pk_cache_attn.cu) and of the
// rotary and logit-rule kernels (pk_rows.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "pk.h"

namespace pk {

// Row geometry.  Q8: head_dim code bytes, one scale word.  Q4: head_dim / 2
// code bytes, two scale words (D and the sub-scales).
inline int kv_row_bytes(int type, int dh) { return type == PK_KV_Q8 ? dh : dh / 2; }
inline int kv_scale_words(int type) { return type == PK_KV_Q8 ? 1 : 2; }

cudaError_t launch_kv_store(const pk_kv_cache &c, const pk_kv_seqs &s, const void *k, const void *v, int type,
                            long tok_stride, long head_stride, cudaStream_t st);
cudaError_t launch_kv_load(const pk_kv_cache &c, const pk_kv_seqs &s, void *k, void *v, int type, long tok_stride,
                           long head_stride, cudaStream_t st);
cudaError_t launch_kv_keep(const pk_kv_cache &c, const pk_kv_seqs &s, const int *keep, int keep_stride,
                           const int *n_keep, cudaStream_t st);

// (0: no partial results)
size_t kv_attn_scratch_bytes(const pk_kv_cache &c, const pk_kv_seqs &s, int n_head, int type);
// err: a device word (or null) that PK_ERR_TIMEOUT is put into when a bounded
// wait runs out; poison: a self-test in which they do.
cudaError_t launch_kv_attn(const pk_kv_cache &c, const pk_kv_seqs &s, const pk_kv_query &q, void *scratch,
                           cudaStream_t st, int *err = nullptr, bool poison = false);
// Whether this call's kernel has bounded waits (the tcgen05 one).
bool kv_attn_waits(const pk_kv_cache &c, const pk_kv_seqs &s, int n_head, int type);

cudaError_t launch_rope(const pk_rope_args &a, cudaStream_t st);
cudaError_t launch_logit_rules(const void *logits, void *out, int type, int rows, int n, long in_stride,
                               long out_stride, const pk_logit_rules &r, cudaStream_t st);

}  // namespace pk
