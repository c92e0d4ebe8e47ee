// C ABI of the text-stage attention (include/bonsai_cuda.h): argument checks,
// then the launchers of text_attention.cu.
#include "../../include/bonsai_cuda.h"
#include "internal.cuh"

#include <cmath>

using namespace bonsai;

namespace {

bool aligned(const void* data) { return (reinterpret_cast<uintptr_t>(data) & 15) == 0; }
// A TMA stride: a positive multiple of 16 bytes below 2^40 (unused where the
// dimension has one element).
bool stride_ok(long long s, long long size) { return size <= 1 || (s > 0 && s % 8 == 0 && s < (1ll << 39)); }

int check_heads(const char* fn, const char* name, const bonsai_heads_t* t, int tokens, int heads,
                TextTensor* out) {
  const std::string at = std::string(fn) + ": " + name;
  if (!t || !t->data) return fail(BONSAI_ERR_ARG, at + " is null");
  if (!aligned(t->data)) return fail(BONSAI_ERR_ARG, at + " must be 16-byte aligned");
  if (!stride_ok(t->stride_token, tokens) || !stride_ok(t->stride_head, heads))
    return fail(BONSAI_ERR_ARG, at + ": strides must be positive multiples of 8 elements");
  out->data = t->data;
  out->token = tokens > 1 ? t->stride_token : 0;
  out->head = heads > 1 ? t->stride_head : 0;
  return 0;
}

int check_pages(const char* fn, const char* name, const bonsai_pages_t* t, int heads, TextTensor* out) {
  const std::string at = std::string(fn) + ": " + name;
  if (!t || !t->data) return fail(BONSAI_ERR_ARG, at + " is null");
  if (!aligned(t->data)) return fail(BONSAI_ERR_ARG, at + " must be 16-byte aligned");
  if (t->n_pages <= 0) return fail(BONSAI_ERR_ARG, at + " has no pages");
  if (t->page_size < 8 || t->page_size > 65536 || (t->page_size & (t->page_size - 1)) != 0)
    return fail(BONSAI_ERR_UNSUPPORTED, at + ": page_size must be a power of two from 8 to 65536");
  if (!stride_ok(t->stride_page, t->n_pages) || !stride_ok(t->stride_token, t->page_size) ||
      !stride_ok(t->stride_head, heads))
    return fail(BONSAI_ERR_ARG, at + ": strides must be positive multiples of 8 elements");
  out->data = t->data;
  out->page = t->n_pages > 1 ? t->stride_page : 0;
  out->token = t->stride_token;
  out->head = heads > 1 ? t->stride_head : 0;
  return 0;
}

int check_shape(const char* fn, int n_seqs, int total, int n_heads, int n_kv, int head_dim, int dtype,
                float scale) {
  const std::string at = std::string(fn) + ": ";
  if (n_seqs < 0 || total < 0) return fail(BONSAI_ERR_ARG, at + "negative count");
  if (n_heads <= 0 || n_kv <= 0 || n_heads % n_kv != 0)
    return fail(BONSAI_ERR_ARG, at + "n_heads must be a positive multiple of n_kv_heads");
  if (n_heads / n_kv > 128)
    return fail(BONSAI_ERR_UNSUPPORTED, at + "more than 128 query heads to one key/value head");
  if (head_dim != 64 && head_dim != 128)
    return fail(BONSAI_ERR_UNSUPPORTED, at + "head_dim must be 64 or 128");
  if (dtype != BONSAI_DTYPE_F16 && dtype != BONSAI_DTYPE_BF16)
    return fail(BONSAI_ERR_ARG, at + "unknown dtype");
  if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(BONSAI_ERR_ARG, at + "scale must be positive");
  return 0;
}

int log2_of(int pow2) {
  int s = 0;
  while ((1 << s) < pow2) ++s;
  return s;
}

}  // namespace

extern "C" {

int bonsai_prompt_attention(const bonsai_heads_t* q, const bonsai_heads_t* k, const bonsai_heads_t* v,
                            const int* cu_seqlens, int n_seqs, int total_tokens, int n_heads,
                            int n_kv_heads, int head_dim, int dtype, int causal, float scale,
                            const bonsai_heads_t* out, void* stream) {
  static const char* fn = "prompt_attention";
  int rc = check_shape(fn, n_seqs, total_tokens, n_heads, n_kv_heads, head_dim, dtype, scale);
  if (rc) return rc;
  if (n_seqs == 0 || total_tokens == 0) return 0;
  TextAttention a;
  if ((rc = check_heads(fn, "q", q, total_tokens, n_heads, &a.q))) return rc;
  if ((rc = check_heads(fn, "k", k, total_tokens, n_kv_heads, &a.k))) return rc;
  if ((rc = check_heads(fn, "v", v, total_tokens, n_kv_heads, &a.v))) return rc;
  if ((rc = check_heads(fn, "out", out, total_tokens, n_heads, &a.out))) return rc;
  if (!cu_seqlens) return fail(BONSAI_ERR_ARG, "prompt_attention: cu_seqlens is null");
  a.cu = cu_seqlens;
  a.n_seqs = n_seqs;
  a.total_q = total_tokens;
  a.max_ctx = total_tokens;
  a.n_heads = n_heads;
  a.n_kv = n_kv_heads;
  a.head_dim = head_dim;
  a.bf16 = dtype == BONSAI_DTYPE_BF16;
  a.causal = causal != 0;
  a.scale = scale;
  return launch_text_attention(a, static_cast<cudaStream_t>(stream));
}

int bonsai_paged_append(const bonsai_heads_t* k, const bonsai_heads_t* v, const bonsai_pages_t* k_cache,
                        const bonsai_pages_t* v_cache, const int* page_table, long long table_ld,
                        int table_width, const int* cu_q, const int* ctx_lens, int n_seqs, int total_q,
                        int n_kv_heads, int head_dim, void* stream) {
  static const char* fn = "paged_append";
  int rc = check_shape(fn, n_seqs, total_q, n_kv_heads, n_kv_heads, head_dim, BONSAI_DTYPE_F16, 1.0f);
  if (rc) return rc;
  if (n_seqs == 0 || total_q == 0) return 0;
  TextTensor tk, tv, kc, vc;
  if ((rc = check_heads(fn, "k", k, total_q, n_kv_heads, &tk))) return rc;
  if ((rc = check_heads(fn, "v", v, total_q, n_kv_heads, &tv))) return rc;
  if ((rc = check_pages(fn, "k_cache", k_cache, n_kv_heads, &kc))) return rc;
  if ((rc = check_pages(fn, "v_cache", v_cache, n_kv_heads, &vc))) return rc;
  if (k_cache->n_pages != v_cache->n_pages || k_cache->page_size != v_cache->page_size)
    return fail(BONSAI_ERR_ARG, "paged_append: k_cache and v_cache must have the same pages");
  if (!page_table || !cu_q || !ctx_lens) return fail(BONSAI_ERR_ARG, "paged_append: null page_table, cu_q or ctx_lens");
  if (table_width < 0 || table_ld < table_width)
    return fail(BONSAI_ERR_ARG, "paged_append: table_ld smaller than table_width");
  return launch_paged_append(tk, tv, kc, vc, page_table, table_ld, table_width, log2_of(k_cache->page_size),
                             k_cache->n_pages, cu_q, ctx_lens, n_seqs, total_q, n_kv_heads, head_dim,
                             static_cast<cudaStream_t>(stream));
}

int bonsai_paged_attention(const bonsai_heads_t* q, const bonsai_pages_t* k_cache, const bonsai_pages_t* v_cache,
                           const int* page_table, long long table_ld, int table_width, const int* cu_q,
                           const int* ctx_lens, int n_seqs, int total_q, int max_ctx, int n_heads,
                           int n_kv_heads, int head_dim, int dtype, float scale, const bonsai_heads_t* out,
                           void* stream) {
  static const char* fn = "paged_attention";
  int rc = check_shape(fn, n_seqs, total_q, n_heads, n_kv_heads, head_dim, dtype, scale);
  if (rc) return rc;
  if (max_ctx < 0) return fail(BONSAI_ERR_ARG, "paged_attention: negative max_ctx");
  if (n_seqs == 0 || total_q == 0) return 0;
  TextAttention a;
  if ((rc = check_heads(fn, "q", q, total_q, n_heads, &a.q))) return rc;
  if ((rc = check_pages(fn, "k_cache", k_cache, n_kv_heads, &a.k))) return rc;
  if ((rc = check_pages(fn, "v_cache", v_cache, n_kv_heads, &a.v))) return rc;
  if ((rc = check_heads(fn, "out", out, total_q, n_heads, &a.out))) return rc;
  if (k_cache->n_pages != v_cache->n_pages || k_cache->page_size != v_cache->page_size)
    return fail(BONSAI_ERR_ARG, "paged_attention: k_cache and v_cache must have the same pages");
  if (!page_table || !cu_q || !ctx_lens)
    return fail(BONSAI_ERR_ARG, "paged_attention: null page_table, cu_q or ctx_lens");
  if (table_width < 0 || table_ld < table_width)
    return fail(BONSAI_ERR_ARG, "paged_attention: table_ld smaller than table_width");
  a.cu = cu_q;
  a.ctx = ctx_lens;
  a.table = page_table;
  a.table_ld = table_ld;
  a.table_width = table_width;
  a.page_shift = log2_of(k_cache->page_size);
  a.n_pages = k_cache->n_pages;
  a.n_seqs = n_seqs;
  a.total_q = total_q;
  a.max_ctx = max_ctx;
  a.n_heads = n_heads;
  a.n_kv = n_kv_heads;
  a.head_dim = head_dim;
  a.bf16 = dtype == BONSAI_DTYPE_BF16;
  a.causal = true;
  a.scale = scale;
  return launch_text_attention(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
