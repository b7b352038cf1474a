// C ABI of the serving operators: argument checks and launches. See include/gemq_b200.h
// for the contract.
#include <string>

#include <nvtx3/nvToolsExt.h>

#include "paged.cuh"

namespace gemq {
namespace {

struct TraceRange {
  explicit TraceRange(const char* name) { nvtxRangePushA(name); }
  ~TraceRange() { nvtxRangePop(); }
  TraceRange(const TraceRange&) = delete;
  TraceRange& operator=(const TraceRange&) = delete;
};

int fail(int code, const char* msg) {
  set_error(msg);
  return code;
}

int launched(cudaError_t e, const char* where) {
  if (e == cudaSuccess) return GEMQ_OK;
  set_error(std::string(where) + ": " + cudaGetErrorString(e));
  return GEMQ_ERR_CUDA;
}

// Runs an entry point's body; nothing thrown in it (an error text that cannot be
// allocated) passes the C boundary.
template <typename F>
int guarded(const char* name, F&& body) noexcept {
  try {
    TraceRange trace(name);
    return body();
  } catch (...) {
    return GEMQ_ERR_CUDA;
  }
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int check_cache(const gemq_kv_cache_t* c) {
  if (c == nullptr) return fail(GEMQ_ERR_INVALID_ARGUMENT, "cache: null");
  if (c->bits != 16 && c->bits != 8 && c->bits != 4)
    return fail(GEMQ_ERR_INVALID_ARGUMENT, "cache: bits must be 16, 8 or 4");
  if (c->dtype != GEMQ_FP16 && c->dtype != GEMQ_BF16)
    return fail(GEMQ_ERR_INVALID_ARGUMENT, "cache: dtype must be GEMQ_FP16 or GEMQ_BF16");
  if (c->num_pages <= 0 || c->kv_heads <= 0 || c->page_size <= 0 || c->head_dim <= 0)
    return fail(GEMQ_ERR_INVALID_ARGUMENT, "cache: non-positive size");
  if (c->head_dim % 16 != 0 || c->head_dim > 256)
    return fail(GEMQ_ERR_UNSUPPORTED, "cache: head_dim must be a multiple of 16, at most 256");
  if ((c->page_size & (c->page_size - 1)) != 0 || c->page_size > 65536)
    return fail(GEMQ_ERR_UNSUPPORTED, "cache: page_size must be a power of two, at most 65536");
  if (static_cast<int64_t>(c->num_pages) * c->page_size > INT32_MAX)
    return fail(GEMQ_ERR_UNSUPPORTED, "cache: num_pages * page_size must be below 2^31");
  if (c->k == nullptr || c->v == nullptr || (c->bits != 16 && (c->k_scale == nullptr || c->v_scale == nullptr)))
    return fail(GEMQ_ERR_INVALID_ARGUMENT, "cache: null device pointer");
  const uintptr_t unit = c->bits == 4 && c->head_dim % 32 != 0 ? 8 : 16;
  const uintptr_t sunit = c->bits == 4 ? 8 : 4;
  bool ok = aligned(c->k, unit) && aligned(c->v, unit);
  for (int i = 0; i < 3; ++i) ok = ok && c->strides[i] >= 0 && c->strides[i] % static_cast<int64_t>(unit) == 0;
  if (c->bits != 16) {
    ok = ok && aligned(c->k_scale, sunit) && aligned(c->v_scale, sunit);
    for (int i = 0; i < 3; ++i)
      ok = ok && c->scale_strides[i] >= 0 && (c->bits == 8 || c->scale_strides[i] % 2 == 0);
  }
  if (!ok) return fail(GEMQ_ERR_UNSUPPORTED, "cache: k, v, the scales and the strides must be aligned (16 bytes a row)");
  for (int i = 0; i < 3; ++i)
    if (c->strides[i] / 8 > INT32_MAX || (c->bits != 16 && c->scale_strides[i] > INT32_MAX))
      return fail(GEMQ_ERR_UNSUPPORTED, "cache: a stride of 2^34 bytes or more");
  return GEMQ_OK;
}

KvDev to_dev(const gemq_kv_cache_t& c) {
  KvDev d{};
  d.k = static_cast<uint8_t*>(c.k);
  d.v = static_cast<uint8_t*>(c.v);
  d.k_scale = c.k_scale;
  d.v_scale = c.v_scale;
  d.page_stride = static_cast<uint32_t>(c.strides[0] / 8);
  d.head_stride = static_cast<uint32_t>(c.strides[1] / 8);
  d.token_stride = static_cast<uint32_t>(c.strides[2] / 8);
  d.scale_page_stride = c.bits == 16 ? 0u : static_cast<uint32_t>(c.scale_strides[0]);
  d.scale_head_stride = c.bits == 16 ? 0u : static_cast<uint32_t>(c.scale_strides[1]);
  d.scale_token_stride = c.bits == 16 ? 0u : static_cast<uint32_t>(c.scale_strides[2]);
  d.num_pages = c.num_pages;
  d.kv_heads = c.kv_heads;
  d.page_shift = 0;
  while ((1 << d.page_shift) < c.page_size) ++d.page_shift;
  d.head_dim = c.head_dim;
  return d;
}

int check_rows(const gemq_kv_cache_t* c, int64_t tokens) {
  if (tokens < 0) return fail(GEMQ_ERR_INVALID_ARGUMENT, "tokens must not be negative");
  if (tokens > (int64_t{1} << 29) || tokens * c->kv_heads > (int64_t{1} << 29))
    return fail(GEMQ_ERR_UNSUPPORTED, "tokens * kv_heads above 2^29");
  return GEMQ_OK;
}

// The sizes an attention call's kernels and workspace follow from.
int check_attention(const gemq_kv_cache_t* c, int64_t num_tokens, int32_t q_heads, int32_t num_seqs, int32_t max_pages,
                    int32_t max_q_len, int32_t max_kv_len) {
  if (const int rc = check_cache(c)) return rc;
  if (num_tokens < 0 || num_seqs < 0 || q_heads <= 0 || max_pages < 0 || max_q_len < 0 || max_kv_len < 0)
    return fail(GEMQ_ERR_INVALID_ARGUMENT, "negative size");
  if (q_heads % c->kv_heads != 0)
    return fail(GEMQ_ERR_INVALID_ARGUMENT, "q_heads must be a multiple of the cache's kv_heads");
  if (num_tokens > (int64_t{1} << 29) || num_tokens * q_heads > (int64_t{1} << 29) || num_seqs > (1 << 20))
    return fail(GEMQ_ERR_UNSUPPORTED, "num_tokens * q_heads above 2^29, or more than 2^20 sequences");
  if (static_cast<int64_t>(max_pages) * c->page_size > INT32_MAX)
    return fail(GEMQ_ERR_UNSUPPORTED, "max_pages * page_size must be below 2^31");
  return GEMQ_OK;
}

AttnArgs attn_sizes(const gemq_kv_cache_t* c, int64_t num_tokens, int32_t q_heads, int32_t num_seqs, int32_t max_pages) {
  AttnArgs a{};
  a.kv = to_dev(*c);
  a.num_tokens = static_cast<int>(num_tokens);
  a.num_seqs = num_seqs;
  a.q_heads = q_heads;
  a.group = q_heads / c->kv_heads;
  a.max_pages = max_pages;
  return a;
}

// The bounds that choose kernel and split: what the caller said, within what there is.
int bound_q(int32_t max_q_len, int64_t num_tokens) {
  return max_q_len > 0 && max_q_len < num_tokens ? max_q_len : static_cast<int>(num_tokens);
}
int bound_kv(const gemq_kv_cache_t* c, int32_t max_kv_len, int32_t max_pages) {
  const int all = max_pages * c->page_size;
  return max_kv_len > 0 && max_kv_len < all ? max_kv_len : all;
}

}  // namespace
}  // namespace gemq

using namespace gemq;

extern "C" {

int gemq_kv_cache_write(const gemq_kv_cache_t* cache, const void* k, const void* v, int64_t k_token_stride,
                        int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, const int64_t* slots,
                        int64_t tokens, void* stream) {
  return guarded("gemq_kv_cache_write", [&]() -> int {
    if (const int rc = check_cache(cache)) return rc;
    if (const int rc = check_rows(cache, tokens)) return rc;
    if (tokens == 0) return GEMQ_OK;
    if (k == nullptr || v == nullptr || slots == nullptr) return fail(GEMQ_ERR_INVALID_ARGUMENT, "null pointer");
    if (!aligned(k, 16) || !aligned(v, 16) || k_token_stride % 8 != 0 || k_head_stride % 8 != 0 ||
        v_token_stride % 8 != 0 || v_head_stride % 8 != 0)
      return fail(GEMQ_ERR_UNSUPPORTED, "rows of k and v must start on a 16-byte boundary");
    return launched(launch_cache_write(to_dev(*cache), cache->bits, cache->dtype == GEMQ_BF16, k, v, k_token_stride,
                                       k_head_stride, v_token_stride, v_head_stride, slots, static_cast<int>(tokens),
                                       static_cast<cudaStream_t>(stream)),
                    "kv cache write");
  });
}

int gemq_kv_cache_read(const gemq_kv_cache_t* cache, const int64_t* slots, int64_t tokens, void* k_out, void* v_out,
                       void* stream) {
  return guarded("gemq_kv_cache_read", [&]() -> int {
    if (const int rc = check_cache(cache)) return rc;
    if (const int rc = check_rows(cache, tokens)) return rc;
    if (tokens == 0) return GEMQ_OK;
    if (k_out == nullptr || v_out == nullptr || slots == nullptr)
      return fail(GEMQ_ERR_INVALID_ARGUMENT, "null pointer");
    if (!aligned(k_out, 16) || !aligned(v_out, 16))
      return fail(GEMQ_ERR_UNSUPPORTED, "k_out and v_out must start on a 16-byte boundary");
    return launched(launch_cache_read(to_dev(*cache), cache->bits, cache->dtype == GEMQ_BF16, slots,
                                      static_cast<int>(tokens), k_out, v_out, static_cast<cudaStream_t>(stream)),
                    "kv cache read");
  });
}

size_t gemq_paged_attention_workspace_size(const gemq_kv_cache_t* cache, int64_t num_tokens, int32_t q_heads,
                                           int32_t num_seqs, int32_t max_pages, int32_t max_q_len,
                                           int32_t max_kv_len) {
  size_t bytes = 0;
  guarded("gemq_paged_attention_workspace_size", [&]() -> int {
    if (const int rc = check_attention(cache, num_tokens, q_heads, num_seqs, max_pages, max_q_len, max_kv_len)) return rc;
    if (num_tokens == 0 || num_seqs == 0) return GEMQ_OK;
    bytes = attention_workspace(attn_sizes(cache, num_tokens, q_heads, num_seqs, max_pages), cache->bits,
                                cache->dtype == GEMQ_BF16,
                                bound_q(max_q_len, num_tokens), bound_kv(cache, max_kv_len, max_pages));
    return GEMQ_OK;
  });
  return bytes;
}

int gemq_paged_attention(const gemq_kv_cache_t* cache, const void* q, int64_t q_token_stride, int64_t num_tokens,
                         int32_t q_heads, const int32_t* page_table, int64_t page_table_stride, int32_t max_pages,
                         const int32_t* kv_lens, const int32_t* q_starts, int32_t num_seqs, int32_t max_q_len,
                         int32_t max_kv_len, float scale, int32_t window, void* out, float* lse, void* workspace,
                         size_t workspace_bytes, void* stream) {
  return guarded("gemq_paged_attention", [&]() -> int {
    if (const int rc = check_attention(cache, num_tokens, q_heads, num_seqs, max_pages, max_q_len, max_kv_len)) return rc;
    if (window < 0) return fail(GEMQ_ERR_INVALID_ARGUMENT, "window must not be negative (0: none)");
    if (!(scale > -INFINITY && scale < INFINITY)) return fail(GEMQ_ERR_INVALID_ARGUMENT, "scale must be finite");
    if (num_tokens == 0 || num_seqs == 0) return GEMQ_OK;
    if (q_starts == nullptr && num_tokens % num_seqs != 0)
      return fail(GEMQ_ERR_INVALID_ARGUMENT, "without q_starts num_tokens must be a multiple of num_seqs");
    if (q == nullptr || (page_table == nullptr && max_pages > 0) || kv_lens == nullptr || out == nullptr)
      return fail(GEMQ_ERR_INVALID_ARGUMENT, "null pointer");
    if (page_table_stride < 0) return fail(GEMQ_ERR_INVALID_ARGUMENT, "page_table_stride must not be negative");
    if (!aligned(q, 16) || !aligned(out, 16) || q_token_stride % 8 != 0 || q_token_stride < 0)
      return fail(GEMQ_ERR_UNSUPPORTED, "q and out must start on a 16-byte boundary, q's token stride be a multiple of 8");
    AttnArgs a = attn_sizes(cache, num_tokens, q_heads, num_seqs, max_pages);
    const int mq = bound_q(max_q_len, num_tokens), mk = bound_kv(cache, max_kv_len, max_pages);
    const size_t need = attention_workspace(a, cache->bits, cache->dtype == GEMQ_BF16, mq, mk);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
      return fail(GEMQ_ERR_WORKSPACE, "workspace too small or unaligned");
    a.q = q;
    a.q_token_stride = q_token_stride;
    a.page_table = page_table;
    a.page_table_stride = page_table_stride;
    a.kv_lens = kv_lens;
    a.q_starts = q_starts;
    a.scale = scale;
    a.window = window;
    a.out = out;
    a.lse = lse;
    return launched(launch_attention(a, cache->bits, cache->dtype == GEMQ_BF16, mq, mk, workspace,
                                     static_cast<cudaStream_t>(stream)),
                    "paged attention");
  });
}

size_t gemq_verify_draft_workspace_size(int32_t num_seqs, int32_t num_drafts, int32_t vocab) {
  if (num_seqs <= 0 || num_seqs > 65535 || num_drafts <= 0 || num_drafts > 63 || vocab <= 0 || vocab >= 1 << 30)
    return 0;
  return verify_workspace(num_seqs, num_drafts, vocab);
}

int gemq_verify_draft(const gemq_verify_t* v, int32_t num_seqs, int32_t num_drafts, int32_t vocab, void* workspace,
                      size_t workspace_bytes, void* stream) {
  return guarded("gemq_verify_draft", [&]() -> int {
    if (v == nullptr) return fail(GEMQ_ERR_INVALID_ARGUMENT, "null arguments");
    if (num_seqs < 0 || num_drafts <= 0 || num_drafts > 63 || vocab <= 0)
      return fail(GEMQ_ERR_INVALID_ARGUMENT, "num_drafts must be 1 to 63, vocab positive");
    if (num_seqs > 65535 || vocab >= 1 << 30)
      return fail(GEMQ_ERR_UNSUPPORTED, "num_seqs above 65535 or vocab of 2^30 and more");
    if (num_seqs == 0) return GEMQ_OK;
    if (v->logits == nullptr || v->draft_tokens == nullptr || v->uniforms == nullptr || v->noise == nullptr ||
        v->tokens == nullptr || v->num_accepted == nullptr || v->logprobs == nullptr)
      return fail(GEMQ_ERR_INVALID_ARGUMENT, "null pointer");
    if (v->logits_dtype < GEMQ_FP16 || v->logits_dtype > GEMQ_FP32 ||
        (v->draft_probs != nullptr && (v->probs_dtype < GEMQ_FP16 || v->probs_dtype > GEMQ_FP32)))
      return fail(GEMQ_ERR_INVALID_ARGUMENT, "dtype must be GEMQ_FP16, GEMQ_BF16 or GEMQ_FP32");
    const uintptr_t lu = v->logits_dtype == GEMQ_FP32 ? 4 : 2, pu = v->probs_dtype == GEMQ_FP32 ? 4 : 2;
    if (!aligned(v->logits, lu) || !aligned(v->draft_probs, pu) || v->logits_seq_stride < 0 ||
        v->logits_row_stride < 0 || v->probs_seq_stride < 0 || v->probs_row_stride < 0)
      return fail(GEMQ_ERR_INVALID_ARGUMENT, "unaligned pointer or negative stride");
    if (workspace == nullptr || workspace_bytes < verify_workspace(num_seqs, num_drafts, vocab) ||
        !aligned(workspace, 16))
      return fail(GEMQ_ERR_WORKSPACE, "workspace too small or unaligned");
    return launched(launch_verify(*v, num_seqs, num_drafts, vocab, workspace, static_cast<cudaStream_t>(stream)),
                    "verify draft");
  });
}

}  // extern "C"
