// tc_attn_api.cpp -- argument checks and the extern "C" entry points declared in
// include/tc_attention.h.
#include <cmath>
#include <string>

#include "tc_api_util.hpp"

namespace tc {
namespace api {

int kv_args(const tc_kv_cache *c, const tc_kv_batch *b, int xtype, tc::KvArgs *a) {
    if (!c || !b) return refuse(TC_E_ARG, "null pointer");
    if (c->type != TC_F16 && c->type != TC_BF16 && c->type != TC_I8 && c->type != TC_E4M3)
        return refuse(TC_E_UNSUPPORTED, "unsupported cache type " + std::to_string(c->type));
    if (!row_type(xtype)) return refuse(TC_E_UNSUPPORTED, "unsupported row type " + std::to_string(xtype));
    // (arrays without an entry may have no address)
    if (!c->k || !c->v || !b->start || (b->n_seq != 0 && (!b->len || !b->table))) return refuse(TC_E_ARG, "null pointer");
    const bool scaled = tc::scaled_type(c->type);
    if (scaled != (c->k_scale != nullptr) || scaled != (c->v_scale != nullptr))
        return refuse(TC_E_ARG, "scales go with the 8-bit types and with these only");
    if (c->n_pages == 0 || c->kv_heads == 0 || c->head_dim == 0 || c->page_tokens == 0 || b->table_pages == 0)
        return refuse(TC_E_UNSUPPORTED, "empty cache or page table");
    if (c->head_dim % 16 || c->head_dim > tc::kMaxHeadDim)
        return refuse(TC_E_UNSUPPORTED, "head_dim=" + std::to_string(c->head_dim) + " is not a multiple of 16 up to 256");
    if (c->page_tokens % 16 || c->page_tokens > (1u << 30))
        return refuse(TC_E_UNSUPPORTED, "page_tokens=" + std::to_string(c->page_tokens) + " is not a multiple of 16 up to 2^30");
    if (c->kv_heads > 4096) return refuse(TC_E_UNSUPPORTED, "kv_heads=" + std::to_string(c->kv_heads) + " > 4096");
    if (c->n_pages > 0x7FFFFFFFu || b->n_seq > (1u << 20) || b->n_tokens > (1u << 24))
        return refuse(TC_E_UNSUPPORTED, "more than 2^31 - 1 pages, 2^20 sequences or 2^24 rows");
    // (the kernels work on 2^31 parts of rows at most)
    if ((uint64_t(b->n_tokens) + 15) * 2 * c->kv_heads >= (uint64_t(1) << 31))
        return refuse(TC_E_UNSUPPORTED, "too many rows");
    // (runs of 16 rows are numbered in 32 bits)
    if (uint64_t(c->n_pages) * c->kv_heads > (uint64_t(1) << 48) / c->page_tokens ||
        uint64_t(c->n_pages) * c->kv_heads * (c->page_tokens / 16) >= 0xFFFFFFFFu)
        return refuse(TC_E_UNSUPPORTED, "2^36 cache rows or more");
    for (const void *p : {c->k, c->v})
        if (!aligned16(p)) return refuse(TC_E_UNSUPPORTED, "the cache must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale) |
         reinterpret_cast<uintptr_t>(b->start) | reinterpret_cast<uintptr_t>(b->len) | reinterpret_cast<uintptr_t>(b->table)) & 3)
        return refuse(TC_E_UNSUPPORTED, "scales and batch arrays must be 4-byte aligned");
    a->k = static_cast<uint8_t *>(c->k);
    a->v = static_cast<uint8_t *>(c->v);
    a->ks = c->k_scale;
    a->vs = c->v_scale;
    a->n_pages = c->n_pages;
    a->kv_heads = c->kv_heads;
    a->page = c->page_tokens;
    a->dim = c->head_dim;
    a->page_div = tc::make_divmod(c->page_tokens);
    a->start = b->start;
    a->len = b->len;
    a->table = b->table;
    a->n_seq = b->n_seq;
    a->n_tokens = b->n_tokens;
    a->table_pages = b->table_pages;
    return TC_OK;
}

int check_rows(const char *name, const void *p, uint32_t stride, uint64_t width, uint32_t n, int xtype) {
    if (!p) return refuse(TC_E_ARG, "null pointer");
    if (n > 1 && stride < width) return refuse(TC_E_ARG, std::string(name) + ": rows overlap");
    if (!aligned16(p) || (n > 1 && uint64_t(stride) * tc::elem_bytes(xtype) % 16))
        return refuse(TC_E_UNSUPPORTED, std::string(name) + ": rows must be 16-byte aligned");
    return TC_OK;
}

}  // namespace api
}  // namespace tc

using namespace tc::api;

extern "C" {

int tc_kv_write(const tc_kv_cache *cache, const tc_kv_batch *batch, int xtype, const void *k, const void *v,
                uint32_t k_stride, uint32_t v_stride, void *stream) {
    tc::KvArgs a;
    int rc = kv_args(cache, batch, xtype, &a);
    if (rc) return rc;
    if (a.n_tokens == 0 || a.n_seq == 0) return TC_OK;
    const uint64_t width = uint64_t(a.kv_heads) * a.dim;
    if ((rc = check_rows("k", k, k_stride, width, a.n_tokens, xtype))) return rc;
    if ((rc = check_rows("v", v, v_stride, width, a.n_tokens, xtype))) return rc;
    if (tc::device_cu_count() == 0) return no_device();
    return hip_rc(tc::launch_kv_write(a, cache->type, xtype, k, v, k_stride, v_stride, static_cast<hipStream_t>(stream)),
                  "cache write");
}

int tc_kv_read(const tc_kv_cache *cache, const tc_kv_batch *batch, int xtype, void *k, void *v, void *stream) {
    tc::KvArgs a;
    int rc = kv_args(cache, batch, xtype, &a);
    if (rc) return rc;
    if (a.n_tokens == 0 || a.n_seq == 0) return TC_OK;
    if (!k || !v) return refuse(TC_E_ARG, "null pointer");
    if (!aligned16(k) || !aligned16(v)) return refuse(TC_E_UNSUPPORTED, "rows must be 16-byte aligned");
    if (tc::device_cu_count() == 0) return no_device();
    return hip_rc(tc::launch_kv_read(a, cache->type, xtype, k, v, static_cast<hipStream_t>(stream)), "cache read");
}

int tc_attn(const tc_kv_cache *cache, const tc_kv_batch *batch, int xtype, const void *q, uint32_t q_stride, void *out,
            uint32_t heads, float scale, uint32_t window, void *stream) {
    tc::AttnArgs a;
    int rc = kv_args(cache, batch, xtype, &a.kv);
    if (rc) return rc;
    if (heads == 0 || heads % a.kv.kv_heads || heads > 4096)
        return refuse(TC_E_UNSUPPORTED, "heads=" + std::to_string(heads) + " is not a multiple of the cache's up to 4096");
    if (!std::isfinite(scale) || scale < 0.0f) return refuse(TC_E_ARG, "scale is negative or not finite");
    const uint32_t n = a.kv.n_tokens;
    if (n == 0 || a.kv.n_seq == 0) return TC_OK;
    if ((rc = check_rows("q", q, q_stride, uint64_t(heads) * a.kv.dim, n, xtype))) return rc;
    if ((rc = check_rows("out", out, heads * a.kv.dim, uint64_t(heads) * a.kv.dim, n, xtype))) return rc;
    if (uint64_t(n) * heads >= (uint64_t(1) << 31)) return refuse(TC_E_UNSUPPORTED, "2^31 rows of heads or more");
    a.q = q;
    a.out = out;
    a.heads = heads;
    a.group = heads / a.kv.kv_heads;
    a.group_div = tc::make_divmod(a.group);
    a.q_stride = n > 1 ? q_stride : heads * a.kv.dim;
    a.scale = scale;
    a.cap = int32_t(std::min(uint64_t(a.kv.table_pages) * a.kv.page, uint64_t(tc::kMaxPos - 64)));
    a.span = window == 0 ? INT32_MAX : int32_t(std::min(window, uint32_t(INT32_MAX)));
    a.xtype = xtype;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int num_cu = tc::device_cu_count();
    if (num_cu == 0) return no_device();
    void *scratch = nullptr;
    const size_t need = tc::attn_scratch_bytes(num_cu);
    if (need != 0 && !(scratch = tc::aux_scratch(need, st))) return TC_E_LAUNCH;
    return hip_rc(tc::launch_attn(a, cache->type, num_cu, scratch, st), "attention");
}

int tc_attn_reserve(uint32_t heads, uint32_t n_tokens) {
    if (heads == 0 || n_tokens == 0) return TC_OK;
    if (heads > 4096 || n_tokens > (1u << 24)) return refuse(TC_E_UNSUPPORTED, "more than 4096 heads or 2^24 rows");
    const int num_cu = tc::device_cu_count();
    if (num_cu == 0) return no_device();
    size_t need = tc::attn_scratch_bytes(num_cu);
    if (n_tokens <= 65535) need = std::max(need, tc::verify_scratch_bytes(n_tokens, n_tokens));
    return tc::aux_scratch(need, nullptr) ? TC_OK : TC_E_LAUNCH;
}

int tc_spec_verify(const float *logits, const float *draft_probs, uint32_t vocab, uint32_t n_seq, uint32_t n_tokens,
                   const int32_t *start, const int32_t *tokens, const float *temperature, const float *accept_u,
                   const float *sample_u, int32_t *n_accepted, int32_t *next_token, void *stream) {
    if (n_seq == 0) return TC_OK;
    if (!logits || !start || !tokens || !temperature || !accept_u || !sample_u || !n_accepted || !next_token)
        return refuse(TC_E_ARG, "null pointer");
    if (vocab == 0 || n_tokens == 0) return refuse(TC_E_UNSUPPORTED, "no rows or an empty vocabulary");
    if (vocab > (1u << 30) || n_tokens > 65535 || n_seq > 65535)
        return refuse(TC_E_UNSUPPORTED, "more than 2^30 tokens in the vocabulary, 65535 rows or 65535 sequences");
    for (const void *p : {static_cast<const void *>(logits), static_cast<const void *>(draft_probs),
                          static_cast<const void *>(start), static_cast<const void *>(tokens),
                          static_cast<const void *>(temperature), static_cast<const void *>(accept_u),
                          static_cast<const void *>(sample_u), static_cast<const void *>(n_accepted),
                          static_cast<const void *>(next_token)})
        if (reinterpret_cast<uintptr_t>(p) & 3) return refuse(TC_E_UNSUPPORTED, "arrays must be 4-byte aligned");
    const tc::VerifyArgs a{logits, draft_probs, vocab, n_seq, n_tokens, start, tokens, temperature, accept_u,
                           sample_u, n_accepted, next_token};
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int num_cu = tc::device_cu_count();
    if (num_cu == 0) return no_device();
    void *scratch = tc::aux_scratch(tc::verify_scratch_bytes(n_tokens, n_seq), st);
    if (!scratch) return TC_E_LAUNCH;
    return hip_rc(tc::launch_verify(a, num_cu, scratch, st), "draft verification");
}

}  // extern "C"
