// tc_step_api.cpp -- argument checks and the extern "C" entry points declared in
// include/tc_step.h.
#include <algorithm>
#include <cmath>
#include <string>

#include "tc_api_util.hpp"
#include "tc_kernels.hpp"
#include "tc_step.hpp"

using namespace tc::api;

namespace {

bool aligned_to(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int check_rope(const tc_rope *r, uint32_t head_dim, tc::RopeArgs *a) {
    if (!r || !r->turns) return refuse(TC_E_ARG, "null pointer");
    if (r->layout != TC_ROPE_HALF && r->layout != TC_ROPE_PAIRS)
        return refuse(TC_E_UNSUPPORTED, "unsupported rope layout " + std::to_string(r->layout));
    if (r->n_rot == 0 || r->n_rot % 2 || r->n_rot > head_dim)
        return refuse(TC_E_UNSUPPORTED, "n_rot=" + std::to_string(r->n_rot) + " is not even, from 2 to the head's size");
    if (!std::isfinite(r->factor)) return refuse(TC_E_ARG, "the rope's factor is not finite");
    if (!aligned_to(r->turns, 8)) return refuse(TC_E_UNSUPPORTED, "turns must be 8-byte aligned");
    *a = {r->turns, r->n_rot, r->n_rot / 2, r->layout, r->factor};
    return TC_OK;
}

// `units` heads of each of n rows: what the kernels count in 32 bits, and the threads of a grid, whose
// workgroups are of 256.
int check_rope_size(uint32_t n, uint64_t units, uint32_t head_dim) {
    if (n * units >= (uint64_t(1) << 31) - 256) return refuse(TC_E_UNSUPPORTED, "2^31 heads of rows or more");
    const uint64_t groups = (units + tc::kRopeUnits - 1) / tc::kRopeUnits;
    if ((n * groups << tc::rope_lane_log(head_dim)) > (uint64_t(1) << 32) - 256)
        return refuse(TC_E_UNSUPPORTED, "2^32 lanes or more (head_dim / 8, up to a power of two, for every 4 heads of a row)");
    return TC_OK;
}

int check_norm(const tc_norm *n, tc::NormArgs *a) {
    *a = {nullptr, nullptr, 0.0f, 0.0f, -1};
    if (!n) return TC_OK;
    if (n->kind != TC_NORM_RMS && n->kind != TC_NORM_LAYER)
        return refuse(TC_E_UNSUPPORTED, "unsupported norm " + std::to_string(n->kind));
    if (!std::isfinite(n->eps) || n->eps < 0.0f) return refuse(TC_E_ARG, "eps is negative or not finite");
    if (!aligned_to(n->weight, 4) || !aligned_to(n->bias, 4))
        return refuse(TC_E_UNSUPPORTED, "a norm's weights must be 4-byte aligned");
    *a = {n->weight, n->bias, n->eps, n->weight ? n->offset : 0.0f, n->kind};
    return TC_OK;
}

// Rows that need no other alignment than their elements'.
int check_norm_rows(const char *name, const void *p, int type, uint32_t stride, const tc_norm_rows &r) {
    if (!row_type(type)) return refuse(TC_E_UNSUPPORTED, std::string(name) + ": unsupported row type " + std::to_string(type));
    if (r.n_rows > 1 && stride < r.cols) return refuse(TC_E_ARG, std::string(name) + ": rows overlap");
    if (!aligned_to(p, tc::elem_bytes(type))) return refuse(TC_E_UNSUPPORTED, std::string(name) + ": not aligned to its type");
    return TC_OK;
}

}  // namespace

extern "C" {

int tc_kv_plan(const tc_plan *p, void *stream) {
    if (!p) return refuse(TC_E_ARG, "null pointer");
    if (p->page_tokens == 0 || p->table_pages == 0 || p->ring_pages == 0)
        return refuse(TC_E_UNSUPPORTED, "empty page, page table or ring");
    if (p->n_seq > (1u << 16) || p->n_tokens > (1u << 24)) return refuse(TC_E_UNSUPPORTED, "more than 2^16 sequences or 2^24 rows");
    if (p->page_tokens > (1u << 30) || p->table_pages > (1u << 30) || p->ring_pages > (1u << 30))
        return refuse(TC_E_UNSUPPORTED, "more than 2^30 tokens in a page, pages in a table or in the ring");
    if (uint64_t(p->n_seq) * p->table_pages > (1u << 30)) return refuse(TC_E_UNSUPPORTED, "more than 2^30 pages in the tables");
    // (arrays without an entry may have no address)
    if (!p->free || !p->free_out || !p->start || !p->ring) return refuse(TC_E_ARG, "null pointer");
    if (p->n_seq != 0 && (!p->new_tokens || !p->held || !p->pages || !p->table || !p->len || !p->pages_out))
        return refuse(TC_E_ARG, "null pointer");
    for (const void *q : {static_cast<const void *>(p->new_tokens), static_cast<const void *>(p->held),
                          static_cast<const void *>(p->pages), static_cast<const void *>(p->free),
                          static_cast<const void *>(p->table), static_cast<const void *>(p->ring),
                          static_cast<const void *>(p->start), static_cast<const void *>(p->len),
                          static_cast<const void *>(p->pages_out), static_cast<const void *>(p->free_out),
                          static_cast<const void *>(p->sequence), static_cast<const void *>(p->position)})
        if (!aligned_to(q, 4)) return refuse(TC_E_UNSUPPORTED, "arrays must be 4-byte aligned");
    if (!aligned_to(p->slot, 8)) return refuse(TC_E_UNSUPPORTED, "slots must be 8-byte aligned");
    if (tc::device_cu_count() == 0) return no_device();
    return hip_rc(tc::launch_plan(*p, static_cast<hipStream_t>(stream)), "step plan");
}

int tc_norm_add(const tc_norm_rows *r, void *stream) {
    if (!r) return refuse(TC_E_ARG, "null pointer");
    tc::NormCall c{};
    int rc;
    if ((rc = check_norm(r->post, &c.post)) || (rc = check_norm(r->pre, &c.pre))) return rc;
    if (r->cols == 0 || r->cols > 32768)
        return refuse(TC_E_UNSUPPORTED, "cols=" + std::to_string(r->cols) + " is not from 1 to 32768");
    if (r->n_rows > 0x7FFFFFFFu) return refuse(TC_E_UNSUPPORTED, "2^31 rows or more");
    if (r->gate_kind < TC_GATE_NONE || r->gate_kind > TC_GATE_FULL)
        return refuse(TC_E_UNSUPPORTED, "unsupported gate " + std::to_string(r->gate_kind));
    if (!std::isfinite(r->scale)) return refuse(TC_E_ARG, "scale is not finite");
    const bool gated = r->gate_kind != TC_GATE_NONE;
    if (gated != (r->gate != nullptr)) return refuse(TC_E_ARG, "a gate goes with its kind");
    if (!r->y && (r->post || gated)) return refuse(TC_E_ARG, "a norm behind the block, or a gate, without the block's output");
    if (!r->pre && (r->x || r->act)) return refuse(TC_E_ARG, "an output of the norm without the norm");
    if (r->n_rows == 0) return TC_OK;
    if (!r->h) return refuse(TC_E_ARG, "null pointer");
    if ((rc = check_norm_rows("h", r->h, r->h_type, r->h_stride, *r))) return rc;
    if (r->y && (rc = check_norm_rows("y", r->y, r->y_type, r->y_stride, *r))) return rc;
    if (r->y && r->h_out && (rc = check_norm_rows("h_out", r->h_out, r->h_type, r->h_out_stride, *r))) return rc;
    if (r->x && (rc = check_norm_rows("x", r->x, r->x_type, r->x_stride, *r))) return rc;
    if (gated && (rc = check_norm_rows("gate", r->gate, r->gate_type, r->cols, *r))) return rc;
    if (r->y && r->h_out == r->h && r->n_rows > 1 && r->h_out_stride != r->h_stride)
        return refuse(TC_E_ARG, "h_out is h with another stride");
    if (r->act) {
        // (the size is 0 where tc_act_quantize refuses the type)
        if (tc_act_bytes(r->act_type, r->n_rows, r->cols) == 0)
            return refuse(TC_E_UNSUPPORTED, "type " + std::to_string(r->act_type) + " has no quantized activations");
        if (r->cols % 256 || r->cols > 12288)
            return refuse(TC_E_UNSUPPORTED, "quantized activations of cols=" + std::to_string(r->cols));
        if (!aligned_to(r->act, 256)) return refuse(TC_E_ARG, "act must be 256-byte aligned");
        const tc::ActLayout L = tc::act_layout(r->act_type, r->n_rows, r->cols);
        char *const base = static_cast<char *>(r->act);
        c.qs = reinterpret_cast<int8_t *>(base + L.qs_off);
        c.d = reinterpret_cast<float *>(base + L.d_off);
        c.bsums = reinterpret_cast<int16_t *>(base + L.bs_off);
        c.dg = reinterpret_cast<uint16_t *>(base + L.dg_off);
        c.act_q8_0 = r->act_type == tc::kQ8_0;
    }
    c.rows = r->n_rows;
    c.cols = r->cols;
    c.h = r->h;
    c.y = r->y;
    c.gate = r->gate;
    c.h_out = r->y ? r->h_out : nullptr;
    c.x = r->x;
    c.h_type = r->h_type, c.y_type = r->y_type, c.x_type = r->x_type;
    c.gate_type = r->gate_type, c.gate_kind = r->gate_kind, c.gate_sigmoid = r->gate_sigmoid;
    c.h_stride = r->h_stride, c.y_stride = r->y_stride, c.h_out_stride = r->h_out_stride, c.x_stride = r->x_stride;
    c.scale = r->scale;
    if (!c.h_out && !c.x && !c.qs) return TC_OK;  // nothing to write
    const int num_cu = tc::device_cu_count();
    if (num_cu == 0) return no_device();
    return hip_rc(tc::launch_norm(c, num_cu, static_cast<hipStream_t>(stream)), "norm");
}

int tc_rope_turns(const tc_rope_scaling *scaling, uint32_t n_rot, double theta, double *turns, float *factor, void *stream) {
    if (!turns || !factor) return refuse(TC_E_ARG, "null pointer");
    if (n_rot == 0 || n_rot % 2 || n_rot > (1u << 16)) return refuse(TC_E_UNSUPPORTED, "n_rot is not even, from 2 to 65536");
    if (!aligned_to(turns, 8)) return refuse(TC_E_UNSUPPORTED, "turns must be 8-byte aligned");
    if (!std::isfinite(theta) || theta <= 0.0) return refuse(TC_E_ARG, "theta is not above 0");
    tc::TurnsCall c{TC_ROPE_NONE, n_rot, theta, 1.0, 0.0, 0.0, 0.0, 0.0, 1.0, nullptr, turns};
    float m = 1.0f;
    if (scaling) {
        const int kind = scaling->kind;
        if (kind < TC_ROPE_NONE || kind > TC_ROPE_BANDS) return refuse(TC_E_UNSUPPORTED, "unsupported scaling " + std::to_string(kind));
        c.kind = kind;
        c.divisors = scaling->divisors;
        if (!aligned_to(c.divisors, 4)) return refuse(TC_E_UNSUPPORTED, "divisors must be 4-byte aligned");
        if (kind != TC_ROPE_NONE) {
            c.factor = scaling->factor;
            if (!std::isfinite(c.factor) || c.factor <= 0.0) return refuse(TC_E_ARG, "the scaling's factor is not above 0");
        }
        if (kind == TC_ROPE_NTK && n_rot <= 2) return refuse(TC_E_ARG, "NTK scaling of a single pair");
        if (kind == TC_ROPE_YARN || kind == TC_ROPE_BANDS) {
            c.original = scaling->original, c.low = scaling->low, c.high = scaling->high;
            if (kind == TC_ROPE_YARN && c.high == 0.0) c.high = 32.0;
            if (kind == TC_ROPE_YARN && c.low == 0.0) c.low = 1.0;
            if (!std::isfinite(c.original) || c.original <= 0.0) return refuse(TC_E_ARG, "the scaling's original length is not above 0");
            if (!std::isfinite(c.low) || !std::isfinite(c.high) || c.low < 0.0 || c.high <= c.low)
                return refuse(TC_E_ARG, "the scaling's high is not above its low");
        }
        if (kind == TC_ROPE_YARN) {
            if (theta <= 1.0) return refuse(TC_E_ARG, "YARN scaling with a theta of 1 or below");
            // the pair that turns r times in `original` positions: original * theta^(-2i/n) = 2 pi r
            auto pair = [&](double r) { return n_rot * std::log(c.original / (r * 6.283185307179586)) / (2.0 * std::log(theta)); };
            c.first = std::max(std::floor(pair(c.high)), 0.0);
            const double last = std::min(std::ceil(pair(c.low)), double(n_rot) - 1.0);
            c.ramp = std::max(last - c.first, 0.001);
            if (c.factor > 1.0) m = float(0.1 * std::log(c.factor) + 1.0);
        }
    }
    if (tc::device_cu_count() == 0) return no_device();
    const int rc = hip_rc(tc::launch_rope_turns(c, static_cast<hipStream_t>(stream)), "rope frequencies");
    if (rc == TC_OK) *factor = m;
    return rc;
}

int tc_rope_apply(const tc_rope *rope, int xtype, const void *x, uint32_t x_stride, void *out, uint32_t out_stride,
                  const int32_t *position, uint32_t n_tokens, uint32_t heads, uint32_t head_dim, void *stream) {
    if (!row_type(xtype)) return refuse(TC_E_UNSUPPORTED, "unsupported row type " + std::to_string(xtype));
    if (head_dim == 0 || head_dim % 16 || head_dim > tc::kMaxHeadDim)
        return refuse(TC_E_UNSUPPORTED, "head_dim=" + std::to_string(head_dim) + " is not a multiple of 16 up to 256");
    if (heads == 0 || heads > 4096) return refuse(TC_E_UNSUPPORTED, "heads=" + std::to_string(heads) + " is not from 1 to 4096");
    tc::RopeCall c{};
    int rc = check_rope(rope, head_dim, &c.rope);
    if (rc) return rc;
    if (n_tokens > (1u << 24)) return refuse(TC_E_UNSUPPORTED, "more than 2^24 rows");
    if ((rc = check_rope_size(n_tokens, heads, head_dim))) return rc;
    if (n_tokens == 0) return TC_OK;
    const uint64_t width = uint64_t(heads) * head_dim;
    if ((rc = check_rows("x", x, x_stride, width, n_tokens, xtype))) return rc;
    if ((rc = check_rows("out", out, out_stride, width, n_tokens, xtype))) return rc;
    if (!position) return refuse(TC_E_ARG, "null pointer");
    if (!aligned_to(position, 4)) return refuse(TC_E_UNSUPPORTED, "positions must be 4-byte aligned");
    if (out == x && n_tokens > 1 && out_stride != x_stride) return refuse(TC_E_ARG, "out is x with another stride");
    if (tc::device_cu_count() == 0) return no_device();
    c.kv.n_tokens = n_tokens;
    c.kv.dim = head_dim;
    c.q = {x, x_stride, heads, nullptr};
    c.q_out = out;
    c.q_out_stride = out_stride;
    c.position = position;
    c.xtype = xtype;
    return hip_rc(tc::launch_rope_rows(c, static_cast<hipStream_t>(stream)), "rope");
}

int tc_rope_kv_write(const tc_kv_cache *cache, const tc_kv_batch *batch, const tc_rope *rope, int xtype, const void *q,
                     uint32_t q_stride, void *q_out, uint32_t heads, const void *k, uint32_t k_stride, const void *v,
                     uint32_t v_stride, const float *q_norm, const float *k_norm, float eps, void *stream) {
    tc::RopeCall c{};
    int rc = kv_args(cache, batch, xtype, &c.kv);
    if (rc) return rc;
    if ((rc = check_rope(rope, c.kv.dim, &c.rope))) return rc;
    if (heads > 4096) return refuse(TC_E_UNSUPPORTED, "heads=" + std::to_string(heads) + " > 4096");
    if (heads == 0 && (q || q_out)) return refuse(TC_E_ARG, "q and q_out go with their heads");
    if (!std::isfinite(eps) || eps < 0.0f) return refuse(TC_E_ARG, "eps is negative or not finite");
    if (!aligned_to(q_norm, 4) || !aligned_to(k_norm, 4))
        return refuse(TC_E_UNSUPPORTED, "a norm's weights must be 4-byte aligned");
    const uint32_t n = c.kv.n_tokens;
    if ((rc = check_rope_size(n, uint64_t(heads) + 2 * c.kv.kv_heads, c.kv.dim))) return rc;
    if (n == 0 || c.kv.n_seq == 0) return TC_OK;
    const uint64_t width = uint64_t(c.kv.kv_heads) * c.kv.dim, q_width = uint64_t(heads) * c.kv.dim;
    if (heads != 0) {
        if ((rc = check_rows("q", q, q_stride, q_width, n, xtype))) return rc;
        if ((rc = check_rows("q_out", q_out, uint32_t(q_width), q_width, n, xtype))) return rc;
    }
    if ((rc = check_rows("k", k, k_stride, width, n, xtype))) return rc;
    if ((rc = check_rows("v", v, v_stride, width, n, xtype))) return rc;
    if (tc::device_cu_count() == 0) return no_device();
    c.q = {q, q_stride, heads, q_norm};
    c.k = {k, k_stride, c.kv.kv_heads, k_norm};
    c.v = {v, v_stride, c.kv.kv_heads, nullptr};
    c.q_out = q_out;
    c.q_out_stride = q_out == q ? q_stride : q_width;  // in place: where q's rows are
    c.eps = eps;
    c.xtype = xtype;
    return hip_rc(tc::launch_rope_kv(c, cache->type, static_cast<hipStream_t>(stream)), "rope and cache write");
}

int tc_logits_adjust(const tc_logit_rules *r, int xtype, const void *logits, uint32_t x_stride, uint32_t vocab,
                     uint32_t n_seq, uint32_t n_tokens, const int32_t *start, const int32_t *tokens, float *out,
                     uint32_t out_stride, void *stream) {
    if (!r) return refuse(TC_E_ARG, "null pointer");
    if (!row_type(xtype)) return refuse(TC_E_UNSUPPORTED, "unsupported row type " + std::to_string(xtype));
    if (vocab == 0 || vocab > (1u << 30) || n_tokens > 65535 || n_seq > 65535)
        return refuse(TC_E_UNSUPPORTED, "an empty vocabulary, more than 2^30 tokens in it, 65535 rows or 65535 sequences");
    // (a token's count, of the history and 65535 rows, has 31 bits)
    if (r->n_history > 0x7FFF0000u || r->n_bias > 0x7FFFFFFFu)
        return refuse(TC_E_UNSUPPORTED, "more than 2^31 - 2^16 tokens of history, or 2^31 biases or more");
    if (r->history_start && r->n_history != 0 && !r->history) return refuse(TC_E_ARG, "a history without its tokens");
    if (r->bias_start && r->n_bias != 0 && (!r->bias_token || !r->bias_value)) return refuse(TC_E_ARG, "biases without tokens or values");
    if (r->mask && uint64_t(r->mask_words) * 32 < vocab) return refuse(TC_E_ARG, "mask_words is too small for the vocabulary");
    if (n_seq == 0 || n_tokens == 0) return TC_OK;
    if (!logits || !out || !start) return refuse(TC_E_ARG, "null pointer");
    if (n_tokens > 1 && (x_stride < vocab || out_stride < vocab)) return refuse(TC_E_ARG, "rows overlap");
    for (const void *p : {static_cast<const void *>(r->repetition), static_cast<const void *>(r->frequency),
                          static_cast<const void *>(r->presence), static_cast<const void *>(r->history),
                          static_cast<const void *>(r->history_start), static_cast<const void *>(r->prompt),
                          static_cast<const void *>(r->bias_start), static_cast<const void *>(r->bias_token),
                          static_cast<const void *>(r->bias_value), static_cast<const void *>(r->mask),
                          static_cast<const void *>(r->mask_of), static_cast<const void *>(start),
                          static_cast<const void *>(tokens), static_cast<const void *>(out)})
        if (!aligned_to(p, 4)) return refuse(TC_E_UNSUPPORTED, "arrays must be 4-byte aligned");
    if (!aligned_to(logits, tc::elem_bytes(xtype))) return refuse(TC_E_UNSUPPORTED, "logits: not aligned to their type");
    if (static_cast<const void *>(out) == logits && (xtype != TC_F32 || (n_tokens > 1 && x_stride != out_stride)))
        return refuse(TC_E_ARG, "out is logits of another type or stride");
    const int num_cu = tc::device_cu_count();
    if (num_cu == 0) return no_device();
    const tc::LogitCall c{*r, logits, out, x_stride, out_stride, xtype, vocab, n_seq, n_tokens, start, tokens};
    return hip_rc(tc::launch_logits(c, num_cu, static_cast<hipStream_t>(stream)), "rules on logits");
}

}  // extern "C"
