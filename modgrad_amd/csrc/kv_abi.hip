// C ABI of the rotary and key/value-cache operators (declarations and
// contracts: include/modgrad_q4k.h). Every argument the host can see is checked
// here, before any device call; device arrays (positions, lengths, page
// tables) are bounded by the kernels themselves.
#include "kv_device.hpp"
#include "kv_launch.hpp"

namespace mgq {
namespace {

bool bad4(const void *p) { return !p || ((uintptr_t)p & 3u); }
bool bad16(const void *p) { return !p || ((uintptr_t)p & 15u); }
constexpr int64_t kMaxGrid = 0x7FFFFFFF;

bool bad_rope(const mgq_rope &r, int head_dim) {
    return bad4(r.table) || r.n_pos <= 0 || r.rot_dim <= 0 || r.rot_dim % 2 || r.rot_dim > 512 ||
           r.rot_dim > head_dim || (r.style != MGQ_ROPE_INTERLEAVED && r.style != MGQ_ROPE_HALF);
}

hipError_t rope_check(const float *x, const float *y, const int *pos, const mgq_rope *r, int n_tokens, int n_heads,
                      int head_dim, int64_t xs, int64_t ys) {
    if (!r || bad4(x) || bad4(y) || bad4(pos) || n_tokens <= 0 || n_heads <= 0 || head_dim <= 0 || head_dim % 2)
        return hipErrorInvalidValue;
    if (bad_rope(*r, head_dim)) return hipErrorInvalidValue;
    const int64_t row = (int64_t)n_heads * head_dim;
    if (row > kMaxGrid || xs < row || ys < row || (x == y && xs != ys)) return hipErrorInvalidValue;
    return row * n_tokens / 512 >= kMaxGrid ? hipErrorInvalidValue : hipSuccess;
}

int page_shift(int tokens) { return tokens == 16 ? 4 : tokens == 32 ? 5 : tokens == 64 ? 6 : tokens == 128 ? 7 : -1; }

// The parts of a cache that every entry point needs.
hipError_t cache_check(const mgq_kv_cache *c) {
    if (!c || bad16(c->k) || bad16(c->v) || bad4(c->k_scale) || bad4(c->v_scale)) return hipErrorInvalidValue;
    if (c->n_pages <= 0 || c->n_kv_heads <= 0 || page_shift(c->page_tokens) < 0) return hipErrorInvalidValue;
    if (c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128 && c->head_dim != 256) return hipErrorInvalidValue;
    if (c->format != MGQ_KV_I8 && c->format != MGQ_KV_E4M3) return hipErrorInvalidValue;
    if (c->n_kv_heads > (1 << 15)) return hipErrorInvalidValue;
    if (c->page_stride % 16 || c->page_stride < (int64_t)c->n_kv_heads * c->page_tokens * c->head_dim)
        return hipErrorInvalidValue;
    return c->page_stride > INT64_MAX / c->n_pages ? hipErrorInvalidValue : hipSuccess;
}

// ... and what a call on sequences needs.
hipError_t call_check(const mgq_kv_cache *c, int n_tokens, int max_new) {
    const hipError_t e = cache_check(c);
    if (e != hipSuccess) return e;
    if (bad4(c->page_table) || bad4(c->seq_len) || (c->cu_tokens && bad4(c->cu_tokens))) return hipErrorInvalidValue;
    if (c->n_seqs <= 0 || c->max_pages <= 0 || n_tokens <= 0 || max_new <= 0) return hipErrorInvalidValue;
    if ((int64_t)c->max_pages * c->page_tokens >= (1 << 30)) return hipErrorInvalidValue;
    if (max_new > n_tokens || (!c->cu_tokens && (max_new != 1 || n_tokens != c->n_seqs))) return hipErrorInvalidValue;
    return hipSuccess;
}

KvView view(const mgq_kv_cache &c, int n_tokens, int max_new) {
    KvView v;
    v.k = static_cast<uint8_t *>(c.k);
    v.v = static_cast<uint8_t *>(c.v);
    v.ks = c.k_scale;
    v.vs = c.v_scale;
    v.table = c.page_table;
    v.len = c.seq_len;
    v.cu = c.cu_tokens;
    v.page_stride = c.page_stride;
    v.n_pages = c.n_pages;
    v.page_shift = page_shift(c.page_tokens);
    v.hkv = c.n_kv_heads;
    v.n_seqs = c.n_seqs;
    v.max_pages = c.max_pages;
    v.n_tokens = n_tokens;
    v.max_new = max_new;
    return v;
}

hipError_t append_check(const mgq_kv_cache *c, const mgq_rope *rope, const float *k, const float *v, int64_t kvs,
                        const float *q, int64_t qs, const float *qo, int64_t qos, int hq, int n_tokens, int max_new) {
    const hipError_t e = call_check(c, n_tokens, max_new);
    if (e != hipSuccess) return e;
    if (bad4(k) || bad4(v) || kvs < (int64_t)c->n_kv_heads * c->head_dim) return hipErrorInvalidValue;
    if (rope && (bad_rope(*rope, c->head_dim) || rope->n_pos < (int64_t)c->max_pages * c->page_tokens))
        return hipErrorInvalidValue;
    if (q) {
        const int64_t row = (int64_t)hq * c->head_dim;
        if (bad4(q) || bad4(qo) || hq <= 0 || row > (1 << 24) || qs < row || qos < row || (q == qo && qs != qos))
            return hipErrorInvalidValue;
    } else if (qo) {
        return hipErrorInvalidValue;
    }
    // work-groups: pages that new tokens may touch, and chunks of query rows
    const int64_t blocks = ((int64_t)max_new + c->page_tokens - 2) / c->page_tokens + 1;
    // query pairs of a sequence are counted in 32 bits
    if (q && (int64_t)max_new * hq * c->head_dim >= (INT64_C(1) << 32)) return hipErrorInvalidValue;
    const int64_t query = q ? (int64_t)max_new * hq * c->head_dim / 512 + 1 : 0;
    const int64_t most = kMaxGrid / c->n_seqs;
    return blocks * 2 * c->n_kv_heads >= most / 2 || query >= most / 2 ? hipErrorInvalidValue : hipSuccess;
}

bool attn_heads_ok(const mgq_kv_cache *c, int hq) {
    return hq > 0 && hq % c->n_kv_heads == 0 && (int64_t)hq * c->head_dim <= (1 << 24);
}

// What the kernels count in 32 bits: query rows and work-groups, and where few rows
// take a call all its tiles.
bool attn_fits(const mgq_kv_cache *c, int hq, int max_new) {
    const int64_t rows = (int64_t)max_new * (hq / c->n_kv_heads);
    if (rows >= (1 << 28)) return false;
    const int64_t lines = (rows + 15) / 16 * c->n_kv_heads;
    if (lines * c->n_seqs > kMaxGrid / 16) return false;
    if (kv_attn_is_wide(c->head_dim, rows)) return true;
    const int64_t tiles = ((int64_t)c->max_pages * c->page_tokens + 63) / 64;
    // the runs of the 512 work-groups at most end up to 511 tiles past the last
    constexpr int64_t kMostTiles = kMaxGrid - 511;
    return lines <= kMostTiles / tiles && lines * tiles <= kMostTiles / c->n_seqs;
}

hipError_t attn_check(const mgq_kv_cache *c, const float *q, int64_t qs, int hq, const void *out, int64_t os, int type,
                      int n_tokens, int max_new, float scale, float softcap, int window, const void *ws, size_t bytes) {
    const hipError_t e = call_check(c, n_tokens, max_new);
    if (e != hipSuccess) return e;
    if (!attn_heads_ok(c, hq) || !attn_fits(c, hq, max_new)) return hipErrorInvalidValue;
    if (type != MGQ_OUT_F32 && type != MGQ_OUT_F16) return hipErrorInvalidValue;
    const int64_t row = (int64_t)hq * c->head_dim;
    if (bad4(q) || !out || ((uintptr_t)out & (type == MGQ_OUT_F32 ? 3u : 1u)) || qs < row || os < row)
        return hipErrorInvalidValue;
    if (!(scale >= 0.0f) || !(softcap >= 0.0f) || window < 0) return hipErrorInvalidValue;
    // as the kernels take them: times log2 e, or scale / softcap
    if (!std::isfinite(scale * 1.4426950408889634f) || !std::isfinite(softcap * 1.4426950408889634f) ||
        (softcap > 0.0f && !std::isfinite(scale / softcap)))
        return hipErrorInvalidValue;
    if (bad16(ws) || bytes < mgq_kv_attention_workspace_bytes(c, hq, max_new)) return hipErrorInvalidValue;
    return hipSuccess;
}

}  // namespace

hipError_t kv_op_check(int op, const void *args) {
    if (!args) return hipErrorInvalidValue;
    if (op == MGQ_OP_ROPE) {
        const auto &a = *static_cast<const mgq_rope_args *>(args);
        return rope_check(a.x, a.y, a.pos, &a.rope, a.n_tokens, a.n_heads, a.head_dim, a.x_stride, a.y_stride);
    }
    if (op == MGQ_OP_KV_APPEND) {
        const auto &a = *static_cast<const mgq_kv_append_args *>(args);
        return append_check(&a.cache, a.rope.table ? &a.rope : nullptr, a.k, a.v, a.kv_stride, a.q, a.q_stride,
                            a.q_out, a.q_out_stride, a.n_q_heads, a.n_tokens, a.max_new);
    }
    const auto &a = *static_cast<const mgq_kv_attention_args *>(args);
    return attn_check(&a.cache, a.q, a.q_stride, a.n_q_heads, a.out, a.out_stride, a.out_type, a.n_tokens, a.max_new,
                      a.scale, a.softcap, a.window, a.workspace, a.workspace_bytes);
}

hipError_t kv_op_launch(int op, const void *args, hipStream_t stream) {
    if (op == MGQ_OP_ROPE) {
        const auto &a = *static_cast<const mgq_rope_args *>(args);
        return launch_rope_ex(a.x, a.y, a.pos, &a.rope, a.n_tokens, a.n_heads, a.head_dim, a.x_stride, a.y_stride,
                              stream);
    }
    if (op == MGQ_OP_KV_APPEND) {
        const auto &a = *static_cast<const mgq_kv_append_args *>(args);
        return launch_kv_append_ex(&a.cache, a.rope.table ? &a.rope : nullptr, a.k, a.v, a.kv_stride, a.q, a.q_stride,
                                   a.q_out, a.q_out_stride, a.n_q_heads, a.n_tokens, a.max_new, stream);
    }
    const auto &a = *static_cast<const mgq_kv_attention_args *>(args);
    return launch_kv_attention_ex(&a.cache, a.q, a.q_stride, a.n_q_heads, a.out, a.out_stride, a.out_type, a.n_tokens,
                                  a.max_new, a.scale, a.softcap, a.window, a.workspace, a.workspace_bytes, stream);
}

}  // namespace mgq

using namespace mgq;

extern "C" {

hipError_t launch_rope_table_ex(float *table, int n_pos, int first_pos, int rot_dim, const mgq_rope_scaling *s,
                                hipStream_t stream) {
    if (bad4(table) || !s || n_pos <= 0 || first_pos < 0 || rot_dim <= 0 || rot_dim % 2 || rot_dim > 512)
        return hipErrorInvalidValue;
    if ((int64_t)first_pos + n_pos > kMaxGrid || (s->factors && bad4(s->factors))) return hipErrorInvalidValue;
    // written so that NaN fails
    if (!(s->base > 0.0) || !(s->freq_scale > 0.0) || !std::isfinite(s->base) || !std::isfinite(s->freq_scale) ||
        !std::isfinite(s->ext_factor) || !std::isfinite(s->attn_factor))
        return hipErrorInvalidValue;
    if (s->ext_factor != 0.0 && (!(s->base > 1.0) || !(s->beta_fast > 0.0) || !(s->beta_slow > 0.0) ||
                                 !(s->orig_ctx > 0.0) || !std::isfinite(s->beta_fast) ||
                                 !std::isfinite(s->beta_slow) || !std::isfinite(s->orig_ctx)))
        return hipErrorInvalidValue;
    return rope_table_launch(table, n_pos, first_pos, rot_dim, *s, stream);
}

hipError_t launch_rope_ex(const float *x, float *y, const int *pos, const mgq_rope *rope, int n_tokens, int n_heads,
                          int head_dim, int64_t x_stride, int64_t y_stride, hipStream_t stream) {
    const hipError_t e = rope_check(x, y, pos, rope, n_tokens, n_heads, head_dim, x_stride, y_stride);
    if (e != hipSuccess) return e;
    return rope_launch(x, y, pos, *rope, n_tokens, n_heads, head_dim, x_stride, y_stride, stream);
}

hipError_t launch_kv_append_ex(const mgq_kv_cache *c, const mgq_rope *rope, const float *k, const float *v,
                               int64_t kv_stride, const float *q, int64_t q_stride, float *q_out,
                               int64_t q_out_stride, int n_q_heads, int n_tokens, int max_new, hipStream_t stream) {
    const hipError_t e = append_check(c, rope, k, v, kv_stride, q, q_stride, q_out, q_out_stride, n_q_heads, n_tokens,
                                      max_new);
    if (e != hipSuccess) return e;
    const KvAppend a = {k, v, kv_stride, q, q_out, q_stride, q_out_stride, n_q_heads};
    return kv_append_launch(view(*c, n_tokens, max_new), c->head_dim, c->format, rope, a, stream);
}

hipError_t launch_kv_dequant_ex(const mgq_kv_cache *c, const int *pages, int n, float *k_out, float *v_out,
                                hipStream_t stream) {
    const hipError_t e = cache_check(c);
    if (e != hipSuccess) return e;
    if (bad4(pages) || n <= 0 || bad4(k_out) || bad4(v_out) || (int64_t)n * c->n_kv_heads * 2 > kMaxGrid)
        return hipErrorInvalidValue;
    return kv_dequant_launch(view(*c, 0, 0), c->head_dim, c->format, pages, n, k_out, v_out, stream);
}

size_t mgq_kv_attention_workspace_bytes(const mgq_kv_cache *c, int n_q_heads, int max_new) {
    if (cache_check(c) != hipSuccess || !attn_heads_ok(c, n_q_heads) || c->n_seqs <= 0 || c->max_pages <= 0 ||
        max_new <= 0 || (int64_t)c->max_pages * c->page_tokens >= (1 << 30) || !attn_fits(c, n_q_heads, max_new))
        return 0;
    return kv_attn_workspace(c->head_dim, n_q_heads, c->n_kv_heads, c->n_seqs, max_new,
                             (int64_t)c->max_pages * c->page_tokens);
}

hipError_t launch_kv_attention_ex(const mgq_kv_cache *c, const float *q, int64_t q_stride, int n_q_heads, void *out,
                                  int64_t out_stride, int out_type, int n_tokens, int max_new, float scale,
                                  float softcap, int window, void *workspace, size_t workspace_bytes,
                                  hipStream_t stream) {
    const hipError_t e = attn_check(c, q, q_stride, n_q_heads, out, out_stride, out_type, n_tokens, max_new, scale,
                                    softcap, window, workspace, workspace_bytes);
    if (e != hipSuccess) return e;
    KvAttn a;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.hq = n_q_heads;
    a.out_f16 = out_type == MGQ_OUT_F16;
    a.scale = scale;
    a.softcap = softcap;
    a.window = window;
    a.ws = static_cast<float *>(workspace);
    return kv_attn_launch(view(*c, n_tokens, max_new), c->head_dim, c->format, a, stream);
}

}  // extern "C"
