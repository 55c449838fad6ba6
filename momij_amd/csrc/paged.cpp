// paged.cpp -- C entries of the pages of many sequences and of their drafts' acceptance: argument checks,
// workspaces, launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "mj_abi_internal.h"
#include "mj_paged.h"

namespace {

constexpr int kMaxGroup = 64;            // query heads a KV head
constexpr int kMaxTokens = 1 << 30;      // tokens a table row can hold
constexpr int kMaxRowsInAll = 65535;
constexpr int kMaxVocab = 1 << 23;
constexpr int kMaxPages = 1 << 28;       // (16 KB each at least)

mj_status check_pages(mj_ctx* ctx, const mj_pages* c, const char* what, PgPool& p) {
    if (!c || !c->k || !c->v || !c->table || !c->lens || !c->refs)
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: null pointer in the pages", what);
    if (c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128 && c->page_tokens != 256)
        return mj_fail(ctx, MJ_UNSUPPORTED_SHAPE, "%s: page_tokens=%d (32, 64, 128 or 256)", what,
                       c->page_tokens);
    if (c->n_kv_heads < 1 || c->n_kv_heads > 1024 || c->n_pages < 1 || c->n_pages > kMaxPages || c->n_layers < 1 ||
        c->n_layers > PG_MAX_LAYERS || c->n_seqs < 1 || c->n_seqs > PG_MAX_SEQS || c->table_stride < 1 ||
        (int64_t)c->table_stride * c->page_tokens > kMaxTokens)
        return mj_fail(ctx, MJ_INVALID_ARG,
                       "%s: n_layers=%d n_kv_heads=%d n_pages=%d n_seqs=%d table_stride=%d", what,
                       c->n_layers, c->n_kv_heads, c->n_pages, c->n_seqs, c->table_stride);
    if (!aligned16({c->k, c->v, c->table, c->lens, c->refs, c->served}))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: the pages' arrays need 16-byte alignment", what);
    int shift = 5;
    while (1 << shift < c->page_tokens) ++shift;
    p = PgPool{(uint16_t*)c->k, (uint16_t*)c->v, c->table, c->lens, c->refs, c->served, c->n_kv_heads,
               c->n_pages, c->page_tokens, shift, c->n_seqs, c->table_stride, c->n_layers};
    return MJ_OK;
}

mj_status check_batch(mj_ctx* ctx, const mj_batch* b, int n_seqs, const char* what, PgRows& r) {
    if (!b || !b->row_start) return mj_fail(ctx, MJ_INVALID_ARG, "%s: null batch", what);
    if (b->n_seqs < 1 || b->n_seqs > PG_MAX_SEQS || (n_seqs && b->n_seqs != n_seqs) || b->rows < 0 ||
        b->rows > kMaxRowsInAll || b->max_rows < 1 || b->max_rows > MJ_MAX_ROWS)
        return mj_fail(ctx, MJ_INVALID_ARG,
                       "%s: a batch of n_seqs=%d (the pages': %d) rows=%d max_rows=%d", what, b->n_seqs,
                       n_seqs, b->rows, b->max_rows);
    if (((uintptr_t)b->row_start & 3) || ((uintptr_t)b->anc & 7))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: unaligned batch", what);
    r = PgRows{b->row_start, b->anc, b->rows, b->max_rows, b->n_seqs};
    return MJ_OK;
}

// Rows of fp16 values: their stride in halves (0: packed).
mj_status check_rows(mj_ctx* ctx, const void* p, int64_t& ld, int64_t width, const char* what) {
    if (ld == 0) ld = width;
    if (!p || ld < width || ld % 8 != 0 || ld > (1ll << 31) || !aligned16({p}))
        return mj_fail(ctx, MJ_INVALID_ARG,
                       "%s: rows of %lld halves in a stride of %lld (a multiple of 8, 16-byte aligned)",
                       what, (long long)width, (long long)ld);
    return MJ_OK;
}

// Whether rows of wa bytes at a in steps of lda lie over rows of wb bytes at b in steps of ldb.  Columns
// of one wide buffer do not; of two different steps, any common stretch counts.
bool rows_overlap(const void* a, int64_t lda, int64_t wa, const void* b, int64_t ldb, int64_t wb, int rows) {
    if (!overlap(a, (rows - 1) * lda + wa, b, (rows - 1) * ldb + wb)) return false;
    if (lda != ldb) return true;
    int64_t d = ((intptr_t)b - (intptr_t)a) % lda;
    if (d < 0) d += lda;
    return d < wa || lda - d < wb;
}

mj_status check_heads(mj_ctx* ctx, int n_heads, int n_kv, const char* what) {
    if (n_kv < 1 || n_heads < 1 || n_heads % n_kv != 0 || n_heads / n_kv > kMaxGroup || n_heads > 65535)
        return mj_fail(ctx, MJ_UNSUPPORTED_SHAPE,
                       "%s: n_heads=%d over n_kv_heads=%d (a multiple, at most %d times)", what, n_heads,
                       n_kv, kMaxGroup);
    return MJ_OK;
}

struct Span {
    const void* p;
    size_t bytes;
};
// Whether an array lies over one of others.
bool over_any(Span a, std::initializer_list<Span> others) {
    for (const Span& o : others)
        if (o.p && o.bytes && overlap(a.p, a.bytes, o.p, o.bytes)) return true;
    return false;
}
// Whether rows of `width` bytes at p in steps of ld lie over one of others (columns beside the rows do not count).
bool rows_over_any(const void* p, int64_t ld, int64_t width, int rows, std::initializer_list<Span> others) {
    for (const Span& o : others) {
        if (!o.p || !o.bytes || !overlap(p, (rows - 1) * ld + width, o.p, o.bytes)) continue;
        const int64_t d = (intptr_t)o.p - (intptr_t)p;
        if (d < 0 || d % ld < width || d % ld + (int64_t)o.bytes > ld) return true;
    }
    return false;
}
Span k_of(const PgPool& p) { return {p.k, p.n_layers * p.layer_halves() * 2}; }
Span v_of(const PgPool& p) { return {p.v, p.n_layers * p.layer_halves() * 2}; }
Span table_of(const PgPool& p) { return {p.table, (size_t)p.n_seqs * p.stride * 4}; }
Span lens_of(const PgPool& p) { return {p.lens, (size_t)p.n_seqs * 4}; }
Span refs_of(const PgPool& p) { return {p.refs, (size_t)p.n_pages * 4}; }
Span served_of(const PgPool& p) { return {p.served, (size_t)p.n_seqs * 4}; }
Span starts_of(const PgRows& b) { return {b.start, (size_t)(b.n_seqs + 1) * 4}; }
Span masks_of(const PgRows& b) { return {b.anc, (size_t)b.rows * 8}; }

}  // namespace

extern "C" {

mj_status mj_paged_append(mj_ctx* ctx, const mj_attn_config* cfg, const mj_pages* pages, int layer,
                          const mj_batch* batch, const void* qkv, int64_t ld_qkv,
                          const void* q_norm_w, const void* k_norm_w, void* q_out) {
    const char* what = "paged_append";
    if (!ctx) return MJ_INVALID_ARG;
    PgAppendArgs a{};
    mj_status s = check_pages(ctx, pages, what, a.p);
    if (s == MJ_OK) s = check_batch(ctx, batch, a.p.n_seqs, what, a.b);
    if (s != MJ_OK) return s;
    if (!cfg) return mj_fail(ctx, MJ_INVALID_ARG, "%s: null configuration", what);
    s = check_heads(ctx, cfg->n_heads, cfg->n_kv_heads, what);
    if (s != MJ_OK) return s;
    if (cfg->head_dim != 128 || cfg->n_kv_heads != a.p.nKV ||
        (cfg->rope_dim != 0 && cfg->rope_dim != 32 && cfg->rope_dim != 64 && cfg->rope_dim != 128))
        return mj_fail(ctx, MJ_UNSUPPORTED_SHAPE, "%s: n_kv_heads=%d (the pages': %d) head_dim=%d rope_dim=%d",
                       what, cfg->n_kv_heads, a.p.nKV, cfg->head_dim, cfg->rope_dim);
    if (!std::isfinite(cfg->eps) || cfg->eps < 0 || (cfg->rope_dim && !(cfg->rope_base > 0)) || layer < 0 ||
        layer >= a.p.n_layers)
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: eps=%g rope_base=%g layer=%d", what, (double)cfg->eps,
                       (double)cfg->rope_base, layer);
    if (a.b.rows == 0) return MJ_OK;
    const int64_t width = (int64_t)(cfg->n_heads + 2 * cfg->n_kv_heads) * 128;
    s = check_rows(ctx, qkv, ld_qkv, width, what);
    if (s != MJ_OK) return s;
    if (!q_out || !aligned16({q_norm_w, k_norm_w, q_out}))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: null or unaligned pointer", what);
    if (rows_overlap(qkv, ld_qkv * 2, width * 2, q_out, cfg->n_heads * 256, cfg->n_heads * 256, a.b.rows))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: q_out over qkv", what);
    if (over_any({q_out, (size_t)a.b.rows * cfg->n_heads * 256},
                 {k_of(a.p), v_of(a.p), table_of(a.p), lens_of(a.p), refs_of(a.p), served_of(a.p), starts_of(a.b),
                  masks_of(a.b), {q_norm_w, 256}, {k_norm_w, 256}}))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: q_out over another array", what);
    a.qkv = (const uint16_t*)qkv;
    a.ld = ld_qkv;
    a.qw = (const uint16_t*)q_norm_w;
    a.kw = (const uint16_t*)k_norm_w;
    a.q_out = (uint16_t*)q_out;
    a.layer = layer;
    a.nQ = cfg->n_heads;
    a.half = cfg->rope_dim / 2;
    a.eps = cfg->eps;
    a.abort = ctx->abort_dev;
    const long double step = a.half ? std::pow((long double)cfg->rope_base, -1.0L / a.half) : 1.0L;
    long double turn = 0.5L / 3.14159265358979323846264338327950288L;
    for (int i = 0; i < a.half; ++i, turn *= step) a.turns[i] = (double)turn;
    OnDevice on(ctx->device);
    return mj_hip(ctx, launch_paged_append(a, ctx->stream), what);
}

size_t mj_paged_workspace(int n_heads, int n_kv_heads, int max_rows) {
    if (n_kv_heads < 1 || n_kv_heads > 1024 || n_heads < 1 || n_heads > 65535 || n_heads % n_kv_heads != 0 ||
        n_heads / n_kv_heads > kMaxGroup || max_rows < 1 || max_rows > MJ_MAX_ROWS)
        return 0;
    PgAttnArgs a{};
    a.G = n_heads / n_kv_heads;
    a.b.max_rows = max_rows;
    return paged_attn_plan(a, nullptr);
}

mj_status mj_paged_attn(mj_ctx* ctx, const mj_pages* pages, int layer, const mj_batch* batch,
                        int n_heads, int window, const void* q, int64_t ld_q, void* out,
                        int64_t ld_out, void* ws, size_t ws_bytes) {
    const char* what = "paged_attn";
    if (!ctx) return MJ_INVALID_ARG;
    PgAttnArgs a{};
    mj_status s = check_pages(ctx, pages, what, a.p);
    if (s == MJ_OK) s = check_batch(ctx, batch, a.p.n_seqs, what, a.b);
    if (s == MJ_OK) s = check_heads(ctx, n_heads, a.p.nKV, what);
    if (s != MJ_OK) return s;
    if (layer < 0 || layer >= a.p.n_layers || window < 0)
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: layer=%d (of %d) window=%d", what, layer, a.p.n_layers,
                       window);
    if (a.b.rows == 0) return MJ_OK;
    const int64_t width = (int64_t)n_heads * 128;
    s = check_rows(ctx, q, ld_q, width, what);
    if (s == MJ_OK) s = check_rows(ctx, out, ld_out, width, what);
    if (s != MJ_OK) return s;
    if (rows_overlap(q, ld_q * 2, width * 2, out, ld_out * 2, width * 2, a.b.rows))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: out over q", what);
    const std::initializer_list<Span> read = {k_of(a.p),    v_of(a.p),      table_of(a.p), lens_of(a.p),
                                              refs_of(a.p), served_of(a.p), starts_of(a.b), masks_of(a.b)};
    if (rows_over_any(out, ld_out * 2, width * 2, a.b.rows, read))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: out over another array", what);
    a.q = (const uint16_t*)q;
    a.ldq = ld_q;
    a.out = (uint16_t*)out;
    a.ldo = ld_out;
    a.layer = layer;
    a.G = n_heads / a.p.nKV;
    a.window = window;
    a.abort = ctx->abort_dev;
    OnDevice on(ctx->device);
    void* base = nullptr;
    const size_t need = paged_attn_plan(a, nullptr);
    s = take_ws(ctx, ws, ws_bytes, need, what, &base);
    if (s != MJ_OK) return s;
    if (ws && (over_any({ws, need}, read) || rows_over_any(q, ld_q * 2, width * 2, a.b.rows, {{ws, need}}) ||
               rows_over_any(out, ld_out * 2, width * 2, a.b.rows, {{ws, need}})))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: the workspace over another array", what);
    paged_attn_plan(a, base);
    return mj_hip(ctx, launch_paged_attn(a, ctx->stream), what);
}

mj_status mj_pages_reserve(mj_ctx* ctx, const mj_pages* pages, const mj_batch* batch, int32_t* out) {
    const char* what = "pages_reserve";
    if (!ctx) return MJ_INVALID_ARG;
    PgPool p;
    PgRows b;
    mj_status s = check_pages(ctx, pages, what, p);
    if (s == MJ_OK) s = check_batch(ctx, batch, p.n_seqs, what, b);
    if (s != MJ_OK) return s;
    if (!out || !aligned16({out}) ||
        over_any({out, (size_t)p.n_seqs * 16},
                 {k_of(p), v_of(p), table_of(p), lens_of(p), refs_of(p), served_of(p), starts_of(b)}))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: out null, unaligned or over another array", what);
    OnDevice on(ctx->device);
    return mj_hip(ctx, launch_pages_reserve(p, b, out, ctx->abort_dev, ctx->stream), what);
}

mj_status mj_pages_fork(mj_ctx* ctx, const mj_pages* pages, const int32_t* from) {
    const char* what = "pages_fork";
    if (!ctx) return MJ_INVALID_ARG;
    PgPool p;
    mj_status s = check_pages(ctx, pages, what, p);
    if (s != MJ_OK) return s;
    if (!from || ((uintptr_t)from & 3) ||
        over_any({from, (size_t)p.n_seqs * 4}, {table_of(p), lens_of(p), refs_of(p), served_of(p)}))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: from null, unaligned or over another array", what);
    OnDevice on(ctx->device);
    return mj_hip(ctx, launch_pages_fork(p, from, ctx->abort_dev, ctx->stream), what);
}

mj_status mj_pages_truncate(mj_ctx* ctx, const mj_pages* pages, const int32_t* len) {
    const char* what = "pages_truncate";
    if (!ctx) return MJ_INVALID_ARG;
    PgPool p;
    mj_status s = check_pages(ctx, pages, what, p);
    if (s != MJ_OK) return s;
    // (each sequence's own number is read before its length is written: len may be the lengths)
    if (!len || ((uintptr_t)len & 3) || over_any({len, (size_t)p.n_seqs * 4}, {table_of(p), refs_of(p), served_of(p)}) ||
        (len != p.lens && over_any({len, (size_t)p.n_seqs * 4}, {lens_of(p)})))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: len null, unaligned or over another array", what);
    OnDevice on(ctx->device);
    return mj_hip(ctx, launch_pages_truncate(p, len, ctx->abort_dev, ctx->stream), what);
}

mj_status mj_pages_commit(mj_ctx* ctx, const mj_pages* pages, const mj_batch* batch,
                          const int32_t* accepted, const int32_t* path, int32_t* lens_out) {
    const char* what = "pages_commit";
    if (!ctx) return MJ_INVALID_ARG;
    PgPool p;
    PgRows b;
    mj_status s = check_pages(ctx, pages, what, p);
    if (s == MJ_OK) s = check_batch(ctx, batch, p.n_seqs, what, b);
    if (s != MJ_OK) return s;
    const Span acc{accepted, (size_t)p.n_seqs * 4}, way{path, (size_t)b.rows * 4};
    const Span to{lens_out, (size_t)p.n_seqs * 4};
    if (!accepted || !lens_out || ((uintptr_t)accepted & 3) || ((uintptr_t)path & 3) ||
        ((uintptr_t)lens_out & 3) || over_any(to, {k_of(p), v_of(p), table_of(p), refs_of(p), served_of(p), starts_of(b), acc, way}) ||
        (lens_out != p.lens && over_any(to, {lens_of(p)})))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: null or unaligned pointer, or lens_out over another array",
                       what);
    OnDevice on(ctx->device);
    return mj_hip(ctx, launch_pages_commit(p, b, accepted, path, lens_out, ctx->abort_dev, ctx->stream),
                  what);
}

size_t mj_accept_workspace(int n_seqs, int rows, int V) {
    if (n_seqs < 1 || n_seqs > PG_MAX_SEQS || rows < 0 || rows > kMaxRowsInAll || V < 1 || V > kMaxVocab)
        return 0;
    AcceptArgs a{};
    a.b.n_seqs = n_seqs;
    a.b.rows = rows;
    a.V = V;
    return accept_rows_layout(a, nullptr);
}

mj_status mj_accept_rows(mj_ctx* ctx, const mj_batch* batch, const float* logits, int64_t ld_logits,
                         int V, const int32_t* tokens, const float* q, int64_t ld_q,
                         const float* temperature, const float* u_accept, const float* u_sample,
                         int32_t* accepted, int32_t* path, int32_t* token, void* ws,
                         size_t ws_bytes) {
    const char* what = "accept_rows";
    if (!ctx) return MJ_INVALID_ARG;
    AcceptArgs a{};
    mj_status s = check_batch(ctx, batch, 0, what, a.b);
    if (s != MJ_OK) return s;
    if (ld_logits == 0) ld_logits = V;
    if (ld_q == 0) ld_q = V;
    if (V < 1 || V > kMaxVocab || ld_logits < V || ld_logits > (1ll << 31) ||
        (q && (ld_q < V || ld_q > (1ll << 31))))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: V=%d in rows of %lld and %lld", what, V,
                       (long long)ld_logits, (long long)(q ? ld_q : 0));
    if (q && a.b.anc)
        return mj_fail(ctx, MJ_UNSUPPORTED_SHAPE, "%s: distributions of the drafts are of chains", what);
    const size_t R = (size_t)a.b.rows, n = (size_t)a.b.n_seqs;
    uintptr_t bits = 0;
    for (const void* p : {(const void*)logits, (const void*)tokens, (const void*)q, (const void*)temperature,
                          (const void*)u_accept, (const void*)u_sample, (const void*)accepted,
                          (const void*)path, (const void*)token})
        bits |= (uintptr_t)p;
    if (!temperature || !u_sample || !accepted || !token || (bits & 3) ||
        (R && (!logits || !tokens || !u_accept || !path)))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: null or unaligned pointer", what);
    const Span out[3] = {{accepted, n * 4}, {path, R * 4}, {token, n * 4}};
    const std::initializer_list<Span> read = {starts_of(a.b), masks_of(a.b), {tokens, R * 4}, {temperature, n * 4},
                                              {u_accept, R * 4}, {u_sample, n * 4},
                                              {logits, R ? ((R - 1) * ld_logits + V) * 4 : 0},
                                              {q, R ? ((R - 1) * ld_q + V) * 4 : 0}};
    for (int i = 0; i < 3; ++i)
        if (out[i].bytes && (over_any(out[i], read) || over_any(out[i], {out[(i + 1) % 3]})))
            return mj_fail(ctx, MJ_INVALID_ARG, "%s: an output over another array", what);
    a.logits = logits;
    a.ld = ld_logits;
    a.V = V;
    a.tokens = tokens;
    a.q = q;
    a.ldq = ld_q;
    a.temperature = temperature;
    a.u_accept = u_accept;
    a.u_sample = u_sample;
    a.accepted = accepted;
    a.path = path;
    a.token = token;
    a.abort = ctx->abort_dev;
    OnDevice on(ctx->device);
    void* base = nullptr;
    const size_t need = accept_rows_layout(a, nullptr);
    s = take_ws(ctx, ws, ws_bytes, need, what, &base);
    if (s != MJ_OK) return s;
    if (ws && (over_any({ws, need}, read) || over_any({ws, need}, {out[0], out[1], out[2]})))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: the workspace over another array", what);
    accept_rows_layout(a, base);
    return mj_hip(ctx, launch_accept_rows(a, ctx->stream), what);
}

}  // extern "C"
