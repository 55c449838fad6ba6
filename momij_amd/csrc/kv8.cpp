// kv8.cpp -- C entries of the 8-bit KV cache: argument checks, workspaces, launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "mj_abi_internal.h"
#include "mj_kv8.h"

namespace {

// The context's device for the time of one call.
struct OnDevice {
    int prev = -1;
    explicit OnDevice(int dev) {
        if (hipGetDevice(&prev) != hipSuccess) prev = -1;
        if (prev != dev) (void)hipSetDevice(dev);
        else prev = -1;
    }
    ~OnDevice() {
        if (prev >= 0) (void)hipSetDevice(prev);
    }
};

bool aligned16(std::initializer_list<const void*> ps) {
    uintptr_t bits = 0;
    for (const void* p : ps) bits |= (uintptr_t)p;
    return (bits & 15) == 0;
}

bool overlap(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y ? y - x < a_bytes : x - y < b_bytes;
}

constexpr int kMaxGroup = 64;              // query heads a KV head
constexpr int kMaxBlocks = 1 << 20;        // blocks a head lists
constexpr int64_t kMaxRing = 1ll << 30;    // slots (slots are counted in 32 bits)
constexpr int64_t kMaxPosition = 1ll << 52;

mj_status check_pool(mj_ctx* ctx, const mj_kv8* c, const char* what, Kv8Pool& p) {
    if (!c || !c->k_codes || !c->v_codes || !c->k_scale || !c->v_scale || !c->k_bounds || !c->table)
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: null pointer in the cache", what);
    if (c->n_kv_heads < 1 || c->n_kv_heads > 1024 || c->n_pages < 1 || c->table_stride < 1 ||
        c->table_stride > kMaxBlocks)
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: n_kv_heads=%d n_pages=%d table_stride=%d", what,
                       c->n_kv_heads, c->n_pages, c->table_stride);
    if (!aligned16({c->k_codes, c->v_codes, c->k_scale, c->v_scale, c->k_bounds, c->table}))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: the cache's arrays need 16-byte alignment", what);
    p = Kv8Pool{(uint8_t*)c->k_codes, (uint8_t*)c->v_codes, c->k_scale, c->v_scale, c->k_bounds,
                c->table, c->n_kv_heads, c->n_pages, c->table_stride};
    return MJ_OK;
}

mj_status check_ring(mj_ctx* ctx, const mj_kv_ring* r, const char* what, Kv8Ring& out) {
    if (!r || !r->k || !r->v) return mj_fail(ctx, MJ_INVALID_ARG, "%s: null ring", what);
    if (r->capacity < 1 || r->capacity >= kMaxRing)
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: ring capacity %lld", what, (long long)r->capacity);
    if (!aligned16({r->k, r->v}))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: the ring needs 16-byte alignment", what);
    out = Kv8Ring{(uint16_t*)r->k, (uint16_t*)r->v, r->capacity};
    return MJ_OK;
}

mj_status check_span(mj_ctx* ctx, const Kv8Pool& p, const Kv8Ring& r, int64_t pos, int count, int at,
                     const char* what) {
    if (pos < 0 || pos > kMaxPosition || count < 0 || at < 0 || (int64_t)at + count > p.stride)
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: pos=%lld count=%d at=%d (table_stride %d)", what,
                       (long long)pos, count, at, p.stride);
    if ((int64_t)count * KV8_B > r.C)
        return mj_fail(ctx, MJ_CAPACITY, "%s: %d blocks in a ring of %lld rows", what, count,
                       (long long)r.C);
    return MJ_OK;
}

// Query rows: heads, rows and their stride in halves (0: packed).
mj_status check_rows(mj_ctx* ctx, int n_heads, int n_kv, int M, const void* q, int64_t& ld,
                     int64_t width, const char* what) {
    if (!q || M < 1 || M > MJ_MAX_ROWS)
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: null pointer or M=%d outside 1..%d", what, M,
                       MJ_MAX_ROWS);
    if (n_heads < 1 || n_heads % n_kv != 0 || n_heads / n_kv > kMaxGroup)
        return mj_fail(ctx, MJ_UNSUPPORTED_SHAPE,
                       "%s: n_heads=%d over n_kv_heads=%d (a multiple, at most %d times)", what,
                       n_heads, n_kv, kMaxGroup);
    if (ld == 0) ld = width;
    if (ld < width || ld % 8 != 0 || ld > (1ll << 31) || !aligned16({q}))
        return mj_fail(ctx, MJ_INVALID_ARG,
                       "%s: rows of %lld halves in a stride of %lld (a multiple of 8, 16-byte aligned)",
                       what, (long long)width, (long long)ld);
    return MJ_OK;
}

// Device scratch of one call: the caller's, or the context's (not while its stream is captured).
mj_status take_ws(mj_ctx* ctx, void* ws, size_t ws_bytes, size_t need, const char* what, void** out) {
    if (!ws) {
        mj_status s = mj_refuse_capture(ctx, what);
        if (s == MJ_OK) s = mj_scratch_reserve(ctx, need);
        *out = ctx->scratch;
        return s;
    }
    if (!aligned16({ws}) || ws_bytes < need)
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: workspace of %zu bytes (needs %zu, 16-byte aligned)",
                       what, ws_bytes, need);
    *out = ws;
    return MJ_OK;
}

size_t select_bytes(int M, int n_kv, int n_blocks) {
    return (size_t)M * n_kv * std::max(n_blocks, 1) * 4;
}

// The sizes of an attention call into its plan's inputs.
void attn_sizes(Kv8AttnArgs& a, int n_kv, int n_heads, int M, int n_blocks, int n_sel,
                int64_t ring_rows) {
    a.p.nKV = n_kv;
    a.G = n_heads / n_kv;
    a.M = M;
    a.n = n_blocks;
    a.n_sel = n_sel;
    a.R = (int)(ring_rows - M);
}

mj_status fill_attn(mj_ctx* ctx, Kv8AttnArgs& a, const Kv8Pool& p, const Kv8Ring& r, int n_heads,
                    int M, int n_blocks, const int32_t* sel, int n_sel, int64_t start, int64_t L,
                    const int32_t* parents, const float* mass_in, float* mass_out, const char* what) {
    if (n_blocks < 0 || n_blocks > p.stride)
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: n_blocks=%d (table_stride %d)", what, n_blocks,
                       p.stride);
    if (start < 0 || start > L || L > kMaxPosition)
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: start=%lld L=%lld", what, (long long)start,
                       (long long)L);
    if (L - start + M > r.C)
        return mj_fail(ctx, MJ_CAPACITY, "%s: ring of %lld rows for %lld open ones and %d new", what,
                       (long long)r.C, (long long)(L - start), M);
    if (sel ? n_sel < 1 || n_sel > kMaxBlocks : n_sel != 0)
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: n_sel=%d", what, n_sel);
    if (sel && mass_out)
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: masses are of attention over every block", what);
    const size_t mass_bytes = (size_t)p.nKV * p.stride * 4;
    if (mass_in && mass_in != mass_out && overlap(mass_in, mass_bytes, mass_out, mass_bytes))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: mass_out over a part of mass_in", what);
    StepDesc sd{};
    mj_status s = fill_tree(ctx, &sd, parents, M);
    if (s != MJ_OK) return s;
    attn_sizes(a, p.nKV, n_heads, M, n_blocks, n_sel, L - start + M);
    a.p = p;
    a.ring = r;
    a.sel = sel;
    a.mass_in = mass_in;
    a.mass_out = mass_out;
    a.slot0 = (int)(start % r.C);
    std::copy(sd.anc, sd.anc + M, a.anc);
    a.abort = ctx->abort_dev;
    return MJ_OK;
}

mj_status fill_append(mj_ctx* ctx, Kv8AppendArgs& a, const mj_attn_config& c, const void* qkv,
                      int64_t ld, const void* qw, const void* kw, const Kv8Ring& r, int64_t L,
                      const int32_t* parents, int M, void* q_out, const char* what) {
    if (L < 0 || L > kMaxPosition)
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: L=%lld", what, (long long)L);
    if (!std::isfinite(c.eps) || c.eps < 0 || (c.rope_dim && !(c.rope_base > 0)))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: eps=%g rope_base=%g", what, (double)c.eps,
                       (double)c.rope_base);
    if (M > r.C)
        return mj_fail(ctx, MJ_CAPACITY, "%s: %d rows in a ring of %lld", what, M, (long long)r.C);
    StepDesc sd{};
    mj_status s = fill_tree(ctx, &sd, parents, M);
    if (s != MJ_OK) return s;
    a.qkv = (const uint16_t*)qkv;
    a.ld = ld;
    a.qw = (const uint16_t*)qw;
    a.kw = (const uint16_t*)kw;
    a.ring = r;
    a.q_out = (uint16_t*)q_out;
    a.L = L;
    a.slot0 = L % r.C;
    a.M = M;
    a.nQ = c.n_heads;
    a.nKV = c.n_kv_heads;
    a.half = c.rope_dim / 2;
    a.eps = c.eps;
    a.abort = ctx->abort_dev;
    // base^(-i / half) / 2 pi by products of 64 bits' mantissa (a power each takes longer than the
    // rest of the call)
    const long double step = a.half ? std::pow((long double)c.rope_base, -1.0L / a.half) : 1.0L;
    long double turn = 0.5L / 3.14159265358979323846264338327950288L;
    for (int i = 0; i < a.half; ++i, turn *= step) a.turns[i] = (double)turn;
    for (int i = 0; i < M; ++i) a.depth[i] = (uint8_t)sd.depth[i];
    return MJ_OK;
}

mj_status check_heads(mj_ctx* ctx, const mj_attn_config* c, const char* what) {
    if (!c) return mj_fail(ctx, MJ_INVALID_ARG, "%s: null configuration", what);
    if (c->head_dim != 128 || c->n_kv_heads < 1 || c->n_kv_heads > 1024 || c->n_heads < 1 ||
        c->n_heads % c->n_kv_heads != 0 || c->n_heads / c->n_kv_heads > kMaxGroup ||
        (c->rope_dim != 0 && c->rope_dim != 32 && c->rope_dim != 64 && c->rope_dim != 128))
        return mj_fail(ctx, MJ_UNSUPPORTED_SHAPE,
                       "%s: n_heads=%d n_kv_heads=%d head_dim=%d rope_dim=%d", what, c->n_heads,
                       c->n_kv_heads, c->head_dim, c->rope_dim);
    return MJ_OK;
}

mj_status check_select(mj_ctx* ctx, const Kv8Pool& p, int n_blocks, int n_sel, int n_first,
                       int n_last, const char* what) {
    if (n_blocks < 0 || n_blocks > p.stride || n_sel < 1 || n_sel > kMaxBlocks || n_first < 0 ||
        n_last < 0 || (int64_t)n_first + n_last > n_sel)
        return mj_fail(ctx, MJ_INVALID_ARG,
                       "%s: n_blocks=%d n_sel=%d n_first=%d n_last=%d (table_stride %d)", what,
                       n_blocks, n_sel, n_first, n_last, p.stride);
    return MJ_OK;
}

// A tree's parents are a host array: not while the stream is captured.
mj_status refuse_tree(mj_ctx* ctx, const int32_t* parents, const char* what) {
    return parents ? mj_refuse_capture(ctx, what) : MJ_OK;
}

}  // namespace

extern "C" {

mj_status mj_qkv_append(mj_ctx* ctx, const mj_attn_config* cfg, const void* qkv, int64_t ld_qkv,
                        const void* q_norm_w, const void* k_norm_w, const mj_kv_ring* ring,
                        int64_t L, const int32_t* parents_host, int M, void* q_out) {
    const char* what = "qkv_append";
    if (!ctx) return MJ_INVALID_ARG;
    mj_status s = check_heads(ctx, cfg, what);
    if (s != MJ_OK) return s;
    s = check_rows(ctx, cfg->n_heads, cfg->n_kv_heads, M, qkv, ld_qkv,
                   (int64_t)(cfg->n_heads + 2 * cfg->n_kv_heads) * 128, what);
    if (s != MJ_OK) return s;
    if (!q_norm_w || !k_norm_w || !q_out || !aligned16({q_norm_w, k_norm_w, q_out}))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: null or unaligned pointer", what);
    Kv8Ring r;
    s = check_ring(ctx, ring, what, r);
    if (s != MJ_OK) return s;
    Kv8AppendArgs a{};
    s = fill_append(ctx, a, *cfg, qkv, ld_qkv, q_norm_w, k_norm_w, r, L, parents_host, M, q_out, what);
    if (s != MJ_OK) return s;
    // rows are read by several blocks, each when it comes
    for (int i = 0; i < M; ++i)
        if (overlap(q_out, (size_t)M * cfg->n_heads * 256, a.qkv + i * ld_qkv,
                    (size_t)(cfg->n_heads + 2 * cfg->n_kv_heads) * 256))
            return mj_fail(ctx, MJ_INVALID_ARG, "%s: q_out over qkv", what);
    OnDevice on(ctx->device);
    s = refuse_tree(ctx, parents_host, what);
    if (s != MJ_OK) return s;
    return mj_hip(ctx, launch_qkv_append(a, ctx->stream), what);
}

mj_status mj_kv8_seal(mj_ctx* ctx, const mj_kv8* cache, const mj_kv_ring* ring, int64_t pos,
                      int count, int at) {
    const char* what = "kv8_seal";
    if (!ctx) return MJ_INVALID_ARG;
    Kv8Pool p;
    Kv8Ring r;
    mj_status s = check_pool(ctx, cache, what, p);
    if (s == MJ_OK) s = check_ring(ctx, ring, what, r);
    if (s == MJ_OK) s = check_span(ctx, p, r, pos, count, at, what);
    if (s != MJ_OK || count == 0) return s;
    OnDevice on(ctx->device);
    return mj_hip(ctx, launch_kv8_seal(p, r, pos % r.C, count, at, ctx->abort_dev, ctx->stream), what);
}

mj_status mj_kv8_unseal(mj_ctx* ctx, const mj_kv8* cache, int at, int count,
                        const mj_kv_ring* ring, int64_t pos) {
    const char* what = "kv8_unseal";
    if (!ctx) return MJ_INVALID_ARG;
    Kv8Pool p;
    Kv8Ring r;
    mj_status s = check_pool(ctx, cache, what, p);
    if (s == MJ_OK) s = check_ring(ctx, ring, what, r);
    if (s == MJ_OK) s = check_span(ctx, p, r, pos, count, at, what);
    if (s != MJ_OK || count == 0) return s;
    OnDevice on(ctx->device);
    return mj_hip(ctx, launch_kv8_unseal(p, r, pos % r.C, count, at, ctx->abort_dev, ctx->stream),
                  what);
}

mj_status mj_kv8_select(mj_ctx* ctx, const mj_kv8* cache, int n_heads, const void* q, int64_t ld_q,
                        int M, int n_blocks, int n_sel, int n_first, int n_last, int32_t* sel,
                        void* ws, size_t ws_bytes) {
    const char* what = "kv8_select";
    if (!ctx) return MJ_INVALID_ARG;
    Kv8Pool p;
    mj_status s = check_pool(ctx, cache, what, p);
    if (s == MJ_OK) s = check_rows(ctx, n_heads, p.nKV, M, q, ld_q, (int64_t)n_heads * 128, what);
    if (s == MJ_OK) s = check_select(ctx, p, n_blocks, n_sel, n_first, n_last, what);
    if (s != MJ_OK) return s;
    if (!sel) return mj_fail(ctx, MJ_INVALID_ARG, "%s: null sel", what);
    OnDevice on(ctx->device);
    void* base = nullptr;
    s = take_ws(ctx, ws, ws_bytes, select_bytes(M, p.nKV, n_blocks), what, &base);
    if (s != MJ_OK) return s;
    Kv8SelectArgs a{p, (const uint16_t*)q, ld_q, M, n_heads / p.nKV, n_blocks, n_sel,
                    std::min(n_first, n_blocks), std::min(n_last, n_blocks), (float*)base, sel,
                    ctx->abort_dev};
    return mj_hip(ctx, launch_kv8_select(a, ctx->stream), what);
}

mj_status mj_kv8_attn(mj_ctx* ctx, const mj_kv8* cache, const mj_kv_ring* ring, int n_heads,
                      const void* q, int64_t ld_q, int M, int n_blocks, const int32_t* sel,
                      int n_sel, int64_t start, int64_t L, const int32_t* parents_host, void* out,
                      int64_t ld_out, const float* mass_in, float* mass_out, void* ws,
                      size_t ws_bytes) {
    const char* what = "kv8_attn";
    if (!ctx) return MJ_INVALID_ARG;
    Kv8Pool p;
    Kv8Ring r;
    mj_status s = check_pool(ctx, cache, what, p);
    if (s == MJ_OK) s = check_ring(ctx, ring, what, r);
    if (s == MJ_OK) s = check_rows(ctx, n_heads, p.nKV, M, q, ld_q, (int64_t)n_heads * 128, what);
    if (s == MJ_OK) s = check_rows(ctx, n_heads, p.nKV, M, out, ld_out, (int64_t)n_heads * 128, what);
    if (s != MJ_OK) return s;
    if (mass_in && !mass_out)
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: mass_in without mass_out", what);
    Kv8AttnArgs a{};
    s = fill_attn(ctx, a, p, r, n_heads, M, n_blocks, sel, n_sel, start, L, parents_host,
                  mass_in, mass_out, what);
    if (s != MJ_OK) return s;
    a.q = (const uint16_t*)q;
    a.ldq = ld_q;
    a.out = (uint16_t*)out;
    a.ldo = ld_out;
    OnDevice on(ctx->device);
    s = refuse_tree(ctx, parents_host, what);
    if (s != MJ_OK) return s;
    const bool mass = mass_out && n_blocks > 0;
    void* base = nullptr;
    s = take_ws(ctx, ws, ws_bytes, kv8_attn_plan(a, mass, nullptr), what, &base);
    if (s != MJ_OK) return s;
    kv8_attn_plan(a, mass, base);
    return mj_hip(ctx, launch_kv8_attn(a, ctx->stream), what);
}

mj_status mj_kv8_evict(mj_ctx* ctx, const mj_kv8* cache, int n_blocks, int keep, int n_first,
                       int n_last, const float* mass_in, int32_t* table_out, float* mass_out) {
    const char* what = "kv8_evict";
    if (!ctx) return MJ_INVALID_ARG;
    Kv8Pool p;
    mj_status s = check_pool(ctx, cache, what, p);
    if (s != MJ_OK) return s;
    const size_t bytes = (size_t)p.nKV * p.stride * 4;
    auto over = [&](const void* a, const void* b) { return overlap(a, bytes, b, bytes); };
    if (!mass_in || !table_out || !mass_out || over(table_out, cache->table) || over(mass_out, mass_in) ||
        over(table_out, mass_in) || over(mass_out, cache->table) || over(table_out, mass_out))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: null pointer, or an output over another array", what);
    if (n_blocks < 0 || n_blocks > p.stride || keep < 0 || keep > n_blocks || n_first < 0 ||
        n_last < 0 || (int64_t)n_first + n_last > keep)
        return mj_fail(ctx, MJ_INVALID_ARG,
                       "%s: n_blocks=%d keep=%d n_first=%d n_last=%d (table_stride %d)", what,
                       n_blocks, keep, n_first, n_last, p.stride);
    OnDevice on(ctx->device);
    return mj_hip(ctx, launch_kv8_evict(p, n_blocks, keep, n_first, n_last, mass_in, table_out,
                                        mass_out, ctx->abort_dev, ctx->stream), what);
}

size_t mj_kv8_workspace(int n_heads, int n_kv_heads, int M, int n_blocks, int n_sel,
                        int64_t ring_rows, int mass) {
    if (n_kv_heads < 1 || n_kv_heads > 1024 || n_heads < 1 || n_heads % n_kv_heads != 0 ||
        n_heads / n_kv_heads > kMaxGroup || M < 1 || M > MJ_MAX_ROWS || n_blocks < 0 ||
        n_blocks > kMaxBlocks || n_sel < 0 || n_sel > kMaxBlocks || ring_rows < M ||
        ring_rows >= kMaxRing)
        return 0;
    return std::max(kv8_attn_bound(n_kv_heads, M * n_heads, n_sel > 0 ? n_sel : n_blocks, ring_rows,
                                   mass && n_sel == 0 ? n_blocks : 0),
                    select_bytes(M, n_kv_heads, n_blocks));
}

mj_status mj_attn_block_kv8(mj_ctx* ctx, const mj_attn_config* cfg, const mj_attn_weights* w,
                            const mj_kv8* cache, const mj_kv_ring* ring, void* h, int n_blocks,
                            int n_sel, int n_first, int n_last, int64_t start, int64_t L,
                            const int32_t* parents_host, int M, const float* mass_in,
                            float* mass_out) {
    const char* what = "attn_block_kv8";
    if (!ctx) return MJ_INVALID_ARG;
    Kv8Pool p;
    Kv8Ring r;
    mj_status s = check_heads(ctx, cfg, what);
    if (s == MJ_OK) s = check_pool(ctx, cache, what, p);
    if (s == MJ_OK) s = check_ring(ctx, ring, what, r);
    if (s != MJ_OK) return s;
    const mj_attn_config& c = *cfg;
    const int H = c.H, nQ = c.n_heads, nKV = c.n_kv_heads, qkvN = (nQ + 2 * nKV) * 128;
    if (!w || !h || !w->norm_w || !w->qkv_w || !w->qkv_s || !w->qkv_b || !w->q_norm_w ||
        !w->k_norm_w || !w->o_w || !w->o_s || !w->o_b || M < 1 || M > MJ_MAX_ROWS ||
        (mass_in && !mass_out) || !aligned16({h, w->norm_w, w->q_norm_w, w->k_norm_w}))
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: null or unaligned pointer, or M=%d outside 1..%d",
                       what, M, MJ_MAX_ROWS);
    if (nQ % 4 != 0 || H < 2048 || H % 2048 != 0 || H > 4096 || (c.gs != 64 && c.gs != 128) ||
        c.window != 0 || nKV != p.nKV)
        return mj_fail(ctx, MJ_UNSUPPORTED_SHAPE,
                       "%s: H=%d n_heads=%d n_kv_heads=%d (cache: %d) gs=%d window=%d", what, H, nQ,
                       nKV, p.nKV, c.gs, c.window);
    if (n_sel < 0) return mj_fail(ctx, MJ_INVALID_ARG, "%s: n_sel=%d", what, n_sel);
    if (n_sel > 0) {
        s = check_select(ctx, p, n_blocks, n_sel, n_first, n_last, what);
        if (s != MJ_OK) return s;
    }
    // lists that would name every block are left out
    const bool pick = n_sel > 0 && n_sel < n_blocks;
    if (n_sel > 0 && mass_out)
        return mj_fail(ctx, MJ_INVALID_ARG, "%s: masses are of attention over every block", what);
    Kv8AttnArgs a{};
    Kv8AppendArgs ap{};
    s = fill_attn(ctx, a, p, r, nQ, M, n_blocks, pick ? p.table : nullptr, pick ? n_sel : 0, start, L,
                  parents_host, mass_in, mass_out, what);
    if (s == MJ_OK)
        s = fill_append(ctx, ap, c, nullptr, qkvN, w->q_norm_w, w->k_norm_w, r, L, parents_host, M,
                        nullptr, what);
    if (s != MJ_OK) return s;
    OnDevice on(ctx->device);
    s = mj_hip(ctx, set_kernel_attributes(), "kernel attributes");
    if (s == MJ_OK) s = mj_refuse_capture(ctx, what);
    if (s != MJ_OK) return s;
    const bool mass = mass_out && n_blocks > 0;
    const size_t attn_ws = kv8_attn_plan(a, mass, nullptr);
    void* b[9];
    auto layout = [&](Arena& ar) {
        b[0] = ar.take((size_t)M * H * 2);            // normed rows, qx
        b[1] = ar.take((size_t)M * (H / 64) * 8);
        b[2] = ar.take((size_t)M * qkvN * 2);         // raw projection
        b[3] = ar.take((size_t)M * nQ * 128 * 2);     // finished queries
        b[4] = ar.take((size_t)M * nQ * 128 * 2);     // attention output, qx
        b[5] = ar.take((size_t)M * nQ * 2 * 8);
        b[6] = ar.take(pick ? (size_t)M * nKV * n_sel * 4 : 4);
        b[7] = ar.take(pick ? select_bytes(M, nKV, n_blocks) : 4);
        b[8] = ar.take(attn_ws);
    };
    Arena count;
    layout(count);
    s = mj_scratch_reserve(ctx, count.off);
    if (s != MJ_OK) return s;
    Arena real{ctx->scratch, 0};
    layout(real);
    hipStream_t st = ctx->stream;
    const int* ab = ctx->abort_dev;
    s = mj_hip(ctx, launch_rmsnorm_qx((const uint16_t*)h, (const uint16_t*)w->norm_w, c.eps, nullptr,
                                      (uint16_t*)b[0], (float2*)b[1], M, H, ab, st), "attn norm");
    if (s != MJ_OK) return s;
    GatherArgs q{};
    q.xperm = (uint16_t*)b[0];
    q.xsum = (float2*)b[1];
    q.w = w->qkv_w;
    q.s = (const uint16_t*)w->qkv_s;
    q.b = (const uint16_t*)w->qkv_b;
    q.dense_rows = M;
    q.y = (uint16_t*)b[2];
    q.K = H;
    q.N = qkvN;
    q.gs = c.gs;
    q.x_div = 1;
    q.abort = ab;
    s = mj_hip(ctx, launch_gather(q, EPI_STORE, M, 1, st), "qkv");
    if (s != MJ_OK) return s;
    ap.qkv = (const uint16_t*)b[2];
    ap.q_out = (uint16_t*)b[3];
    s = mj_hip(ctx, launch_qkv_append(ap, st), "append");
    if (s != MJ_OK) return s;
    if (pick) {
        Kv8SelectArgs sa{p, (const uint16_t*)b[3], (int64_t)nQ * 128, M, nQ / nKV, n_blocks, n_sel,
                         std::min(n_first, n_blocks), std::min(n_last, n_blocks), (float*)b[7],
                         (int32_t*)b[6], ab};
        s = mj_hip(ctx, launch_kv8_select(sa, st), "select");
        if (s != MJ_OK) return s;
        a.sel = (const int32_t*)b[6];
    }
    kv8_attn_plan(a, mass, b[8]);
    a.q = (const uint16_t*)b[3];
    a.ldq = (int64_t)nQ * 128;
    a.out_perm = (uint16_t*)b[4];
    a.out_sum = (float2*)b[5];
    s = mj_hip(ctx, launch_kv8_attn(a, st), "attention");
    if (s != MJ_OK) return s;
    GatherArgs o{};
    o.xperm = (uint16_t*)b[4];
    o.xsum = (float2*)b[5];
    o.w = w->o_w;
    o.s = (const uint16_t*)w->o_s;
    o.b = (const uint16_t*)w->o_b;
    o.dense_rows = M;
    o.y = (uint16_t*)h;
    o.K = nQ * 128;
    o.N = H;
    o.gs = c.gs;
    o.x_div = 1;
    o.abort = ab;
    return mj_hip(ctx, launch_gather(o, EPI_ADD, M, 1, st), "o proj");
}

}  // extern "C"
