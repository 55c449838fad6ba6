// paged_attn.hip -- attention of a batch's rows over the fp16 pages of their sequences.
//
// softmax(q k^T / sqrt(128)) v in one pass over the keys with a running reference and sum.  A unit is
// 32 keys of one sequence, KV head and column group (at most `cols` query vectors: a row's heads of the group,
// row by row); the units of the batch are numbered in that order, so a block takes a run of consecutive
// ones and its work does not depend on how long which sequence is.  A run is cut where a sequence, head or
// column group ends; a segment that is all of its group's keys is finished by its block, others leave a
// partial result, and k_paged_join puts these together.  Scores are kept in log2 units.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "mj_abi_internal.h"
#include "mj_device.h"
#include "mj_paged.h"

#define HD 128
#define SC2 (1.44269504088896341f * 0.08838834764831845f)  // log2 e / sqrt(128)

// What a sequence's rows attend to, in units.
struct SeqUnits {
    int m, r0, L;   // rows, the first of them, committed tokens
    int lo, nu;     // first unit, units
    int ncg;        // column groups
};
__device__ __forceinline__ SeqUnits seq_units(const PgAttnArgs& a, int m, int r0, int L) {
    SeqUnits u;
    u.m = m;
    u.r0 = r0;
    u.L = L;
    const int end = min(u.L + u.m, a.p.room());
    u.lo = (a.window > 0 ? max(0, u.L - a.window + 1) : 0) / PG_UNIT;
    u.nu = u.m > 0 ? max(0, (end + PG_UNIT - 1) / PG_UNIT - u.lo) : 0;
    u.ncg = (u.m * a.G + a.cols - 1) / a.cols;
    return u;
}

// A tile of 16 query vectors, outputs turned: lane (ln, lq) holds vector ln's reference, its share of the
// sum, and dims 16 dt + 4 lq + r of its output.
typedef float f2v __attribute__((ext_vector_type(2)));

struct PgTile {
    float m, l;
    f4 o[8];
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) o[dt] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    }
};

// The reference follows the maximum where that is more than 2^SLACK above it, and weights are lifted by
// 2^LIFT before they are rounded to fp16 for the product with V (SLACK + LIFT = 15: below fp16's
// greatest): a weight is off by half a step, 2^-11 of itself, or by at most 2^-34 of the greatest one.
// The factor is the same in outputs and sums, and leaves with the division; sums take the weights before
// the rounding.
#define SLACK 6.0f
#define LIFT 9.0f
// Scores past FAR, whose steps in fp32 are an eighth and more: a weight's one fma differs from the rounded
// score by more than the slack allows, so the reference is taken off the rounded score.
#define FAR 1048576.0f

// x *= f in place.  (Behind a branch the compiler keeps the accumulators in two places and copies all of
// them at every step.)  The values are results of matrix instructions: scale_ready() first, which waits for these
// to be there, and scaled() before the next ones read them.
__device__ __forceinline__ void scale_ready() { asm volatile("s_nop 15\n\ts_nop 15\n\ts_nop 15" ::: "memory"); }
__device__ __forceinline__ void scale(f4& x, float f) {
    float a = x[0], b = x[1], c = x[2], d = x[3];
    asm volatile("v_mul_f32 %0, %4, %0\n\tv_mul_f32 %1, %4, %1\n\tv_mul_f32 %2, %4, %2\n\tv_mul_f32 %3, %4, %3"
                 : "+v"(a), "+v"(b), "+v"(c), "+v"(d)
                 : "v"(f));
    x = (f4){a, b, c, d};
}
__device__ __forceinline__ void scaled() { asm volatile("s_nop 7" ::: "memory"); }

// Softmax of U units' scores of T tiles against the running states, in two parts.  S[y][2 u + t]: tile y's
// vector ln against tokens 8 lq + 4 t + r of unit u, without the scale; masked ones -inf.
// The references moved, for all tiles in one branch; c: what makes exp2(S SC2 - c) the weights.  True: some
// score is far.
template <int T, int U>
__device__ __forceinline__ bool move_refs(PgTile* tl, const f4 (*S)[2 * U], float* c) {
    float s[T];
    bool rare = false, far = false;
#pragma unroll
    for (int y = 0; y < T; ++y) {
        float x = fmaxf(S[y][0][0], S[y][0][1]);
#pragma unroll
        for (int i = 1; i < 4 * U; ++i)
            x = fmaxf(fmaxf(x, S[y][i >> 1][2 * (i & 1)]), S[y][i >> 1][2 * (i & 1) + 1]);
        s[y] = product(x4_max(x), SC2);
        rare |= s[y] > tl[y].m + SLACK;
    }
    if (__any(rare)) {
        scale_ready();
#pragma unroll
        for (int y = 0; y < T; ++y) {
            const float mn = fmaxf(tl[y].m, s[y]);
            const float alpha = tl[y].m == mn ? 1.0f : __builtin_amdgcn_exp2f(tl[y].m - mn);  // (both may be -inf)
            tl[y].m = mn;
            tl[y].l *= alpha;
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) scale(tl[y].o[dt], alpha);
        }
        scaled();
    }
#pragma unroll
    for (int y = 0; y < T; ++y) {
        // no key seen: any finite reference (a masked score still gives 0, a NaN stays one)
        c[y] = (tl[y].m == -INFINITY ? 0.0f : tl[y].m) - LIFT;
        far |= fabsf(c[y]) > FAR;
    }
    return __any(far);
}
// p[u]: unit u's weights as the B operand of the product with V.
template <int U, bool FARS>
__device__ __forceinline__ void unit_weights(PgTile& T, const f4* S, float c, u4v* p) {
    float sum = 0.0f;
    const float ref = T.m == -INFINITY ? 0.0f : T.m;
    auto weight = [&](float x) {
        if (!FARS) return __builtin_amdgcn_exp2f(fmaf(x, SC2, -c));
        // (the lift last: far from 0 it would be lost in the reference)
        return __builtin_amdgcn_exp2f(product(x, SC2) - ref + LIFT);
    };
#pragma unroll
    for (int i = 0; i < 4 * U; ++i) {
        const f2v w = {weight(S[i >> 1][2 * (i & 1)]), weight(S[i >> 1][2 * (i & 1) + 1])};
        sum += w.x;
        sum += w.y;
        p[i >> 2][i & 3] = __builtin_bit_cast(uint32_t, __builtin_convertvector(w, h2v));
    }
    T.l += sum;
}
template <int T, int U>
__device__ __forceinline__ void softmax(PgTile* tl, const f4 (*S)[2 * U], u4v (*p)[U]) {
    float c[T];
    if (move_refs<T, U>(tl, S, c)) {
#pragma unroll
        for (int y = 0; y < T; ++y) unit_weights<U, true>(tl[y], S[y], c[y], p[y]);
    } else {
#pragma unroll
        for (int y = 0; y < T; ++y) unit_weights<U, false>(tl[y], S[y], c[y], p[y]);
    }
}

// The query vectors of a tile.
struct PgCol {
    bool on;        // there is such a vector
    uint64_t anc;   // rows of the sequence that its row sees
    int first;      // the first committed token that it sees
    __device__ __forceinline__ uint32_t mask(int pos, int L) const {  // of tokens pos .. pos + 31
        uint32_t ok = 0;
        if (L > pos) ok = L - pos >= 32 ? ~0u : (1u << (L - pos)) - 1u;
        if (first > pos) ok = first - pos >= 32 ? 0u : ok & (~0u << (first - pos));
        const int d = pos - L;  // the own row of the unit's first token
        const uint32_t own = d >= 64 ? 0u : d >= 0 ? (uint32_t)(anc >> d) : d > -32 ? (uint32_t)(anc << -d) : 0u;
        return on ? ok | own : 0u;
    }
};

// Bits 0 and 16: of two halves, those that are infinities or NaN (an exponent of all ones carries into the
// sign's place).  In whole numbers: as comparisons they would take a scalar mask each.
__device__ __forceinline__ uint32_t bad_halves(uint32_t y) {
    return ((y & 0x7C007C00u) + 0x04000400u) >> 15 & 0x00010001u;
}

// Infinities and NaN of V in a unit that not every row sees whole (0 times an infinity is a NaN): they are
// left out of the product and added here to the outputs of the vectors that attend to them, whatever
// their weights (which are above 0, if not in fp32).  ok: the unit's tokens that vector ln sees.
__device__ __forceinline__ void add_bad(PgTile& T, const uint16_t* vu, uint32_t bad, uint32_t ok) {
    const int lq = (threadIdx.x & 63) >> 4;
#pragma unroll 1
    for (; bad; bad &= bad - 1) {
        const int t = __builtin_ctz(bad);
        const uint32_t sees = 0u - ((ok >> t) & 1u);
        const uint16_t* row = vu + pg_v_at(t, 4 * lq);
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t v = row[512 * dt + 8 * r];
                T.o[dt][r] += h2f((uint16_t)(v & sees & (0u - bad_halves(v))));
            }
            __builtin_amdgcn_sched_barrier(0);  // (32 requests at once take 40 registers from the main loop)
        }
    }
}

// a / b of numbers from 0 up.  (A division of 64 bits takes half a microsecond.)
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    return (a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// The batch as a block needs it: units before each sequence, and its rows and length as they were read.
struct PgPlan {
    int64_t off[PG_MAX_SEQS + 1], wsum[8];
    int rows[PG_MAX_SEQS], len[PG_MAX_SEQS];  // first row, and count << 16
    int abort;
};
// The run of this block.  Every segment counts `extra` units more than it has, at its beginning: what it
// costs a block to begin one, so that blocks with several have less keys to read.
struct PgRun {
    int64_t b0, b1, per;
    int s;  // the sequence that the run begins in
};
// One round of requests and a scan for every NT sequences; a.off gets the units for the join (also of a call
// that is aborted: the word may be cleared before the join reads it).  False: the call was aborted.
template <int NT>
__device__ __forceinline__ bool plan_run(const PgAttnArgs& a, PgPlan& P, PgRun& run) {
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, n = a.b.n_seqs;
    const int ab = abort_word(a.abort);
    int64_t before = 0;
    for (int c = 0; c < n; c += NT) {
        int64_t u = 0;
        if (c + t < n) {
            int r0;
            const int m = pg_rows(a.b, c + t, r0), L = pg_len(a.p, c + t);
            const SeqUnits q = seq_units(a, m, r0, L);
            u = q.nu > 0 ? (int64_t)(q.nu + a.extra) * q.ncg * a.p.nKV : 0;
            P.rows[c + t] = r0 | m << 16;
            P.len[c + t] = L;
        }
        int64_t inc = u;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t x = __shfl_up(inc, o, MJ_WAVE);
            inc += lane >= o ? x : 0;
        }
        if (c) __syncthreads();
        if (lane == 63) P.wsum[w] = inc;
        if (t == 0 && c == 0) P.abort = ab;
        __syncthreads();
        int64_t at = before, all = before;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) {
            at += i < w ? P.wsum[i] : 0;
            all += P.wsum[i];
        }
        if (c + t <= n) P.off[c + t] = at + inc - u;
        if (c + t + 1 == n) P.off[n] = at + inc;
        before = all;
    }
    __syncthreads();
    run.per = max(quotient(before + a.blocks - 1, a.blocks), (int64_t)a.least);
    if (blockIdx.x == 0)
        for (int i = t; i <= n + 1; i += NT) a.off[i] = i <= n ? P.off[i] : run.per;
    if (P.abort) return false;
    run.b0 = blockIdx.x * run.per;
    run.b1 = min(before, run.b0 + run.per);
    run.s = 0;
    if (run.b0 < run.b1) {  // the last sequence that begins at or before the run
        int hi = n;
        while (hi - run.s > 1) {
            const int mid = (run.s + hi) >> 1;
            if (P.off[mid] <= run.b0) run.s = mid;
            else hi = mid;
        }
    }
    return true;
}

// A segment: units lo + i0 .. lo + i1 - 1 of a sequence, head and column group.
struct PgSeg {
    SeqUnits su;
    int s, g, i0, i1, v0, vend;  // query vectors v0 .. vend - 1 of the sequence's rows and the group's heads
    int clean0, clean1;          // units that every row sees whole
    bool whole;                  // all of the group's units
    int64_t slot;                // where a partial result goes
};
// The segment at x, which moves past it; i1 <= i0: only its beginning lies in the run.
__device__ __forceinline__ PgSeg next_seg(const PgAttnArgs& a, const PgPlan& P, PgRun& run, int64_t& x) {
    while (P.off[run.s + 1] <= x) ++run.s;
    PgSeg S;
    S.s = __builtin_amdgcn_readfirstlane(run.s);
    const int rw = __builtin_amdgcn_readfirstlane(P.rows[S.s]);
    S.su = seq_units(a, rw >> 16, rw & 0xFFFF, __builtin_amdgcn_readfirstlane(P.len[S.s]));
    const int64_t rel = x - P.off[S.s];
    const int len = S.su.nu + a.extra;
    int gc, at;
    if (rel >> 31) {
        gc = (int)(rel / len);
        at = (int)(rel - (int64_t)gc * len);
    } else {
        gc = (int)((uint32_t)rel / (uint32_t)len);
        at = (int)rel - gc * len;
    }
    gc = __builtin_amdgcn_readfirstlane(gc);
    at = __builtin_amdgcn_readfirstlane(at);
    const int take = (int)min((int64_t)(len - at), run.b1 - x);
    S.slot = (int64_t)blockIdx.x * 2 + (x == run.b0 ? 0 : 1);
    x += take;
    S.i0 = max(at - a.extra, 0);
    S.i1 = __builtin_amdgcn_readfirstlane(at - a.extra + take);
    S.g = gc / S.su.ncg;
    S.v0 = (gc - S.g * S.su.ncg) * a.cols;
    S.vend = min(S.su.m * a.G, S.v0 + a.cols);
    S.clean0 = a.window > 0 ? (max(0, S.su.L + MJ_ROWS - a.window + 1) + PG_UNIT - 1) / PG_UNIT : 0;
    S.clean1 = S.su.L / PG_UNIT;
    S.whole = S.i0 == 0 && S.i1 == S.su.nu;
    return S;
}
// The page of the segment's unit i, or -1.
__device__ __forceinline__ int seg_page(const PgAttnArgs& a, const PgSeg& S, int i) {
    return pg_page(a.p, S.s, ((S.su.lo + i) * PG_UNIT) >> a.p.shift);
}
// Halves from a layer's first to the segment's unit i in page pg.
__device__ __forceinline__ size_t seg_at(const PgAttnArgs& a, const PgSeg& S, int i, int pg) {
    const int in = ((S.su.lo + i) * PG_UNIT) & (a.p.page - 1);
    return (((size_t)pg * a.p.nKV + S.g) << (a.p.shift + 7)) + (size_t)(in >> 5) * PG_UNIT_HALVES;
}

// Query vector v (lanes without one take the group's first, unused).
__device__ __forceinline__ void load_vector(const PgAttnArgs& a, const PgSeg& S, int v, u4v q[4]) {
    const int lq = (threadIdx.x & 63) >> 4;
    const bool on = v < S.vend;
    const int r = on ? v / a.G : 0, h = S.g * a.G + (on ? v - r * a.G : 0);
    const uint16_t* qp = a.q + (S.su.r0 + r) * a.ldq + h * HD + 8 * lq;
#pragma unroll
    for (int k = 0; k < 4; ++k) q[k] = *(const u4v*)(qp + 32 * k);
}
// What its row sees.
__device__ __forceinline__ PgCol load_col(const PgAttnArgs& a, const PgSeg& S, int v) {
    PgCol col;
    col.on = v < S.vend;
    const int r = col.on ? v / a.G : 0;
    col.anc = pg_anc(a.b, S.su.r0 + r, r);
    const int depth = pg_depth(col.anc, r);
    if (S.su.m < 64) col.anc &= (1ull << S.su.m) - 1;  // (a row that there is not is nobody's ancestor)
    col.first = a.window > 0 ? max(0, S.su.L + depth - a.window + 1) : 0;
    return col;
}

// Scores of tokens that vector ln does not see taken out (ok: those that it sees).
__device__ __forceinline__ void mask_scores(f4 S[2], uint32_t ok) {
    const uint32_t mine = ok >> (8 * ((threadIdx.x & 63) >> 4));
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[t][r] = (mine >> (4 * t + r)) & 1 ? S[t][r] : -INFINITY;
}
// Infinities and NaN of a unit's V operands taken as 0; which tokens hold any, the same in every lane.
// Lane (ln, lq) has tokens 8 lq + j of dims 16 k + ln.
__device__ __forceinline__ uint32_t clear_bad(u4v v[8]) {
    uint32_t my = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t any = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t b = bad_halves(v[k][j]);
            any |= b;
            v[k][j] &= ~(b * 0xFFFFu);
        }
        my |= (any & 1u) << (2 * j) | (any >> 16) << (2 * j + 1);
    }
    if (!__any(my != 0)) return 0;
    my <<= 8 * ((threadIdx.x & 63) >> 4);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) my |= __shfl_xor(my, o, MJ_WAVE);
    return __builtin_amdgcn_readfirstlane(my);
}

// Four outputs as fp16.  A mean of V lies among its numbers, but the weights under it are rounded and those in the
// sum are not: up to 2^-11 more, by which fp16's greatest number would round to an infinity.
__device__ __forceinline__ uint2 outputs(f4 o, float l) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (no key seen: zeros)
    uint16_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x = o[i] * inv;
        const uint32_t over = (__float_as_uint(x) & 0x7FFFFFFFu) - 0x477FF000u;  // from 65520 on
        h[i] = (uint16_t)(f2h(x) - (over < 0x7F800000u - 0x477FF000u ? 1 : 0));  // (infinities and NaN stay)
    }
    return make_uint2(pack2(h[0], h[1]), pack2(h[2], h[3]));
}

// A tile's state out: its vectors v .. v + 15 finished, or as a partial result.
__device__ __forceinline__ void write_tile(const PgAttnArgs& a, const PgSeg& S, int v, const PgTile& T, float l) {
    const int lane = threadIdx.x & 63, ln = lane & 15, lq = lane >> 4;
    if (v + ln >= S.vend) return;
    if (S.whole) {
        const int r = (v + ln) / a.G, h = S.g * a.G + (v + ln) - r * a.G;
        uint16_t* o = a.out + (S.su.r0 + r) * a.ldo + h * HD + 4 * lq;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            *(uint2*)(o + 16 * dt) = outputs(T.o[dt], l);
            __builtin_amdgcn_sched_barrier(0);  // (all of them at once take registers that the steps need)
        }
        return;
    }
    const size_t at = (size_t)S.slot * a.cols + (v - S.v0) + ln;
    if (lq == 0) a.pml[at] = make_float2(T.m, l);
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) *(f4*)(a.po + at * HD + 16 * dt + 4 * lq) = T.o[dt];
}

// Several waves' states of the same vectors brought together: the others leave theirs in LDS (put), the
// first takes them up (add).
struct PgLeft {
    f4 o[8][64];
    float m[64], l[64];
};
__device__ __forceinline__ void put_tile(PgLeft& p, const PgTile& T) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) p.o[dt][lane] = T.o[dt];
    p.m[lane] = T.m;
    p.l[lane] = T.l;
}
__device__ __forceinline__ void add_tile(const PgLeft& p, PgTile& T) {
    const int lane = threadIdx.x & 63;
    const float om = p.m[lane], mn = fmaxf(T.m, om);
    const float f0 = T.m == mn ? 1.0f : __builtin_amdgcn_exp2f(T.m - mn);  // (both may be -inf)
    const float f1 = om == mn ? 1.0f : __builtin_amdgcn_exp2f(om - mn);
    T.m = mn;
    T.l = T.l * f0 + p.l[lane] * f1;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) T.o[dt] = T.o[dt] * f0 + p.o[dt][lane] * f1;
}

// A unit that not every row sees whole, straight from the page.
template <int T>
__device__ __forceinline__ void edge_unit(PgTile* tl, const u4v (*q)[4], const PgCol* col, const uint16_t* ku,
                                          const uint16_t* vu, int pos, int L) {
    const int lane = threadIdx.x & 63;
    u4v kr[8], vr[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) kr[k] = ((const u4v*)ku)[64 * k + lane];
#pragma unroll
    for (int k = 0; k < 8; ++k) vr[k] = ((const u4v*)vu)[64 * k + lane];
    __builtin_amdgcn_sched_barrier(0);
    const uint32_t bad = clear_bad(vr);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int y = 0; y < T; ++y) {
        f4 sc[1][2];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
            sc[0][tt] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < 4; ++k) sc[0][tt] = mfma16x16x32(as_h8(kr[4 * tt + k]), as_h8(q[y][k]), sc[0][tt]);
        }
        const uint32_t ok = col[y].mask(pos, L);
        mask_scores(sc[0], ok);
        u4v pw[1][1];
        softmax<1, 1>(&tl[y], sc, pw);
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) tl[y].o[dt] = mfma16x16x32(as_h8(vr[dt]), as_h8(pw[0][0]), tl[y].o[dt]);
        if (bad) add_bad(tl[y], vu, bad, ok);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Up to 16 query vectors a sequence and head.  A block of four waves takes its run of units, a segment at a
// time; a wave takes every fourth unit of it, straight from the pages into registers: a unit's bytes lie in
// the order of the operands.  The next unit's K goes out behind a unit's scores, its V behind the output
// products.  Page numbers of 64 units come with one request a lane.  The states meet in LDS.
// Bound by HBM: one sequence of 131000 tokens and 4 heads takes 50 us (least 49); its 268 MB alone
// would take 45 at the rate of a streaming read.
__global__ __launch_bounds__(256, 2) void k_paged_attn_own(PgAttnArgs a) {
    __shared__ PgPlan plan;
    __shared__ PgLeft s_left[3];
    PgRun run;
    if (!plan_run<256>(a, plan, run)) return;
    const int t = threadIdx.x, lane = t & 63, ln = lane & 15, w = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint16_t* kl = a.p.k + a.layer * a.p.layer_halves();
    const uint16_t* vl = a.p.v + a.layer * a.p.layer_halves();
    bool fresh_block = true;
    for (int64_t x = run.b0; x < run.b1;) {
        const PgSeg S = next_seg(a, plan, run, x);
        if (S.i1 <= S.i0) continue;
        PgTile tl;
        u4v q[1][4];
        bool fresh = true;
        for (int ub = S.i0 + w; ub < S.i1 || fresh; ub += 256) {
            const int mine = ub + 4 * lane;
            const int pl = mine < S.i1 ? seg_page(a, S, mine) : -1;
            if (fresh) {
                load_vector(a, S, S.v0 + ln, q[0]);
                tl.clear();
                fresh = false;
            }
            const int first = S.su.lo + mine;
            const uint64_t edge = __ballot(pl >= 0 && (first < S.clean0 || first >= S.clean1));
            uint64_t todo = __ballot(pl >= 0) & ~edge;
            u4v kr[8], vr[8];
            auto request = [&](u4v* r, const uint16_t* base, int i) {
                const u4v* p =
                    (const u4v*)(base + seg_at(a, S, ub + 4 * i, __builtin_amdgcn_readlane(pl, i))) + lane;
#pragma unroll
                for (int k = 0; k < 8; ++k) r[k] = p[64 * k];
            };
            auto step = [&](int nx, auto more) {  // the unit in registers; unit nx requested behind it
                f4 sc[1][2];
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    sc[0][tt] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        sc[0][tt] = mfma16x16x32(as_h8(kr[4 * tt + k]), as_h8(q[0][k]), sc[0][tt]);
                }
                if constexpr (more.value) request(kr, kl, nx);
                u4v pw[1][1];
                softmax<1, 1>(&tl, sc, pw);
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) tl.o[dt] = mfma16x16x32(as_h8(vr[dt]), as_h8(pw[0][0]), tl.o[dt]);
                if constexpr (more.value) request(vr, vl, nx);
            };
            if (todo) {
                int i0 = __builtin_ctzll(todo);
                request(kr, kl, i0);
                request(vr, vl, i0);
                // (the last unit apart: a request that is not used would be waited for)
                for (todo &= todo - 1; todo; todo &= todo - 1) step(__builtin_ctzll(todo), std::true_type{});
                step(0, std::false_type{});
            }
            if (!edge) continue;
            const PgCol col = load_col(a, S, S.v0 + ln);
#pragma unroll 1
            for (uint64_t e = edge; e; e &= e - 1) {
                const int i = __builtin_ctzll(e);
                const size_t at = seg_at(a, S, ub + 4 * i, __builtin_amdgcn_readlane(pl, i));
                edge_unit<1>(&tl, q, &col, kl + at, vl + at, (S.su.lo + ub + 4 * i) * PG_UNIT, S.su.L);
            }
        }
        if (!fresh_block) __syncthreads();  // (the states of the segment before have been read)
        fresh_block = false;
        if (w > 0) put_tile(s_left[w - 1], tl);
        __syncthreads();
        if (w == 0) {
#pragma unroll 1
            for (int k = 0; k < 3; ++k) add_tile(s_left[k], tl);
            write_tile(a, S, S.v0, tl, x4_sum(tl.l));
        }
    }
}

// More query vectors: a block of eight waves takes its run for up to 256 of them, two tiles a wave.  Units
// go from the pages to LDS by direct loads into a ring of eight, as far ahead as it holds, and the waves
// read their operands from there: one barrier a step, which counts the wave's own requests.  Of few tiles
// the waves split the keys: `ks` groups of waves have all tiles each, and the groups' states meet in LDS at a
// segment's end.  A group takes two units a step (one where ks is 4 and the ring holds two steps of one):
// the softmax's own steps (the maximum over the lanes, the test of the reference) come once for both.
// Where there is one group, the second wave of each SIMD passes the barrier between its weights and its product
// with V instead of before the scores, so that the one multiplies while the other takes exponentials (four
// chunks of 64 rows at 4000 .. 16000 tokens: 48.1 us, in step 49.7; the step before is read a while longer, so
// the ring holds one step less ahead).  Bound by instructions: a step of 64 keys and 256 vectors takes 2.5 us,
// of pages in this XCD's cache 2.4, without the product with V 2.2, and its matrix instructions would take
// 0.85.  Tried: four tiles a wave in four waves (half the LDS reads, no second wave to fill in) 66 us, columns
// of 128 as fast, references moved at every step 56, a wave priority for one of the two no change.
#define PG_SLOTS 8
#define PG_SLOT_BYTES (4 * PG_UNIT_HALVES)
#define PG_CHUNK 1024  // page numbers in LDS
typedef __attribute__((address_space(3))) void* lds_ptr_t;

// At most N of the wave's requests under way, its LDS reads done, then the barrier.
template <int N>
__device__ __forceinline__ void ring_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// U units of LDS against a wave's T tiles, in two halves: scores and weights, then the product with V.  Four
// operands are on their way while the four before them are multiplied (left to itself the compiler requests
// them all at once, and spills).  next: what goes out behind the scores.
template <int T, int U, typename F>
__device__ __forceinline__ void ring_weights(PgTile* tl, const u4v (*q)[4], const char* slot, u4v (*pw)[U], F next) {
    const u4v* base = (const u4v*)slot + (threadIdx.x & 63);
    f4 sc[T][2 * U];
    u4v r[2][4];
    auto at = [&](int i, u4v* x) __attribute__((always_inline)) {  // operands 4 i .. 4 i + 3
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = base[1024 * (i >> 1) + 256 * (i & 1) + 64 * k];
    };
    at(0, r[0]);
#pragma unroll
    for (int i = 0; i < 2 * U; ++i) {
        if (i + 1 < 2 * U) at(i + 1, r[(i + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int y = 0; y < T; ++y) sc[y][i] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int y = 0; y < T; ++y) sc[y][i] = mfma16x16x32(as_h8(r[i & 1][k]), as_h8(q[y][k]), sc[y][i]);
        __builtin_amdgcn_sched_barrier(0);
    }
    next();
    __builtin_amdgcn_sched_barrier(0);
    softmax<T, U>(tl, sc, pw);
    __builtin_amdgcn_sched_barrier(0);
}
template <int T, int U>
__device__ __forceinline__ void ring_values(PgTile* tl, const char* slot, u4v (*pw)[U]) {
    const u4v* base = (const u4v*)slot + 512 + (threadIdx.x & 63);
    u4v r[2][4];
    auto at = [&](int i, u4v* x) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = base[1024 * (i >> 1) + 256 * (i & 1) + 64 * k];
    };
    at(0, r[0]);
#pragma unroll
    for (int i = 0; i < 2 * U; ++i) {
        if (i + 1 < 2 * U) at(i + 1, r[(i + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int y = 0; y < T; ++y) {
                f4& o = tl[y].o[4 * (i & 1) + k];
                o = mfma16x16x32(as_h8(r[i & 1][k]), as_h8(pw[y][i >> 1]), o);
            }
        __builtin_amdgcn_sched_barrier(0);
    }
}

__global__ __launch_bounds__(512, 2) void k_paged_attn_shared(PgAttnArgs a) {
    constexpr int T = 2, NW = 8, NT = 64 * NW;  // tiles a wave, waves
    constexpr int MV = 16 / NW;                 // KB of a unit that a wave moves
    extern __shared__ __align__(16) char ring[];  // [PG_SLOTS][K 8 KB, V 8 KB]; then the states
    __shared__ PgPlan plan;
    __shared__ int s_pg[PG_CHUNK];
    static_assert(3 * NW / 4 * T * sizeof(PgLeft) <= PG_SLOTS * PG_SLOT_BYTES, "states");
    PgRun run;
    if (!plan_run<NT>(a, plan, run)) return;
    const int t = threadIdx.x, lane = t & 63, ln = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint16_t* kl0 = a.p.k + a.layer * a.p.layer_halves();
    const uint16_t* vl0 = a.p.v + a.layer * a.p.layer_halves();
    // the first half of the waves moves K, the other V
    const uint16_t* mover = (w < NW / 2 ? kl0 : vl0) + 512 * MV * (w % (NW / 2)) + 8 * lane;
    for (int64_t x = run.b0; x < run.b1;) {
        const PgSeg S = next_seg(a, plan, run, x);
        if (S.i1 <= S.i0) continue;
        const int tg = (S.vend - S.v0 + 16 * T - 1) / (16 * T);  // waves that have all tiles
        const int ks = NW / tg >= 4 ? 4 : NW / tg >= 2 ? 2 : 1;
        const int kl = w / tg, tw = S.v0 + 16 * T * (w - kl * tg);  // the wave's share of the keys, its first vector
        const bool works = kl < ks;
        PgTile tl[T];
        u4v q[T][4];
#pragma unroll
        for (int i = 0; i < T; ++i) {
            load_vector(a, S, tw + 16 * i + ln, q[i]);
            tl[i].clear();
        }
        // units i0 .. e0 - 1 and e1 .. i1 - 1 are not seen whole by every row
        const int e0 = min(max(S.clean0 - S.su.lo, S.i0), S.i1), e1 = min(max(S.clean1 - S.su.lo, e0), S.i1);
        auto edges = [&]() __attribute__((always_inline)) {
            if (!works || kl >= e0 - S.i0 + S.i1 - e1) return;
            PgCol col[T];
#pragma unroll
            for (int i = 0; i < T; ++i) col[i] = load_col(a, S, tw + 16 * i + ln);
#pragma unroll 1
            for (int e = kl; e < e0 - S.i0 + S.i1 - e1; e += ks) {
                const int i = e < e0 - S.i0 ? S.i0 + e : e1 + e - (e0 - S.i0);
                const int pg = __builtin_amdgcn_readfirstlane(seg_page(a, S, i));
                if (pg < 0) continue;
                const size_t at = seg_at(a, S, i, pg);
                edge_unit<T>(tl, q, col, kl0 + at, vl0 + at, (S.su.lo + i) * PG_UNIT, S.su.L);
            }
        };
        auto go_round = [&](auto us_, auto two_) __attribute__((always_inline)) {
            constexpr int US = us_.value;     // units a group of waves takes a step
            constexpr bool TWO = two_.value;  // one group of waves: half of them a product behind
            const int per = US * ks, slots = PG_SLOTS / per, ahead = slots - 1 - TWO;
            const bool late = TWO && w >= NW / 2;
            for (int c0 = e0; c0 == e0 || c0 < e1; c0 += PG_CHUNK) {  // (once for the edges alone)
                const int n = min(e1 - c0, PG_CHUNK), steps = (n + per - 1) / per;
                for (int i = t; i < n; i += NT) s_pg[i] = seg_page(a, S, c0 + i);
                __syncthreads();  // (and the ring is free)
                auto request = [&](int step) {
#pragma unroll 1
                    for (int u = 0; u < per; ++u) {
                        const int i = min(step * per + u, n - 1), pg = __builtin_amdgcn_readfirstlane(s_pg[i]);
                        const uint16_t* src = mover + seg_at(a, S, c0 + i, max(pg, 0));  // (page 0 for none: unread)
                        char* dst = ring + ((step & (slots - 1)) * per + u) * PG_SLOT_BYTES + 1024 * MV * w;
#pragma unroll
                        for (int k = 0; k < MV; ++k)
                            __builtin_amdgcn_global_load_lds(src + 512 * k, (lds_ptr_t)(dst + 1024 * k), 16, 0, 0);
                    }
                };
                for (int j = 0; j < min(ahead, steps); ++j) request(j);
                if (c0 == e0) edges();  // (while the ring fills)
                // step j is there for all, and everyone is done with the one whose slots are filled next
                auto there = [&](int j) __attribute__((always_inline)) {
                    if (ahead == 1 || steps - 1 - j < ahead - 1) ring_barrier<0>();
                    else ring_barrier<MV * US * (PG_SLOTS / US - 2 - TWO)>();  // (ks 1)
                };
#pragma unroll 1
                for (int j = 0; j < steps; ++j) {
                    if (!late || j == 0) there(j);
                    const bool more = j + ahead < steps;
                    auto next = [&]() __attribute__((always_inline)) {
                        if (more) request(j + ahead);
                    };
                    const int i = per * j + US * kl;
                    bool all = works && i + US <= n;
                    if (all)
#pragma unroll
                        for (int u = 0; u < US; ++u) all &= __builtin_amdgcn_readfirstlane(s_pg[i + u]) >= 0;
                    const char* here = ring + ((j & (slots - 1)) * per + US * kl) * PG_SLOT_BYTES;
                    if (all) {
                        u4v pw[T][US];
                        ring_weights<T, US>(tl, q, here, pw, next);
                        if (late && j + 1 < steps) there(j + 1);
                        ring_values<T, US>(tl, here, pw);
                        continue;
                    }
                    next();
                    if constexpr (US > 1)
                        if (works)
#pragma unroll 1
                            for (int u = 0; u < US; ++u)
                                if (i + u < n && __builtin_amdgcn_readfirstlane(s_pg[i + u]) >= 0) {
                                    u4v p1[T][1];
                                    ring_weights<T, 1>(tl, q, here + u * PG_SLOT_BYTES, p1, []() {});
                                    ring_values<T, 1>(tl, here + u * PG_SLOT_BYTES, p1);
                                }
                    if (late && j + 1 < steps) there(j + 1);
                }
                __syncthreads();  // (the page numbers and the ring have been read)
            }
        };
        using One = std::integral_constant<int, 1>;
        using Two = std::integral_constant<int, 2>;
        if (ks == 4) go_round(One{}, std::false_type{});
        else if (ks == 2) go_round(Two{}, std::false_type{});
        else go_round(Two{}, std::true_type{});
        PgLeft* left = (PgLeft*)ring;
        if (ks > 1) {
            if (works && kl > 0)
#pragma unroll
                for (int i = 0; i < T; ++i) put_tile(left[(w - tg) * T + i], tl[i]);
            __syncthreads();
        }
        if (kl == 0) {
#pragma unroll
            for (int i = 0; i < T; ++i) {
#pragma unroll 1
                for (int k = 1; k < ks; ++k) add_tile(left[(w + (k - 1) * tg) * T + i], tl[i]);
                if (tw + 16 * i < S.vend) write_tile(a, S, tw + 16 * i, tl[i], x4_sum(tl[i].l));
            }
        }
    }
}

// The partial results of a row's heads, where their keys went to several blocks: a block of four waves takes
// one head together, or, of many rows, four heads, a wave each.  A group of 32 lanes has a share of the
// blocks, four dims a lane; references, sums and outputs are requested together, eight blocks a group and
// round.  (References first, then outputs against the greatest: 10 us for 128 blocks; sixteen groups for
// every head: 22 us for 4096 of them.)
template <int WAVES>
__global__ __launch_bounds__(256) void k_paged_join(PgAttnArgs a) {
    constexpr int GR = 2 * WAVES;
    __shared__ f4 s_o[WAVES == 1 ? 1 : GR][32];
    __shared__ float2 s_ml[GR];
    __shared__ int s_abort;
    const int t = threadIdx.x, lane = t & 63, d = t & 31, r = blockIdx.x;
    const int h = WAVES == 1 ? 4 * blockIdx.y + (t >> 6) : blockIdx.y;
    // Of up to 64 sequences all that a row's may need is requested at once, a sequence a lane.
    const int ab = abort_word(a.abort), n_seqs = a.b.n_seqs, mine = min(lane, n_seqs - 1);
    const int64_t per = a.off[n_seqs + 1];
    int r0, m = pg_rows(a.b, mine, r0), L = pg_len(a.p, mine);
    int64_t S = a.off[mine];
    const int s = pg_seq(a.b, r);
    if (t == 0) s_abort = ab;
    __syncthreads();
    if (s_abort || s >= n_seqs || h >= a.p.nKV * a.G) return;  // (h: a whole wave, and the block has no barrier then)
    if (n_seqs <= 64) {
        m = __builtin_amdgcn_readlane(m, s);
        r0 = __builtin_amdgcn_readlane(r0, s);
        L = __builtin_amdgcn_readlane(L, s);
        S = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(S >> 32), s) << 32 |
                      (uint32_t)__builtin_amdgcn_readlane((int)S, s));
    } else {
        m = pg_rows(a.b, s, r0);
        L = pg_len(a.p, s);
        S = a.off[s];
    }
    const SeqUnits su = seq_units(a, m, r0, L);
    const int local = r - su.r0;
    if (local < 0 || local >= su.m) return;
    uint16_t* out = a.out + r * a.ldo + h * HD;
    const int g = h / a.G, v = local * a.G + h - g * a.G, c = v / a.cols, cc = v - c * a.cols;
    S += ((int64_t)g * su.ncg + c) * (su.nu + a.extra);
    const int64_t E = S + su.nu + a.extra;
    if (su.nu == 0) {
        if (WAVES == 1 ? lane < 32 : t < 32) *(uint2*)(out + 4 * d) = make_uint2(0u, 0u);
        return;
    }
    const int bA = (int)quotient(S + a.extra, per), n = (int)quotient(E - 1, per) - bA + 1;
    if (n == 1) return;
    const int k = WAVES == 1 ? lane >> 5 : t >> 5;
    float M = -INFINITY, l = 0.0f;
    f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int i = k; i < n; i += 8 * GR) {
        f4 y[8];
        float2 ml[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // (a block that begins in this segment has it first, another one last)
            const int64_t b = bA + min(i + j * GR, n - 1);
            const size_t at = ((size_t)b * 2 + (S <= b * per ? 0 : 1)) * a.cols + cc;
            ml[j] = a.pml[at];
            y[j] = *(const f4*)(a.po + at * HD + 4 * d);
        }
        float mn = M;
#pragma unroll
        for (int j = 0; j < 8; ++j) mn = i + j * GR < n ? fmaxf(mn, ml[j].x) : mn;
        const float f0 = M == mn ? 1.0f : __builtin_amdgcn_exp2f(M - mn);  // (both may be -inf)
        M = mn;
        l *= f0;
        o *= f0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float f = i + j * GR >= n ? 0.0f : ml[j].x == mn ? 1.0f : __builtin_amdgcn_exp2f(ml[j].x - mn);
            if (i + j * GR < n) {
                l = fmaf(ml[j].y, f, l);
                o += y[j] * f;
            }
        }
    }
    // the groups: two of a wave by lane moves, or all through LDS
    if constexpr (WAVES == 1) {
        const float om = __shfl_xor(M, 32, MJ_WAVE), ol = __shfl_xor(l, 32, MJ_WAVE), mn = fmaxf(M, om);
        const float f0 = M == mn ? 1.0f : __builtin_amdgcn_exp2f(M - mn);
        const float f1 = om == mn ? 1.0f : __builtin_amdgcn_exp2f(om - mn);
        // (the lower group's share first in both, so that both have the same bits)
        l = k == 0 ? l * f0 + ol * f1 : ol * f1 + l * f0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float oo = __shfl_xor(o[j], 32, MJ_WAVE);
            o[j] = o[j] * f0 + oo * f1;
        }
        if (k) return;
    } else {
        if (d == 0) s_ml[k] = make_float2(M, l);
        s_o[k][d] = o;
        __syncthreads();
        if (t >= 32) return;
        M = -INFINITY;
#pragma unroll
        for (int i = 0; i < GR; ++i) M = fmaxf(M, s_ml[i].x);
        l = 0.0f;
        o = (f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < GR; ++i) {
            const float2 ml = s_ml[i];
            const float f = ml.x == M ? 1.0f : __builtin_amdgcn_exp2f(ml.x - M);
            l += ml.y * f;
            o += s_o[i][d] * f;
        }
    }
    *(uint2*)(out + 4 * d) = outputs(o, l);
}

// Up to 16 vectors the blocks are of the first kernel, which needs no barriers: 131000 tokens, one vector a head
// 50.4 us against 54.0, 64 sequences of 200..8000 tokens 55.6 against 62.9, one of 300 7.3 against 11.5.  (The greatest
// count of rows decides for the whole batch: a chunk of 64 rows among 63 of one takes 99 us, the two in calls of their
// own 78.)  Past 16 the ring's: the first kernel with two tiles spills (eight rows at 8000 tokens, four heads a group: 50
// us against 32), and its waves would all read every unit.  One block of 256 vectors, though two of 128 would
// divide the work more evenly: as fast (53.2 and 53.1 us), with half the reads.
// A segment's beginning (its rows' queries, page numbers, the ring filled, the result written) costs as much
// as 10 units of the ring (17 rows of 16 sequences 28.7 us; counted as 6 units 30.5) or 8 of the first kernel
// (64 sequences of 200..8000 tokens 55.6 us, as 2 units 57.5, as 16 56.8).
// A block takes four units at least, those that count for beginnings among them, so a short segment still has
// several blocks (nine rows of four sequences of 200..400 tokens 18 us; with four units of keys at least 23).
size_t paged_attn_plan(PgAttnArgs& a, void* base) {
    const int nv = a.b.max_rows * a.G;
    a.cols = nv <= 16 ? 16 : std::min((nv + 31) / 32 * 32, 256);
    a.blocks = a.cols == 16 ? 512 : 256;  // two a CU, or one
    a.extra = a.cols == 16 ? 8 : 10;
    a.least = 4;
    Arena ar{base, 0};
    a.off = (int64_t*)ar.take((PG_MAX_SEQS + 2) * sizeof(int64_t));
    a.pml = (float2*)ar.take((size_t)a.blocks * 2 * a.cols * sizeof(float2));
    a.po = (float*)ar.take((size_t)a.blocks * 2 * a.cols * HD * sizeof(float));
    return ar.off;
}

static hipError_t launch_shared(const PgAttnArgs& a, hipStream_t st) {
    static std::atomic<uint64_t> raised{0};  // the devices whose LDS limit is raised
    constexpr int lds = PG_SLOTS * PG_SLOT_BYTES;
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (!(raised.load(std::memory_order_relaxed) & bit)) {
        e = hipFuncSetAttribute((const void*)k_paged_attn_shared, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
        raised.fetch_or(bit, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL(k_paged_attn_shared, dim3(a.blocks), dim3(512), lds, st, a);
    return hipSuccess;
}

hipError_t launch_paged_attn(const PgAttnArgs& a, hipStream_t st) {
    if (a.b.n_seqs > PG_MAX_SEQS || a.b.rows < 1 || a.b.max_rows > MJ_ROWS || a.p.page < PG_UNIT ||
        a.blocks > PG_MAX_BLOCKS)
        return hipErrorInvalidValue;
    if (a.cols == 16) {
        hipLaunchKernelGGL(k_paged_attn_own, dim3(a.blocks), dim3(256), 0, st, a);
    } else {
        const hipError_t e = launch_shared(a, st);
        if (e != hipSuccess) return e;
    }
    const int heads = a.p.nKV * a.G;
    if ((int64_t)a.b.rows * heads >= 2048)
        hipLaunchKernelGGL(k_paged_join<1>, dim3(a.b.rows, (heads + 3) / 4), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL(k_paged_join<4>, dim3(a.b.rows, heads), dim3(256), 0, st, a);
    return hipGetLastError();
}
