// paged_attn.hip -- attention of a batch's rows over the fp16 pages of their sequences.
//
// softmax(q k^T / sqrt(128)) v in one pass over the keys with a running reference and sum.  A unit is
// 32 keys of one sequence, KV head and column group (at most `cols` query vectors: a row's heads of the group,
// row by row); the units of the batch are numbered in that order, so a block takes a run of consecutive
// ones and its work does not depend on how long which sequence is.  A run is cut where a sequence, head or
// column group ends; a segment that is all of its group's keys is finished by its block, others leave a
// partial result, and k_paged_join puts these together.  Scores are kept in log2 units.
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
__device__ __forceinline__ SeqUnits seq_units(const PgAttnArgs& a, int s) {
    SeqUnits u;
    u.m = pg_rows(a.b, s, u.r0);
    u.L = pg_len(a.p, s);
    const int end = min(u.L + u.m, a.p.room());
    u.lo = (a.window > 0 ? max(0, u.L - a.window + 1) : 0) / PG_UNIT;
    u.nu = u.m > 0 ? max(0, (end + PG_UNIT - 1) / PG_UNIT - u.lo) : 0;
    u.ncg = (u.m * a.G + a.cols - 1) / a.cols;
    return u;
}

// A tile of 16 query vectors, outputs turned: lane (ln, lq) holds vector ln's reference, its share of the
// sum, and dims 16 dt + 4 lq + r of its output.
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
// Scores past FAR: a weight's one fma differs from the rounded score by more than the slack allows, so
// the reference is taken off the rounded scores, in the branch that moves it.
#define FAR 1048576.0f

// Softmax of a unit's scores against the running state.  S[t]: vector ln against tokens 8 lq + 4 t + r,
// without the scale; masked ones -inf.  p: the weights as the B operand of the product with V.
__device__ __forceinline__ u4v unit_weights(PgTile& T, f4 S[2]) {
    float x = fmaxf(fmaxf(fmaxf(S[0][0], S[0][1]), fmaxf(S[0][2], S[0][3])),
                    fmaxf(fmaxf(S[1][0], S[1][1]), fmaxf(S[1][2], S[1][3])));
    x = x4_max(x);
    const float s = product(x, SC2);
    float ref = T.m;
    if (__any((s > T.m + SLACK) | (fabsf(s) > FAR))) {
        const bool far = fabsf(s) > FAR && s > -INFINITY;  // (-inf: every score is masked)
        const float mn = fmaxf(T.m, s);
        const float alpha = T.m == mn ? 1.0f : __builtin_amdgcn_exp2f(T.m - mn);  // (both may be -inf)
        T.m = mn;
        T.l *= alpha;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) T.o[dt] *= alpha;
        ref = far ? 0.0f : mn;
        if (__any(far)) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    S[t][r] = far ? (product(S[t][r], SC2) - mn) * (1.0f / SC2) : S[t][r];
        }
    }
    // no key seen: any finite reference (a masked score still gives 0, a NaN stays one)
    const float c = LIFT - (ref == -INFINITY ? 0.0f : ref);
    u4v p;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float w0 = __builtin_amdgcn_exp2f(fmaf(S[i >> 1][2 * (i & 1)], SC2, c));
        const float w1 = __builtin_amdgcn_exp2f(fmaf(S[i >> 1][2 * (i & 1) + 1], SC2, c));
        sum += w0;
        sum += w1;
        p[i] = pack2(f2h(w0), f2h(w1));
    }
    T.l += sum;
    return p;
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

// Units before each sequence (s_off[0 .. n]) and the run of this block, by one round of requests and a scan
// for every NT sequences; a.off gets them for the join.  False: the call was aborted.
struct PgRun {
    int64_t b0, b1, per;
    int s;  // the sequence that the run begins in
};
template <int NT>
__device__ __forceinline__ bool plan_run(const PgAttnArgs& a, int64_t* s_off, int64_t* s_wsum, int* s_abort,
                                         PgRun& run) {
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, n = a.b.n_seqs;
    const int ab = a.abort ? *a.abort : 0;
    int64_t before = 0;
    for (int c = 0; c < n; c += NT) {
        int64_t u = 0;
        if (c + t < n) {
            const SeqUnits q = seq_units(a, c + t);
            u = (int64_t)q.nu * q.ncg * a.p.nKV;
        }
        int64_t inc = u;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t x = __shfl_up(inc, o, MJ_WAVE);
            inc += lane >= o ? x : 0;
        }
        if (c) __syncthreads();
        if (lane == 63) s_wsum[w] = inc;
        if (t == 0 && c == 0) *s_abort = ab;
        __syncthreads();
        int64_t at = before, all = before;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) {
            at += i < w ? s_wsum[i] : 0;
            all += s_wsum[i];
        }
        if (c + t <= n) s_off[c + t] = at + inc - u;
        if (c + t + 1 == n) s_off[n] = at + inc;
        before = all;
    }
    __syncthreads();
    if (*s_abort) return false;
    run.per = max((before + a.blocks - 1) / a.blocks, (int64_t)a.least);
    if (blockIdx.x == 0)
        for (int i = t; i <= n + 1; i += NT) a.off[i] = i <= n ? s_off[i] : run.per;
    run.b0 = blockIdx.x * run.per;
    run.b1 = min(before, run.b0 + run.per);
    run.s = 0;
    if (run.b0 < run.b1) {  // the last sequence that begins at or before the run
        int hi = n;
        while (hi - run.s > 1) {
            const int mid = (run.s + hi) >> 1;
            if (s_off[mid] <= run.b0) run.s = mid;
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
__device__ __forceinline__ PgSeg next_seg(const PgAttnArgs& a, const int64_t* s_off, PgRun& run, int64_t x) {
    while (s_off[run.s + 1] <= x) ++run.s;
    PgSeg S;
    S.s = run.s;
    S.su = seq_units(a, S.s);
    const int64_t rel = x - s_off[S.s];
    const int gc = (int)(rel / S.su.nu);
    S.i0 = (int)(rel - (int64_t)gc * S.su.nu);
    S.i1 = (int)min((int64_t)S.su.nu, S.i0 + (run.b1 - x));
    S.g = gc / S.su.ncg;
    S.v0 = (gc - S.g * S.su.ncg) * a.cols;
    S.vend = min(S.su.m * a.G, S.v0 + a.cols);
    S.clean0 = a.window > 0 ? (max(0, S.su.L + MJ_ROWS - a.window + 1) + PG_UNIT - 1) / PG_UNIT : 0;
    S.clean1 = S.su.L / PG_UNIT;
    S.whole = S.i0 == 0 && S.i1 == S.su.nu;
    S.slot = (int64_t)blockIdx.x * 2 + (x == run.b0 ? 0 : 1);
    return S;
}
// The page of the segment's unit i, or -1.
__device__ __forceinline__ int seg_page(const PgAttnArgs& a, const PgSeg& S, int i) {
    return pg_page(a.p, S.s, ((S.su.lo + i) * PG_UNIT) >> a.p.shift);
}
// Halves from a layer's first to the segment's unit i in page pg.
__device__ __forceinline__ size_t seg_at(const PgAttnArgs& a, const PgSeg& S, int i, int pg) {
    const int in = ((S.su.lo + i) * PG_UNIT) & (a.p.page - 1);
    return ((size_t)pg * a.p.nKV + S.g) * a.p.head_halves() + (size_t)(in >> 5) * PG_UNIT_HALVES;
}

// Query vector v (lanes without one take the group's first, unused) and what its row sees.
__device__ __forceinline__ void load_vector(const PgAttnArgs& a, const PgSeg& S, int v, u4v q[4], PgCol& col) {
    const int lq = (threadIdx.x & 63) >> 4;
    col.on = v < S.vend;
    const int r = col.on ? v / a.G : 0, h = S.g * a.G + (col.on ? v - r * a.G : 0);
    const uint16_t* qp = a.q + (S.su.r0 + r) * a.ldq + h * HD + 8 * lq;
#pragma unroll
    for (int k = 0; k < 4; ++k) q[k] = *(const u4v*)(qp + 32 * k);
    col.anc = pg_anc(a.b, S.su.r0 + r, r);
    const int depth = pg_depth(col.anc, r);
    if (S.su.m < 64) col.anc &= (1ull << S.su.m) - 1;  // (a row that there is not is nobody's ancestor)
    col.first = a.window > 0 ? max(0, S.su.L + depth - a.window + 1) : 0;
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
    return my;
}

// A tile's state out: its vectors v .. v + 15 finished, or as a partial result.
__device__ __forceinline__ void write_tile(const PgAttnArgs& a, const PgSeg& S, int v, const PgTile& T, float l) {
    const int lane = threadIdx.x & 63, ln = lane & 15, lq = lane >> 4;
    if (v + ln >= S.vend) return;
    if (S.whole) {
        const int r = (v + ln) / a.G, h = S.g * a.G + (v + ln) - r * a.G;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (no key seen: zeros)
        uint16_t* o = a.out + (S.su.r0 + r) * a.ldo + h * HD + 4 * lq;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt)
            *(uint2*)(o + 16 * dt) = make_uint2(pack2(f2h(T.o[dt][0] * inv), f2h(T.o[dt][1] * inv)),
                                                pack2(f2h(T.o[dt][2] * inv), f2h(T.o[dt][3] * inv)));
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

// Up to 16 T query vectors a sequence and head.  A block of four waves takes its run of units, a segment at a
// time; a wave takes every fourth unit of it, straight from the pages into registers: a unit's bytes lie in
// the order of the operands.  The next unit's K goes out behind a unit's scores, its V behind the output
// products.  Page numbers of 64 units come with one request a lane.  The states meet in LDS.
template <int T>
__global__ __launch_bounds__(256, 2) void k_paged_attn_own(PgAttnArgs a) {
    __shared__ int64_t s_off[PG_MAX_SEQS + 1], s_wsum[4];
    __shared__ int s_abort;
    __shared__ PgLeft s_left[3][T];
    PgRun run;
    if (!plan_run<256>(a, s_off, s_wsum, &s_abort, run)) return;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, ln = lane & 15;
    const uint16_t* kl = a.p.k + a.layer * a.p.layer_halves();
    const uint16_t* vl = a.p.v + a.layer * a.p.layer_halves();
    for (int64_t x = run.b0; x < run.b1;) {
        const PgSeg S = next_seg(a, s_off, run, x);
        PgTile tl[T];
        PgCol col[T];
        u4v q[T][4], kr[8], vr[8];
        bool fresh = true;
        for (int ub = S.i0 + w; ub < S.i1 || fresh; ub += 256) {
            const int mine = ub + 4 * lane;
            const int pl = mine < S.i1 ? seg_page(a, S, mine) : -1;
            if (fresh) {
#pragma unroll
                for (int i = 0; i < T; ++i) {
                    load_vector(a, S, S.v0 + 16 * i + ln, q[i], col[i]);
                    tl[i].clear();
                }
                fresh = false;
            }
            const int first = S.su.lo + mine;
            const uint64_t edge = __ballot(pl >= 0 && (first < S.clean0 || first >= S.clean1));
            uint64_t todo = __ballot(pl >= 0) & ~edge;
            auto request = [&](u4v* r, const uint16_t* base, int i) {
                const u4v* p =
                    (const u4v*)(base + seg_at(a, S, ub + 4 * i, __builtin_amdgcn_readlane(pl, i))) + lane;
#pragma unroll
                for (int k = 0; k < 8; ++k) r[k] = p[64 * k];
            };
            // unit i; MORE: unit nx requested behind it; EDGE: not every row sees all of it
            auto step = [&](int i, int nx, auto more, auto masked) {
                f4 sc[T][2];
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
                    for (int j = 0; j < T; ++j) sc[j][tt] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int j = 0; j < T; ++j)
                            sc[j][tt] = mfma16x16x32(as_h8(kr[4 * tt + k]), as_h8(q[j][k]), sc[j][tt]);
                }
                if constexpr (more.value) request(kr, kl, nx);
                uint32_t bad = 0;
                const int pos = (S.su.lo + ub + 4 * i) * PG_UNIT;
                if constexpr (masked.value) {
#pragma unroll
                    for (int j = 0; j < T; ++j) mask_scores(sc[j], col[j].mask(pos, S.su.L));
                    bad = clear_bad(vr);
                }
                u4v pw[T];
#pragma unroll
                for (int j = 0; j < T; ++j) pw[j] = unit_weights(tl[j], sc[j]);
#pragma unroll
                for (int dt = 0; dt < 8; ++dt)
#pragma unroll
                    for (int j = 0; j < T; ++j)
                        tl[j].o[dt] = mfma16x16x32(as_h8(vr[dt]), as_h8(pw[j]), tl[j].o[dt]);
                if constexpr (more.value) request(vr, vl, nx);
                if constexpr (masked.value)
                    if (bad) {
                        const uint16_t* vu = vl + seg_at(a, S, ub + 4 * i, __builtin_amdgcn_readlane(pl, i));
#pragma unroll
                        for (int j = 0; j < T; ++j) add_bad(tl[j], vu, bad, col[j].mask(pos, S.su.L));
                    }
            };
            int i0 = todo ? __builtin_ctzll(todo) : -1;
            if (i0 >= 0) {
                request(kr, kl, i0);
                request(vr, vl, i0);
            }
            // (the last unit apart: a request that is not used would be waited for)
            while (todo) {
                const int i = i0;
                todo &= todo - 1;
                if (!todo) break;
                i0 = __builtin_ctzll(todo);
                step(i, i0, std::true_type{}, std::false_type{});
            }
            if (i0 >= 0) step(i0, 0, std::false_type{}, std::false_type{});
#pragma unroll 1
            for (uint64_t e = edge; e; e &= e - 1) {
                i0 = __builtin_ctzll(e);
                request(kr, kl, i0);
                request(vr, vl, i0);
                step(i0, 0, std::false_type{}, std::true_type{});
            }
        }
        if (x != run.b0) __syncthreads();  // (the states of the segment before have been read)
        if (w > 0)
#pragma unroll
            for (int i = 0; i < T; ++i) put_tile(s_left[w - 1][i], tl[i]);
        __syncthreads();
        if (w == 0)
#pragma unroll
            for (int i = 0; i < T; ++i) {
#pragma unroll 1
                for (int k = 0; k < 3; ++k) add_tile(s_left[k][i], tl[i]);
                write_tile(a, S, S.v0 + 16 * i, tl[i], x4_sum(tl[i].l));
            }
        x += S.i1 - S.i0;
    }
}

// The partial results of one row and head, where its keys went to several blocks: their references and sums
// first, then sixteen groups of 32 lanes take every sixteenth block's outputs, four dims a lane, with several
// on their way (one at a time, each waited for, 128 blocks took 10 us), and the groups meet in LDS.
#define PG_JOIN 512
__global__ __launch_bounds__(PG_JOIN) void k_paged_join(PgAttnArgs a) {
    __shared__ f4 s_o[PG_JOIN / 32][32];
    __shared__ float s_f[PG_MAX_BLOCKS], s_w[2][PG_JOIN / 64];
    if (block_aborted(a.abort)) return;
    const int t = threadIdx.x, r = blockIdx.x, h = blockIdx.y, s = pg_seq(a.b, r);
    if (s >= a.b.n_seqs) return;
    const SeqUnits su = seq_units(a, s);
    const int local = r - su.r0;
    if (local < 0 || local >= su.m) return;
    uint16_t* out = a.out + r * a.ldo + h * HD;
    const int g = h / a.G, v = local * a.G + h - g * a.G, c = v / a.cols, cc = v - c * a.cols;
    const int64_t per = a.off[a.b.n_seqs + 1];
    const int64_t S = a.off[s] + ((int64_t)g * su.ncg + c) * su.nu, E = S + su.nu;
    if (su.nu == 0) {
        if (t < 16) *(u4v*)(out + 8 * t) = (u4v){0u, 0u, 0u, 0u};
        return;
    }
    const int bA = (int)(S / per), n = (int)((E - 1) / per) - bA + 1;
    if (n == 1) return;
    // (blocks before the last one of a run begin it: their first slot; the first block's last segment is this one)
    auto place = [&](int i) {
        const int64_t b = bA + i;
        return ((size_t)b * 2 + (S <= b * per ? 0 : 1)) * a.cols + cc;
    };
    float M = -INFINITY, l = 0.0f;
    for (int i = t; i < n; i += PG_JOIN) M = fmaxf(M, a.pml[place(i)].x);
    M = wave_max(M);
    if ((t & 63) == 0) s_w[0][t >> 6] = M;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PG_JOIN / 64; ++i) M = fmaxf(M, s_w[0][i]);
    for (int i = t; i < n; i += PG_JOIN) {
        const float2 ml = a.pml[place(i)];
        const float f = ml.x == M ? 1.0f : __builtin_amdgcn_exp2f(ml.x - M);
        s_f[i] = f;
        l = fmaf(ml.y, f, l);
    }
    l = wave_sum(l);
    if ((t & 63) == 0) s_w[1][t >> 6] = l;
    __syncthreads();
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < PG_JOIN / 64; ++i) l += s_w[1][i];
    const int k = t >> 5, d = t & 31;
    f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = k; i < n; i += 4 * (PG_JOIN / 32)) {
        f4 y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int b = min(i + j * (PG_JOIN / 32), n - 1);
            y[j] = *(const f4*)(a.po + place(b) * HD + 4 * d);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j * (PG_JOIN / 32) < n) o += y[j] * s_f[i + j * (PG_JOIN / 32)];
    }
    s_o[k][d] = o;
    __syncthreads();
    if (t >= 32) return;
    o = s_o[0][d];
#pragma unroll
    for (int i = 1; i < PG_JOIN / 32; ++i) o += s_o[i][d];
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (no key seen: zeros)
    *(uint2*)(out + 4 * d) = make_uint2(pack2(f2h(o[0] * inv), f2h(o[1] * inv)),
                                        pack2(f2h(o[2] * inv), f2h(o[3] * inv)));
}

size_t paged_attn_plan(PgAttnArgs& a, void* base) {
    const int nv = a.b.max_rows * a.G;
    a.cols = nv <= 16 ? 16 : 32;
    a.blocks = 512;  // two a CU
    a.least = 4;
    Arena ar{base, 0};
    a.off = (int64_t*)ar.take((PG_MAX_SEQS + 2) * sizeof(int64_t));
    a.pml = (float2*)ar.take((size_t)a.blocks * 2 * a.cols * sizeof(float2));
    a.po = (float*)ar.take((size_t)a.blocks * 2 * a.cols * HD * sizeof(float));
    return ar.off;
}

hipError_t launch_paged_attn(const PgAttnArgs& a, hipStream_t st) {
    if (a.b.n_seqs > PG_MAX_SEQS || a.b.rows < 1 || a.b.max_rows > MJ_ROWS || a.p.page < PG_UNIT)
        return hipErrorInvalidValue;
    if (a.cols == 16)
        hipLaunchKernelGGL(k_paged_attn_own<1>, dim3(a.blocks), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL(k_paged_attn_own<2>, dim3(a.blocks), dim3(256), 0, st, a);
    hipLaunchKernelGGL(k_paged_join, dim3(a.b.rows, a.p.nKV * a.G), dim3(PG_JOIN), 0, st, a);
    return hipGetLastError();
}
