// paged_attn.hip -- attention of a batch's rows over the fp16 pages of their sequences.
//
// softmax(q k^T / sqrt(128)) v in one pass over the keys with a running reference and sum.  A unit is
// 32 keys of one sequence, KV head and column group (at most `cols` query vectors: a row's heads of the group,
// row by row); the units of the batch are numbered in that order, so a block takes a run of consecutive
// ones and its work does not depend on how long which sequence is.  A run is cut where a sequence, head or
// column group ends; a segment that is all of its group's keys is finished by its block, others leave a
// partial result, and k_paged_join puts these together.  Scores are kept in log2 units.
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

// Infinities and NaN of V in a unit that not every row sees whole (0 times an infinity is a NaN): they are
// left out of the product and added here to the outputs of the vectors that attend to them, whatever
// their weights (which are above 0, if not in fp32).  ok: the unit's tokens that vector ln sees.
__device__ __forceinline__ void add_bad(PgTile& T, const uint16_t* vu, uint32_t bad, uint32_t ok) {
    const int lq = (threadIdx.x & 63) >> 4;
#pragma unroll 1
    for (; bad; bad &= bad - 1) {
        const int t = __builtin_ctz(bad);
        const bool sees = (ok >> t) & 1;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float v = h2f(vu[pg_v_at(t, 16 * dt + 4 * lq + r)]);
                T.o[dt][r] += sees && !(fabsf(v) < INFINITY) ? v : 0.0f;
            }
    }
}

// A block of four waves takes its run of units, a segment at a time; a wave takes every fourth unit of
// it, straight from the pages into registers, and the four states meet in LDS.
__global__ __launch_bounds__(256) void k_paged_attn(PgAttnArgs a) {
    __shared__ int64_t s_off[PG_MAX_SEQS + 1];
    __shared__ int64_t s_wsum[4];
    __shared__ float s_o[4][16][HD + 4];
    __shared__ float2 s_ml[4][16];
    if (block_aborted(a.abort)) return;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, ln = lane & 15, lq = lane >> 4;
    {
        int64_t u[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = 0;
            if (4 * t + i < a.b.n_seqs) {
                const SeqUnits q = seq_units(a, 4 * t + i);
                u[i] = (int64_t)q.nu * q.ncg * a.p.nKV;
            }
            sum += u[i];
        }
        int64_t inc = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t x = __shfl_up(inc, o, MJ_WAVE);
            inc += lane >= o ? x : 0;
        }
        if (lane == 63) s_wsum[w] = inc;
        __syncthreads();
        int64_t at = inc - sum;
        for (int i = 0; i < w; ++i) at += s_wsum[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (4 * t + i <= a.b.n_seqs) s_off[4 * t + i] = at;
            at += u[i];
        }
        if (t == 255 && a.b.n_seqs == PG_MAX_SEQS) s_off[PG_MAX_SEQS] = at;
        __syncthreads();
    }
    const int n = a.b.n_seqs;
    const int64_t total = s_off[n];
    const int64_t per = max((total + a.blocks - 1) / a.blocks, (int64_t)4);
    if (blockIdx.x == 0)
        for (int i = t; i <= n + 1; i += 256) a.off[i] = i <= n ? s_off[i] : per;
    const int64_t b0 = blockIdx.x * per, b1 = min(total, b0 + per);
    int64_t x = b0;
    int s = 0;
    if (x < b1) {  // the last sequence that begins at or before the run
        int hi = n;
        while (hi - s > 1) {
            const int mid = (s + hi) >> 1;
            if (s_off[mid] <= x) s = mid;
            else hi = mid;
        }
    }
    while (x < b1) {
        while (s_off[s + 1] <= x) ++s;
        const SeqUnits su = seq_units(a, s);
        const int64_t rel = x - s_off[s];
        const int gc = (int)(rel / su.nu), i0 = (int)(rel - (int64_t)gc * su.nu);
        const int i1 = (int)min((int64_t)su.nu, i0 + (b1 - x));
        const int g = gc / su.ncg, c = gc - g * su.ncg;
        const int v0 = c * a.cols, nv = su.m * a.G;
        // the vectors
        PgCol col;
        const int v = v0 + ln;
        col.on = v < nv;
        const int vr = col.on ? v / a.G : 0, vh = g * a.G + (col.on ? v - vr * a.G : 0);
        col.anc = pg_anc(a.b, su.r0 + vr, vr);
        if (su.m < 64) col.anc &= (1ull << su.m) - 1;  // (a row that there is not is nobody's ancestor)
        col.first = a.window > 0 ? max(0, su.L + pg_depth(col.anc, vr) - a.window + 1) : 0;
        u4v q[4];
        const uint16_t* qp = a.q + (su.r0 + vr) * a.ldq + vh * HD + 8 * lq;
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = *(const u4v*)(qp + 32 * k);
        // units before `clean` (of those behind the window's first whole one) are seen whole by every row
        const int clean0 = a.window > 0 ? (max(0, su.L + MJ_ROWS - a.window + 1) + PG_UNIT - 1) / PG_UNIT : 0;
        const int clean1 = su.L / PG_UNIT;
        PgTile T;
        T.clear();
        for (int i = i0 + w; i < i1; i += 4) {
            const int unit = su.lo + i, pos = unit * PG_UNIT;
            const int pg = pg_page(a.p, s, pos >> a.p.shift);
            if (pg < 0) continue;
            const size_t at = a.layer * a.p.layer_halves() + ((size_t)pg * a.p.nKV + g) * a.p.head_halves() +
                              (size_t)((pos & (a.p.page - 1)) >> 5) * PG_UNIT_HALVES;
            const u4v* ku = (const u4v*)(a.p.k + at) + lane;
            const u4v* vu = (const u4v*)(a.p.v + at) + lane;
            u4v kr[8], vr8[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) kr[k] = ku[64 * k];
#pragma unroll
            for (int k = 0; k < 8; ++k) vr8[k] = vu[64 * k];
            f4 S[2];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                S[tt] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < 4; ++k) S[tt] = mfma16x16x32(as_h8(kr[4 * tt + k]), as_h8(q[k]), S[tt]);
            }
            uint32_t bad = 0, ok = ~0u;
            if (unit < clean0 || unit >= clean1) {
                ok = col.mask(pos, su.L);
                const uint32_t mine = ok >> (8 * lq);
#pragma unroll
                for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        S[tt][r] = (mine >> (4 * tt + r)) & 1 ? S[tt][r] : -INFINITY;
                // which tokens hold an infinity or a NaN: lane (ln, lq) has tokens 8 lq + j of dims 16 dt + ln
                uint32_t my = 0;
#pragma unroll
                for (int k = 0; k < 8; ++k)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t y = vr8[k][j];
                        const bool h0 = (y & 0x7C00u) == 0x7C00u, h1 = (y & 0x7C000000u) == 0x7C000000u;
                        my |= (h0 ? 1u : 0u) << (2 * j) | (h1 ? 2u : 0u) << (2 * j);
                        vr8[k][j] = (h0 ? 0u : y & 0xFFFFu) | (h1 ? 0u : y & 0xFFFF0000u);
                    }
                if (__any(my != 0)) {
                    my <<= 8 * lq;
#pragma unroll
                    for (int o = 1; o < 64; o <<= 1) my |= __shfl_xor(my, o, MJ_WAVE);
                    bad = my;
                }
            }
            const u4v p = unit_weights(T, S);
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) T.o[dt] = mfma16x16x32(as_h8(vr8[dt]), as_h8(p), T.o[dt]);
            if (bad) add_bad(T, a.p.v + at, bad, ok);
        }
        // the four waves' states
        T.l = x4_sum(T.l);
        __syncthreads();  // (the segment before has been read)
        if (lq == 0) s_ml[w][ln] = make_float2(T.m, T.l);
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) *(f4*)&s_o[w][ln][16 * dt + 4 * lq] = T.o[dt];
        __syncthreads();
        const int cc = t >> 4, d0 = 8 * (t & 15);
        float M = -INFINITY, l = 0.0f, o[8] = {};
#pragma unroll
        for (int k = 0; k < 4; ++k) M = fmaxf(M, s_ml[k][cc].x);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 ml = s_ml[k][cc];
            const float f = ml.x == M ? 1.0f : __builtin_amdgcn_exp2f(ml.x - M);
            l = fmaf(f, ml.y, l);
#pragma unroll
            for (int d = 0; d < 8; ++d) o[d] = fmaf(f, s_o[k][cc][d0 + d], o[d]);
        }
        if (v0 + cc < nv) {
            if (i0 == 0 && i1 == su.nu) {
                const int r = (v0 + cc) / a.G, h = g * a.G + (v0 + cc) - r * a.G;
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (no key seen: zeros)
                u4v y;
#pragma unroll
                for (int d = 0; d < 4; ++d) y[d] = pack2(f2h(o[2 * d] * inv), f2h(o[2 * d + 1] * inv));
                *(u4v*)(a.out + (su.r0 + r) * a.ldo + h * HD + d0) = y;
            } else {
                const size_t slot = (size_t)blockIdx.x * 2 + (x == b0 ? 0 : 1);
                const size_t at = slot * a.cols + cc;
                if ((t & 15) == 0) a.pml[at] = make_float2(M, l);
                *(f4*)(a.po + at * HD + d0) = (f4){o[0], o[1], o[2], o[3]};
                *(f4*)(a.po + at * HD + d0 + 4) = (f4){o[4], o[5], o[6], o[7]};
            }
        }
        x += i1 - i0;
    }
}

// The partial results of one row and head, where its keys went to several blocks: eight groups of 32
// lanes take every eighth block, four dims a lane, and the groups meet in LDS.
__global__ __launch_bounds__(256) void k_paged_join(PgAttnArgs a) {
    __shared__ f4 s_o[8][32];
    __shared__ float2 s_ml[8];
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
    const int bA = (int)(S / per), bB = (int)((E - 1) / per);
    if (bA == bB) return;
    const int k = t >> 5, d = t & 31;
    float M = -INFINITY, l = 0.0f;
    f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int b = bA + k; b <= bB; b += 8) {
        const size_t at = ((size_t)b * 2 + (S <= b * per ? 0 : 1)) * a.cols + cc;
        const float2 ml = a.pml[at];
        const f4 y = *(const f4*)(a.po + at * HD + 4 * d);
        const float mn = fmaxf(M, ml.x);
        const float f0 = M == mn ? 1.0f : __builtin_amdgcn_exp2f(M - mn);
        const float f1 = ml.x == mn ? 1.0f : __builtin_amdgcn_exp2f(ml.x - mn);
        M = mn;
        l = l * f0 + ml.y * f1;
        o = o * f0 + y * f1;
    }
    if (d == 0) s_ml[k] = make_float2(M, l);
    s_o[k][d] = o;
    __syncthreads();
    if (t >= 32) return;
    M = -INFINITY;
    for (int i = 0; i < 8; ++i) M = fmaxf(M, s_ml[i].x);
    l = 0.0f;
    o = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < 8; ++i) {
        const float2 ml = s_ml[i];
        const float f = ml.x == M ? 1.0f : __builtin_amdgcn_exp2f(ml.x - M);
        l += ml.y * f;
        o += s_o[i][d] * f;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (no key seen: zeros)
    *(uint2*)(out + 4 * d) = make_uint2(pack2(f2h(o[0] * inv), f2h(o[1] * inv)),
                                        pack2(f2h(o[2] * inv), f2h(o[3] * inv)));
}

#define PG_BLOCKS 512  // two blocks a CU

size_t paged_attn_plan(PgAttnArgs& a, void* base) {
    a.cols = 16;
    a.blocks = PG_BLOCKS;
    Arena ar{base, 0};
    a.off = (int64_t*)ar.take((PG_MAX_SEQS + 2) * sizeof(int64_t));
    a.pml = (float2*)ar.take((size_t)a.blocks * 2 * a.cols * sizeof(float2));
    a.po = (float*)ar.take((size_t)a.blocks * 2 * a.cols * HD * sizeof(float));
    return ar.off;
}

hipError_t launch_paged_attn(const PgAttnArgs& a, hipStream_t st) {
    if (a.b.n_seqs > PG_MAX_SEQS || a.b.rows < 1 || a.b.max_rows > MJ_ROWS || a.p.page < PG_UNIT)
        return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_paged_attn, dim3(a.blocks), dim3(256), 0, st, a);
    hipLaunchKernelGGL(k_paged_join, dim3(a.b.rows, a.p.nKV * a.G), dim3(256), 0, st, a);
    return hipGetLastError();
}
