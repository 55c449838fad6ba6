// accept.hip -- the drafts of a batch of sequences checked against the target's probabilities, from given
// random numbers.
//
// p = softmax(logits / T) of a row.  A drafted token x below row r is accepted if u q(x) rest <= e(x),
// e = exp((logit - greatest) / T), rest the sum of e over the row less the drafts refused before (q: the
// draft's own probability, 1 where it is certain); the last row reached samples its token from what the
// refusals leave of p.  All in 64 bits: the sampled token is where a sum of V terms crosses a number, and
// V = 150000 terms off by fp32's 2^-24 each would move one sample in thirty to a neighbour.  (This chip's
// 64-bit fma runs at the rate of the unpacked 32-bit one, and the logits are read once: memory bounds it.)
//
// Three launches: sums and greatest logits of every row in chunks; a block a sequence for the walk over the
// drafts and the tokens that need no more than these sums; and, a block a chunk, what the draft's
// distribution or many refusals leave of the others' last rows, and their tokens.
#include "mj_abi_internal.h"
#include "mj_device.h"
#include "mj_paged.h"

#define AC_CHUNK 4096  // ids a block takes
#define AC_PER (AC_CHUNK / 256)
#define AC_GREEDY 1e-5f
// Refused drafts that the walk takes out of their chunks itself: a chunk gone through again takes its block 2 us,
// so that of more the third launch, all chunks at once, is not longer.
#define AC_FEW 2

// 2^(i / 32), 0 <= i < 32, in 64 bits, with i << 15 taken off the upper half: n << 15 added there gives 2^(n / 32)
// for any n = i in the lowest five bits (32 << 15 is one in the exponent).  12 terms of the series of exp(i ln 2 / 32 - ln 2 / 2) (the next is
// below 7e-15), times sqrt 2.
__device__ __forceinline__ double root32(int i) {
    const double r = (double)(i - 16) * 0.02166084939249829;
    double p = 1.0 / 39916800.0;
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    p *= 1.4142135623730951;
    return __hiloint2double(__double2hiint(p) - (i << 15), __double2loint(p));
}

// e of many logits of one row: (x - m) a = n + r, a = 32 log2(e) / T, |r| <= 1/2; 2^(n / 32) from a table and the
// exponent, 2^(r / 32) from a polynomial of degree 4 (its coefficients fitted to the least greatest error,
// 8e-14; the series' own would have 1.2e-12).  The difference d = x - m of two floats is exact at 0 and off by 2^-53
// of itself elsewhere, so e is 1 at m wherever the row lies (a x - a m, with a m rounded first, is off by 2^-53 a m:
// at logits of 1e15 and more by whole steps of n).  n comes out of the low bits of a d + 1.5 2^52, r out of a second
// fma with the same product.  The table is 256 bytes, each LDS bank once, so that lanes never wait for one another; of
// 64 entries and one term less they did.  Infinities share the row.
struct Weights {
    double a, least;  // a d = -32000 at `least`: what lies below has no weight
    float m;
    const double* tab;
    // k: 1 / T
    __device__ __forceinline__ Weights(double T, double k, float top, const double* t) : m(top), tab(t) {
        // (an infinite temperature: a is not 0, so that -inf stays below everything, and any finite a d is)
        a = fmax(k * 46.16624130844683, 1e-60);  // 32 log2(e)
        least = fmax(T * -693.1471805599453, -3.2e64);
    }
    __device__ __forceinline__ bool finite() const { return m < INFINITY; }
    // 2^(a d / 32) as a product
    __device__ __forceinline__ void factors(double d, double& p, double& root) const {
        const double t = fma(d, a, 6755399441055744.0), r = fma(d, a, 6755399441055744.0 - t);
        const int n = __double2loint(t);
        p = fma(r, 9.172541587776638e-09, 1.6938633817694331e-06);
        p = fma(p, r, 0.0002345961982133178);
        p = fma(p, r, 0.021660849391723976);
        p = fma(p, r, 1.0);
        root = tab[n & 31];
        root = __hiloint2double(__double2hiint(root) + (n << 15), __double2loint(root));
    }
    // 0 below 2^-1000, for -inf and for NaN
    __device__ __forceinline__ double operator()(float x) const {
        if (!finite()) return x == m ? 1.0 : 0.0;
        const double d = (double)x - (double)m;
        double p, root;
        factors(d, p, root);
        return d > least ? p * root : 0.0;
    }
    // sum + e, of a finite row's sum: what is 0 above counts as 2^-1000, which is lost in the sum (that has a 1)
    __device__ __forceinline__ double onto(double sum, float x) const {
        double p, root;
        factors(fmax((double)x - (double)m, least), p, root);
        return fma(p, root, sum);
    }
};

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, MJ_WAVE);
    return v;
}

// Four floats from any place.
typedef float __attribute__((ext_vector_type(4), aligned(4))) f4_any;

// Sum of e, greatest logit and its lowest place of AC_CHUNK ids of a row.  Bound by memory and by its
// operations in 64 bits alike: 324 rows of 151936 ids take 36 to 39 us, 33 at the rate of a streaming read, and
// the VALU is busy 73% of it (64 roots, the place carried beside the maximum and a load an id: 53 us).
__global__ __launch_bounds__(256) void k_accept_stats(AcceptArgs a) {
    __shared__ double s_tab[32], s_s[4];
    __shared__ float s_m[4];
    __shared__ int s_at, s_abort;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, r = blockIdx.y;
    // what leads to the row's temperature goes out before its logits: they come last, and nothing after them
    const int ab = abort_word(a.abort);
    const int end = lane < a.b.n_seqs ? a.b.start[lane + 1] : INT32_MAX;
    const float* x = a.logits + r * a.ld;
    const int v0 = blockIdx.x * AC_CHUNK;
    f4 y[AC_PER / 4];  // ids v0 + 1024 i + 4 t ..
    if (v0 + AC_CHUNK <= a.V) {
#pragma unroll
        for (int i = 0; i < AC_PER / 4; ++i) y[i] = *(const f4_any*)(x + v0 + 1024 * i + 4 * t);
    } else {
#pragma unroll
        for (int i = 0; i < AC_PER; ++i) {
            const int v = v0 + 1024 * (i >> 2) + 4 * t + (i & 3);
            y[i >> 2][i & 3] = v < a.V ? x[v] : -INFINITY;
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    int s = __popcll(__ballot(end <= r));
    if (s == 64) s = pg_seq(a.b, r);
    const float T = s < a.b.n_seqs ? a.temperature[s] : 0.0f;
    if (t == 0) {
        s_abort = ab;
        s_at = INT32_MAX;
    }
    if (t < 32) s_tab[t] = root32(t);
    float mine = -INFINITY;  // (fmaxf passes NaN over)
#pragma unroll
    for (int i = 0; i < AC_PER / 2; ++i) mine = fmaxf(fmaxf(mine, y[i >> 1][2 * (i & 1)]), y[i >> 1][2 * (i & 1) + 1]);
    const float most = wave_max(mine);
    if (lane == 0) s_m[w] = most;
    __syncthreads();
    if (s_abort || s >= a.b.n_seqs) return;
    const float m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    double sum = 0.0;
    if (m > -INFINITY) {
        if (mine == m) {
            int at = INT32_MAX;
#pragma unroll
            for (int i = AC_PER - 1; i >= 0; --i)
                if (y[i >> 2][i & 3] == m) at = v0 + 1024 * (i >> 2) + 4 * t + (i & 3);
            atomicMin(&s_at, at);
        }
        if (T > AC_GREEDY) {
            const Weights e(T, 1.0 / (double)T, m, s_tab);
            if (e.finite()) {
#pragma unroll
                for (int i = 0; i < AC_PER; ++i) sum = e.onto(sum, y[i >> 2][i & 3]);
            } else {
#pragma unroll
                for (int i = 0; i < AC_PER; ++i) sum += y[i >> 2][i & 3] == m ? 1.0 : 0.0;
            }
            sum = wave_sum64(sum);
            if (lane == 0) s_s[w] = sum;
        }
        __syncthreads();
        if (T > AC_GREEDY) sum = (s_s[0] + s_s[1]) + (s_s[2] + s_s[3]);
    }
    if (t == 0) a.part[(size_t)r * a.chunks + blockIdx.x] = AcceptPart{sum, m, s_at};
}

// How the token of the last row is sampled: from the row's probabilities, from these less the draft's, from
// these without the refused drafts.
enum { LAST_P = 0, LAST_RESIDUAL = 1, LAST_WITHOUT = 2 };

// Inclusive sum over a block of NT threads in a fixed order; *all: of every thread.
template <int NT>
__device__ __forceinline__ double block_scan64(double v, double* s_w, double* all) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double x = __shfl_up(v, o, MJ_WAVE);
        if (lane >= o) v += x;
    }
    __syncthreads();
    if (lane == 63) s_w[w] = v;
    __syncthreads();
    double before = 0.0, sum = 0.0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
        if (i == w) before = sum;
        sum += s_w[i];
    }
    *all = sum;
    return before + v;
}
// The first thread whose share, ending at `upto`, passes `want`; where none does (the parts' rounding), the
// last one that has any.  -1: nobody has.
template <int NT>
__device__ __forceinline__ int first_past(double share, double upto, double want, int* s_first, int* s_last) {
    const int w = threadIdx.x >> 6;
    const uint64_t past = __ballot(share > 0.0 && upto > want), any = __ballot(share > 0.0);
    if ((threadIdx.x & 63) == 0) {
        s_first[w] = past ? 64 * w + __builtin_ctzll(past) : INT32_MAX;
        s_last[w] = any ? 64 * w + 63 - __builtin_clzll(any) : -1;
    }
    __syncthreads();
    int first = INT32_MAX, last = -1;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
        first = min(first, s_first[i]);
        last = max(last, s_last[i]);
    }
    return first != INT32_MAX ? first : last;
}
__device__ __forceinline__ double of_lane(double v, int lane) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane),
                            __builtin_amdgcn_readlane(__double2loint(v), lane));
}


// LDS of a block that samples.
template <int NT>
struct LeftShared {
    double w[NT / 64], fix[AC_FEW], gone_e[MJ_ROWS], before;
    uint32_t gone[AC_CHUNK / 32];
    int out[MJ_ROWS];  // the refused drafts of the row
    int first[NT / 64], last[NT / 64], chunk, bad;
};
// What the walk left of a row's probabilities: methods are for a whole block.
template <int NT>
struct Left {
    static constexpr int PER = AC_CHUNK / NT;
    const float *lx, *lq;
    const AcceptPart* parts;
    double inv;
    Weights e;
    int V, chunks, mode, n_out;
    LeftShared<NT>& S;

    __device__ __forceinline__ void mark(int c) const {  // bits of the refused ids of a chunk
        const int t = threadIdx.x;
        if (mode != LAST_WITHOUT) return;
        if (t < AC_CHUNK / 32) S.gone[t] = 0;
        __syncthreads();
        if (t < n_out) {
            const int d = S.out[t] - c * AC_CHUNK;
            if ((unsigned)d < AC_CHUNK) atomicOr(&S.gone[d >> 5], 1u << (d & 31));
        }
        __syncthreads();
    }
    // of id d of a chunk, of logit x and draft's probability q
    __device__ __forceinline__ double weight(float x, float q, int d) const {
        double z = e(x);
        if (mode == LAST_RESIDUAL) z = fmax(fma(z, inv, -(double)fmaxf(q, 0.0f)), 0.0);  // (a NaN counts as 0)
        if (mode == LAST_WITHOUT && (S.gone[d >> 5] >> (d & 31)) & 1) z = 0.0;
        return z;
    }
    // of the thread's PER ids of chunk c
    __device__ __forceinline__ void own(int c, double* y) const {
        const int d = PER * threadIdx.x, v0 = c * AC_CHUNK + d;
        f4 x[PER / 4], q[PER / 4]{};
        if (c * AC_CHUNK + AC_CHUNK <= V) {
#pragma unroll
            for (int i = 0; i < PER / 4; ++i) x[i] = *(const f4_any*)(lx + v0 + 4 * i);
            if (mode == LAST_RESIDUAL)
#pragma unroll
                for (int i = 0; i < PER / 4; ++i) q[i] = *(const f4_any*)(lq + v0 + 4 * i);
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                x[i >> 2][i & 3] = v0 + i < V ? lx[v0 + i] : -INFINITY;
                if (mode == LAST_RESIDUAL) q[i >> 2][i & 3] = v0 + i < V ? lq[v0 + i] : 0.0f;
            }
        }
        mark(c);
#pragma unroll
        for (int i = 0; i < PER; ++i) y[i] = weight(x[i >> 2][i & 3], q[i >> 2][i & 3], d + i);
    }
    // of a chunk, in every thread
    __device__ __forceinline__ double chunk(int c) const {
        const int t = threadIdx.x;
        double y[PER], sum = 0.0;
        own(c, y);
#pragma unroll
        for (int i = 0; i < PER; ++i) sum += y[i];
        sum = wave_sum64(sum);
        if ((t & 63) == 0) S.w[t >> 6] = sum;
        __syncthreads();
        double all = 0.0;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) all += S.w[i];
        return all;
    }
    // The id where the sums pass u times all, -1 where nothing has any weight; in one thread, the others
    // get -2.  of_chunk(c): what chunk c has left; again(): the same in every thread, after all have asked for
    // their chunks: whether they have to ask once more.
    template <typename F, typename G>
    __device__ __forceinline__ int sample(double u, F of_chunk, G again) {
        const int t = threadIdx.x, per = (chunks + NT - 1) / NT;
        double all = 0.0, upto = 0.0, share = 0.0;
        bool plain = mode == LAST_P;
        auto has = [&](int c) __attribute__((always_inline)) {
            if (c >= chunks) return 0.0;
            if (!plain) return of_chunk(c);
            const AcceptPart p = parts[c];
            return p.s * e(p.m);
        };
        for (;;) {
            share = 0.0;
            for (int i = 0; i < per; ++i) share += has(per * t + i);
            upto = block_scan64<NT>(share, S.w, &all);
            if (!plain && again()) continue;
            if (all > 0.0 || plain) break;
            plain = true;  // nothing left: the row's own probabilities
            mode = LAST_P;
        }
        const double want = u * all;
        const int who = first_past<NT>(share, upto, want, S.first, S.last);
        if (who < 0) return t == 0 ? -1 : -2;
        if (t == who) {
            double at = upto - share;
            int c = t;
            S.before = at;
            if (per > 1)
                for (int i = 0; i < per; ++i) {
                    const double z = has(per * t + i);
                    if (!(z > 0.0)) continue;
                    c = per * t + i;
                    S.before = at;
                    at += z;
                    if (at > want) break;
                }
            S.chunk = c;
        }
        __syncthreads();
        // and the id in it
        const int c = S.chunk;
        const double rest = want - S.before;
        double y[PER];
        own(c, y);
        share = 0.0;
#pragma unroll
        for (int i = 0; i < PER; ++i) share += y[i];
        upto = block_scan64<NT>(share, S.w, &all);
        const int me = first_past<NT>(share, upto, rest, S.first, S.last);
        if (t != me) return me < 0 && t == 0 ? -1 : -2;
        double at = upto - share;
        int id = -1;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const bool past = at > rest && id >= 0;
            at += y[i];
            if (y[i] > 0.0 && !past) id = c * AC_CHUNK + PER * t + i;
        }
        return id;
    }
};

// The rows' totals and the walk over the drafts, a block a sequence; and the token, where it is the greatest
// logit's, or is sampled from the row's sums by chunks as they are or with a few drafts taken out.
// One block's steps one after another bound it, its instructions' own way to it among them: with 256 threads of
// 16 ids each, four times the instructions, a sequence took 14 us, so 11.5, and 9.7 where no chunk is gone
// through again.
#define AC_WALK 1024
__global__ __launch_bounds__(AC_WALK) void k_accept_walk(AcceptArgs a) {
    __shared__ double s_tab[32], s_Z[MJ_ROWS];
    __shared__ float s_m[MJ_ROWS];
    __shared__ int s_at[MJ_ROWS];
    __shared__ uint64_t s_refused;
    __shared__ int s_cur, s_any, s_abort;
    __shared__ LeftShared<AC_WALK> s_left;
    const int s = blockIdx.x, t = threadIdx.x;
    const int ab = abort_word(a.abort);
    int r0;
    const int n = pg_rows(a.b, s, r0);
    const float T = a.temperature[s], u_sample = a.u_sample[s];
    const bool greedy = !(T > AC_GREEDY);
    const double temp = greedy ? 1.0 : (double)T, k = 1.0 / temp;
    // drafts and their logits, on their way while the totals are formed
    int par = -1, tok = -1;
    float x = -INFINITY, q = 1.0f, u = 0.0f;
    if (t < n) {
        tok = a.tokens[r0 + t];
        u = a.u_accept[r0 + t];
        const uint64_t below = pg_anc(a.b, r0 + t, t) & ((1ull << t) - 1);
        par = below ? 63 - __clzll(below) : -1;
        if (par >= 0 && (unsigned)tok < (unsigned)a.V) {
            x = a.logits[(r0 + par) * a.ld + tok];
            if (a.q) q = a.q[(r0 + par) * a.ldq + tok];
        }
    }
    const int r = t >> 4;
    AcceptPart part[4];
    auto fetch = [&](int c0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) part[i] = a.part[(size_t)(r0 + r) * a.chunks + min(c0 + 16 * i, a.chunks - 1)];
    };
    if (r < n) fetch(t & 15);
    if (t < 32) s_tab[t] = root32(t);
    if (t == 0) {
        s_abort = ab;
        a.last[s].row = -1;  // (nothing for the third launch, also where the call was aborted)
        a.last[s].count = 0;
    }
    __syncthreads();
    if (s_abort) return;
    if (n <= 0) {
        if (t == 0) {
            a.accepted[s] = 0;
            a.token[s] = -1;
        }
        return;
    }
    // the rows' totals, a row each 16 lanes, four chunks a lane and turn
    if (r < n) {
        float m = -INFINITY;
        int at = INT32_MAX;
        double Z = 0.0;
        for (int c0 = t & 15; c0 < a.chunks; c0 += 64) {
            if (c0 >= 64) fetch(c0);
            const float before = m;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c0 + 16 * i < a.chunks && part[i].m > m) {
                    m = part[i].m;
                    at = part[i].at;
                }
            const Weights e(temp, k, m, s_tab);
            Z *= e(before);
#pragma unroll
            for (int i = 0; i < 4; ++i) Z += c0 + 16 * i < a.chunks ? part[i].s * e(part[i].m) : 0.0;
        }
        const float mine = m;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
            const float om = __shfl_xor(m, o, 16);
            const int oa = __shfl_xor(at, o, 16);
            if (om > m || (om == m && oa < at)) {
                m = om;
                at = oa;
            }
        }
        Z *= Weights(temp, k, m, s_tab)(mine);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) Z += __shfl_xor(Z, o, 16);
        if ((t & 15) == 0) {
            s_m[r] = m;
            s_at[r] = at;
            s_Z[r] = greedy ? (m > -INFINITY ? 1.0 : 0.0) : Z;
        }
    }
    __syncthreads();
    // the walk: a draft a lane of the first wave, its numbers fetched from lane to lane
    if (t < 64) {
        double e = 0.0;
        if (par >= 0 && (unsigned)tok < (unsigned)a.V && s_Z[par] > 0.0)
            e = greedy ? (tok == s_at[par] ? 1.0 : 0.0) : Weights(temp, k, s_m[par], s_tab)(x);
        const double uq = (double)u * (double)q;
        const uint64_t can = __ballot(q > 0.0f);
        int cur = 0, acc = 0, way = t == 0 ? 0 : -1;
        uint64_t refused = 0, kids = __ballot(par == 0);
        double rest = s_Z[0], gone = 0.0;
        while (kids) {
            const int r = __builtin_ctzll(kids);
            const double er = of_lane(e, r);
            if (er > 0.0 && (can >> r & 1) && of_lane(uq, r) * rest <= er) {
                cur = r;
                rest = s_Z[r];
                refused = 0;
                ++acc;
                if (t == acc) way = r;
                kids = __ballot(par == r);
            } else {
                refused |= 1ull << r;
                rest -= er;
                if (t == r) gone = er;
                // (an equal sibling after it has nothing left)
                if (par == cur && tok == __builtin_amdgcn_readlane(tok, r)) e = 0.0;
                kids &= kids - 1;
            }
        }
        const uint64_t out = refused & __ballot((unsigned)tok < (unsigned)a.V);  // (others have nothing to leave out)
        if (out >> t & 1) {
            const int at = __popcll(out & ((1ull << t) - 1));
            s_left.out[at] = tok;
            s_left.gone_e[at] = gone;
        }
        if (t < n) a.path[r0 + t] = way;
        if (t == 0) {
            s_cur = cur;
            s_left.bad = rest < s_Z[cur] * 0x1p-10;
            s_refused = out;
            s_any = refused != 0;
            a.accepted[s] = acc;
            if (greedy || !(s_Z[cur] > 0.0)) a.token[s] = s_Z[cur] > 0.0 ? s_at[cur] : -1;
        }
    }
    __syncthreads();
    const int cur = s_cur, row = r0 + cur;
    const uint64_t refused = s_refused;
    const int n_out = (int)__popcll(refused);
    const double Z = s_Z[cur];
    if (greedy || !(Z > 0.0)) return;
    const int mode = a.q && s_any ? LAST_RESIDUAL : n_out ? LAST_WITHOUT : LAST_P;
    if (mode == LAST_RESIDUAL || n_out > AC_FEW) {
        if (t == 0) {
            a.last[s].refused = refused;
            a.last[s].Z = Z;
            a.last[s].m = s_m[cur];
            a.last[s].first = r0;
            a.last[s].row = row;
        }
        return;
    }
    Left<AC_WALK> left{a.logits + row * a.ld, nullptr, a.part + (size_t)row * a.chunks, 0.0,
              Weights(temp, k, s_m[cur], s_tab), a.V, a.chunks, mode, n_out, s_left};
    // The drafts' weights are known and taken off their chunks' sums, which have an error of 2^-53 of
    // themselves; where that is not small against what is left, the chunks are gone through again.
    bool exact = false;
    const int id = left.sample(
        (double)u_sample,
        [&](int c) __attribute__((always_inline)) {
            const AcceptPart p = left.parts[c];
            const double z = p.s * left.e(p.m);
            double less = 0.0;
            for (int i = 0; i < n_out; ++i)
                if (s_left.out[i] / AC_CHUNK == c) {
                    if (exact) return s_left.fix[i];
                    less += s_left.gone_e[i];
                }
            if (less > 0.0 && z - less < z * 0x1p-20) s_left.bad = 1;
            return z - less;
        },
        [&]() __attribute__((always_inline)) {
            __syncthreads();
            if (exact || !s_left.bad) return false;
            exact = true;
            for (int i = 0; i < n_out; ++i) {
                const double z = left.chunk(s_left.out[i] / AC_CHUNK);
                if (t == 0) s_left.fix[i] = z;
                __syncthreads();
            }
            return true;
        });
    if (id > -2) a.token[s] = id;
}

// What is left of the other sequences' last rows, a block a chunk; the block that comes last samples.  Bound
// by its operations and a block's few steps one after another (48 rows of 151936 ids with distributions, 58 MB, 20
// us, VALU 64% busy; by 1024 threads of four ids, one block a CU, 43, by 256 of 16 30).
#define AC_LEFT 512
__global__ __launch_bounds__(AC_LEFT) void k_accept_left(AcceptArgs a) {
    __shared__ double s_tab[32];
    __shared__ LeftShared<AC_LEFT> s_left;
    __shared__ int s_last, s_abort;
    const int s = blockIdx.y, c = blockIdx.x, t = threadIdx.x;
    const AcceptLast last = a.last[s];
    if (last.row < 0) return;
    const int ab = abort_word(a.abort);
    const float T = a.temperature[s], u_sample = a.u_sample[s];
    if (t < 32) s_tab[t] = root32(t);
    if (t == 0) s_abort = ab;
    if (t < 64 && last.refused >> t & 1)
        s_left.out[__popcll(last.refused & ((1ull << t) - 1))] = a.tokens[last.first + t];
    __syncthreads();
    if (s_abort) return;
    Left<AC_LEFT> left{a.logits + last.row * a.ld,
              a.q ? a.q + last.row * a.ldq : nullptr,
              a.part + (size_t)last.row * a.chunks,
              1.0 / last.Z,
              Weights(T, 1.0 / (double)T, last.m, s_tab),
              a.V,
              a.chunks,
              a.q ? LAST_RESIDUAL : LAST_WITHOUT,
              (int)__popcll(last.refused),
              s_left};
    double* sums = a.csum + (size_t)s * a.chunks;
    const double z = left.chunk(c);
    if (t == 0) {
        // stored past this XCD's cache, and there before the block counts itself
        __hip_atomic_store(sums + c, z, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        s_last = __hip_atomic_fetch_add(&a.last[s].count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                 (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!s_last) return;
    const int id = left.sample(
        (double)u_sample,
        [&](int i) __attribute__((always_inline)) {
            return __hip_atomic_load(sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        },
        []() { return false; });
    if (id > -2) a.token[s] = id;
}

size_t accept_rows_layout(AcceptArgs& a, void* base) {
    a.chunks = (a.V + AC_CHUNK - 1) / AC_CHUNK;
    Arena ar{base, 0};
    a.part = (AcceptPart*)ar.take((size_t)a.b.rows * a.chunks * sizeof(AcceptPart));
    a.csum = (double*)ar.take((size_t)a.b.n_seqs * a.chunks * sizeof(double));
    a.last = (AcceptLast*)ar.take((size_t)a.b.n_seqs * sizeof(AcceptLast));
    return ar.off;
}

hipError_t launch_accept_rows(const AcceptArgs& a, hipStream_t st) {
    if (a.b.rows < 0 || a.b.rows > 65535 || a.b.n_seqs > 65535 || a.b.max_rows > MJ_ROWS || a.V < 1)
        return hipErrorInvalidValue;
    if (a.b.rows > 0)
        hipLaunchKernelGGL(k_accept_stats, dim3(a.chunks, a.b.rows), dim3(256), 0, st, a);
    hipLaunchKernelGGL(k_accept_walk, dim3(a.b.n_seqs), dim3(AC_WALK), 0, st, a);
    // (a row of a chain has one draft below it, of a tree at most all the others)
    if (a.q || (a.b.anc && a.b.max_rows - 1 > AC_FEW))
        hipLaunchKernelGGL(k_accept_left, dim3(a.chunks, a.b.n_seqs), dim3(AC_LEFT), 0, st, a);
    return hipGetLastError();
}
