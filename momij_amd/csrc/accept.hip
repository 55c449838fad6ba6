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
// Two launches: sums and greatest logits of every row in chunks; then, a block for each chunk and
// sequence, the walk over the drafts (every block of a sequence for itself: it costs them a few rounds of
// requests, as a launch would), its chunk's share of what is left, and in the block that comes last the
// token.
#include "mj_abi_internal.h"
#include "mj_device.h"
#include "mj_paged.h"

#define AC_CHUNK 4096  // ids a block takes
#define AC_PER (AC_CHUNK / 256)
#define AC_GREEDY 1e-5f

// 2^(i / 64), 0 <= i < 64, in 64 bits: 12 terms of the series of exp(i ln 2 / 64 - ln 2 / 2) (the next is
// below 7e-15), times sqrt 2.
__device__ __forceinline__ double root64(int i) {
    const double r = (double)(i - 32) * 0.010830424696249145;
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
    return p * 1.4142135623730951;
}

// e of many logits of one row: y = (x - m) 64 log2(e) / T = n + r, |r| <= 1/2; 2^(n / 64) from a table and the
// exponent, 2^(r / 64) from five terms (the next is below 4e-14).  n comes out of the low bits of y +
// 1.5 2^52.  Eleven operations in 64 bits; the series alone takes 18 and conversions.  0 below 2^-1000, for
// -inf and for NaN; infinities share the row.
struct Weights {
    double a, c;  // y = a x + c
    float m;
    const double* tab;
    __device__ __forceinline__ Weights(double k, float top, const double* t) : m(top), tab(t) {
        a = k * 92.33248261689366;  // 64 log2(e)
        c = top < INFINITY ? -a * (double)top : 0.0;
    }
    __device__ __forceinline__ double operator()(float x) const {
        if (!(m < INFINITY)) return x == m ? 1.0 : 0.0;
        const double y = fma((double)x, a, c), t = y + 6755399441055744.0;
        const double r = y - (t - 6755399441055744.0);
        const int n = __double2loint(t);
        double p = fma(r, 5.732851688640402e-10, 2.1173137155464776e-07);
        p = fma(p, r, 5.86490495505617e-05);
        p = fma(p, r, 0.010830424696249145);
        p = fma(p, r, 1.0) * tab[n & 63];
        p = __hiloint2double(__double2hiint(p) + ((n >> 6) << 20), __double2loint(p));
        return y > -64000.0 ? p : 0.0;
    }
};

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, MJ_WAVE);
    return v;
}

// What a row's logits count as: a NaN as the least.
__device__ __forceinline__ float logit(float x) { return x == x ? x : -INFINITY; }

// Sum of e, greatest logit and its lowest place of AC_CHUNK ids of a row.
__global__ __launch_bounds__(256) void k_accept_stats(AcceptArgs a) {
    __shared__ double s_tab[64];
    __shared__ float s_m[4];
    __shared__ int s_at[4];
    __shared__ double s_s[4];
    if (block_aborted(a.abort)) return;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, r = blockIdx.y;
    const float* x = a.logits + r * a.ld;
    const int v0 = blockIdx.x * AC_CHUNK;
    float y[AC_PER], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < AC_PER; ++i) {
        const int v = v0 + 256 * i + t;
        y[i] = x[v < a.V ? v : a.V - 1];
    }
    if (t < 64) s_tab[t] = root64(t);
    if (blockIdx.x == 0 && r == 0)  // (the second launch counts its blocks here)
        for (int i = t; i < a.b.n_seqs; i += 256) a.count[i] = 0;
    const int s = pg_seq(a.b, r);
    if (s >= a.b.n_seqs) return;
    const float T = a.temperature[s];
    int at = INT32_MAX;
#pragma unroll
    for (int i = 0; i < AC_PER; ++i) {
        const int v = v0 + 256 * i + t;
        y[i] = v < a.V ? logit(y[i]) : -INFINITY;
        if (y[i] > m) {
            m = y[i];
            at = v;
        }
    }
    wave_argmax(m, at);
    if (lane == 0) {
        s_m[w] = m;
        s_at[w] = at;
    }
    __syncthreads();
    m = s_m[0];
    at = s_at[0];
#pragma unroll
    for (int i = 1; i < 4; ++i)
        if (s_m[i] > m || (s_m[i] == m && s_at[i] < at)) {
            m = s_m[i];
            at = s_at[i];
        }
    double sum = 0.0;
    if (T > AC_GREEDY && m > -INFINITY) {
        const Weights e(1.0 / (double)T, m, s_tab);
#pragma unroll
        for (int i = 0; i < AC_PER; ++i) sum += e(y[i]);
        sum = wave_sum64(sum);
        if (lane == 0) s_s[w] = sum;
        __syncthreads();
        sum = (s_s[0] + s_s[1]) + (s_s[2] + s_s[3]);
    }
    if (t == 0) a.part[(size_t)r * a.chunks + blockIdx.x] = AcceptPart{sum, m, at};
}

// How the token of the last row is sampled: from the row's probabilities, from these less the draft's, from
// these without the refused drafts.
enum { LAST_P = 0, LAST_RESIDUAL = 1, LAST_WITHOUT = 2 };

// Inclusive sum over the block in a fixed order; *all: of every thread.
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
    double before = 0.0;
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (i < w) before += s_w[i];
    *all = ((s_w[0] + s_w[1]) + s_w[2]) + s_w[3];
    return before + v;
}
// The first thread whose share, ending at `upto`, passes `want`; where none does (the parts' rounding), the
// last one that has any.  -1: nobody has.
__device__ __forceinline__ int first_past(double share, double upto, double want, int* s_i) {
    if (threadIdx.x == 0) {
        s_i[0] = INT32_MAX;
        s_i[1] = -1;
    }
    __syncthreads();
    if (share > 0.0) {
        if (upto > want) atomicMin(&s_i[0], (int)threadIdx.x);
        atomicMax(&s_i[1], (int)threadIdx.x);
    }
    __syncthreads();
    return s_i[0] != INT32_MAX ? s_i[0] : s_i[1];
}

__global__ __launch_bounds__(256) void k_accept_walk(AcceptArgs a) {
    __shared__ double s_tab[64], s_Z[MJ_ROWS], s_e[MJ_ROWS], s_w[4];
    __shared__ float s_m[MJ_ROWS], s_q[MJ_ROWS], s_u[MJ_ROWS], s_x[MJ_ROWS];
    __shared__ int s_at[MJ_ROWS], s_par[MJ_ROWS], s_tok[MJ_ROWS], s_out[MJ_ROWS];
    __shared__ uint32_t s_gone[AC_CHUNK / 32];
    __shared__ int s_cur, s_n_out, s_i[2], s_last;
    __shared__ double s_d[2];
    if (block_aborted(a.abort)) return;
    const int s = blockIdx.y, t = threadIdx.x, lane = t & 63;
    const bool lead = blockIdx.x == 0;
    int r0;
    const int n = pg_rows(a.b, s, r0);
    if (n <= 0) {
        if (lead && t == 0) {
            a.accepted[s] = 0;
            a.token[s] = -1;
        }
        return;
    }
    const float T = a.temperature[s];
    const bool greedy = !(T > AC_GREEDY);
    const double k = greedy ? 1.0 : 1.0 / (double)T;
    if (t < 64) s_tab[t] = root64(t);
    // drafts and their logits, on their way while the totals are formed
    int par = -1, tok = -1;
    float x = -INFINITY, q = 1.0f;
    if (t < n) {
        tok = a.tokens[r0 + t];
        s_u[t] = a.u_accept[r0 + t];
        const uint64_t below = pg_anc(a.b, r0 + t, t) & ((1ull << t) - 1);
        par = below ? 63 - __clzll(below) : -1;
        if (par >= 0 && (unsigned)tok < (unsigned)a.V) {
            x = a.logits[(r0 + par) * a.ld + tok];
            if (a.q) q = a.q[(r0 + par) * a.ldq + tok];
        }
    }
    __syncthreads();
    // the rows' totals, a row each 16 lanes
    for (int r = t >> 4; r < n; r += 16) {
        const AcceptPart* p = a.part + (size_t)(r0 + r) * a.chunks;
        float m = -INFINITY;
        int at = INT32_MAX;
        for (int c = t & 15; c < a.chunks; c += 16) {
            const AcceptPart y = p[c];
            if (y.m > m) {
                m = y.m;
                at = y.at;
            }
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
            const float om = __shfl_xor(m, o, 16);
            const int oa = __shfl_xor(at, o, 16);
            if (om > m || (om == m && oa < at)) {
                m = om;
                at = oa;
            }
        }
        double Z = 0.0;
        if (m > -INFINITY) {
            const Weights e(k, m, s_tab);
            for (int c = t & 15; c < a.chunks; c += 16) {
                const AcceptPart y = p[c];
                if (y.m > -INFINITY) Z += y.s * e(y.m);
            }
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) Z += __shfl_xor(Z, o, 16);
        if ((t & 15) == 0) {
            s_m[r] = m;
            s_at[r] = at;
            s_Z[r] = greedy ? (m > -INFINITY ? 1.0 : 0.0) : Z;
        }
    }
    if (t < n) {
        s_tok[t] = tok;
        s_par[t] = par;
        s_q[t] = q;
    }
    __syncthreads();
    if (t < n) {
        double e = 0.0;
        if (par >= 0 && (unsigned)tok < (unsigned)a.V && s_Z[par] > 0.0) {
            e = greedy ? (tok == s_at[par] ? 1.0 : 0.0) : Weights(k, s_m[par], s_tab)(logit(x));
            // (the second of two equal siblings has nothing left)
            for (int i = par + 1; i < t; ++i)
                if (s_par[i] == par && s_tok[i] == tok) e = 0.0;
        }
        s_e[t] = e;
    }
    __syncthreads();
    if (t == 0) {
        int cur = 0, acc = 0, out = 0;
        double rest = s_Z[0];
        if (lead) a.path[r0] = 0;
        for (int r = 1; r < n; ++r) {
            if (s_par[r] != cur) continue;
            const double e = s_e[r];
            if (e > 0.0 && s_q[r] > 0.0f && (double)s_u[r] * (double)s_q[r] * rest <= e) {
                cur = r;
                rest = s_Z[r];
                out = 0;
                ++acc;
                if (lead) a.path[r0 + acc] = r;
            } else {
                s_out[out++] = s_tok[r];
                rest -= e;
            }
        }
        s_cur = cur;
        s_n_out = out;
        if (lead) {
            for (int i = acc + 1; i < n; ++i) a.path[r0 + i] = -1;
            a.accepted[s] = acc;
            if (greedy || !(s_Z[cur] > 0.0)) a.token[s] = s_Z[cur] > 0.0 ? s_at[cur] : -1;
        }
    }
    __syncthreads();
    const int cur = s_cur, row = r0 + cur, n_out = s_n_out;
    const double Z = s_Z[cur];
    if (greedy || !(Z > 0.0)) return;
    // what is left of this block's ids
    int mode = n_out == 0 ? LAST_P : a.q ? LAST_RESIDUAL : LAST_WITHOUT;
    const Weights e(k, s_m[cur], s_tab);
    const float* lx = a.logits + row * a.ld;
    const float* lq = a.q + row * a.ldq;
    const double inv = 1.0 / Z;
    auto mark = [&](int v0) {  // bits of the refused ids of a chunk
        if (t < AC_CHUNK / 32) s_gone[t] = 0;
        __syncthreads();
        if (t < n_out) {
            const int v = s_out[t] - v0;
            if ((unsigned)v < AC_CHUNK) atomicOr(&s_gone[v >> 5], 1u << (v & 31));
        }
        __syncthreads();
    };
    // of ids v0 + step i + first (step 256: side by side; step 1: in a row)
    auto left = [&](int v0, int first, int step, double* y) {
        float lo[AC_PER], qo[AC_PER];
#pragma unroll
        for (int i = 0; i < AC_PER; ++i) {
            const int v = min(v0 + first + step * i, a.V - 1);
            lo[i] = lx[v];
            if (mode == LAST_RESIDUAL) qo[i] = lq[v];
        }
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < AC_PER; ++i) {
            const int d = first + step * i;
            double z = v0 + d < a.V ? e(logit(lo[i])) : 0.0;
            if (mode == LAST_RESIDUAL) z = fmax(z * inv - (qo[i] > 0.0f ? (double)qo[i] : 0.0), 0.0);
            if (mode == LAST_WITHOUT && (s_gone[d >> 5] >> (d & 31)) & 1) z = 0.0;
            if (mode == LAST_RESIDUAL && v0 + d >= a.V) z = 0.0;
            y[i] = z;
            sum += z;
        }
        return sum;
    };
    const int v0 = blockIdx.x * AC_CHUNK;
    double y[AC_PER];
    if (mode == LAST_WITHOUT) mark(v0);
    double sum = wave_sum64(left(v0, t, 256, y));
    if (lane == 0) s_w[t >> 6] = sum;
    __syncthreads();
    if (t == 0) {
        // stored past this XCD's cache, and there before the block counts itself
        double* c = a.csum + (size_t)s * a.chunks + blockIdx.x;
        __hip_atomic_store(c, (s_w[0] + s_w[1]) + (s_w[2] + s_w[3]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        s_last = __hip_atomic_fetch_add(&a.count[s], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                 (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!s_last) return;
    // the chunk where the sums pass u times all
    const double* sums = a.csum + (size_t)s * a.chunks;
    const int per = (a.chunks + 255) / 256;
    auto chunk_sum = [&](int c, bool plain) {
        if (c >= a.chunks) return 0.0;
        if (!plain) return __hip_atomic_load(sums + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const AcceptPart p = a.part[(size_t)row * a.chunks + c];
        return p.m > -INFINITY ? p.s * e(p.m) : 0.0;
    };
    double all = 0.0, upto = 0.0, share = 0.0;
    bool plain = false;
    for (int pass = 0; pass < 2; ++pass) {
        share = 0.0;
        for (int i = 0; i < per; ++i) share += chunk_sum(per * t + i, plain);
        upto = block_scan64(share, s_w, &all);
        if (all > 0.0 || mode == LAST_P) break;
        plain = true;  // nothing left: the row's own probabilities
        mode = LAST_P;
    }
    const double want = (double)a.u_sample[s] * all;
    const int who = first_past(share, upto, want, s_i);
    if (who < 0) {
        if (t == 0) a.token[s] = -1;
        return;
    }
    if (t == who) {
        double at = upto - share;
        int c = -1;
        for (int i = 0; i < per; ++i) {
            const double z = chunk_sum(per * t + i, plain);
            if (!(z > 0.0)) continue;
            c = per * t + i;
            s_d[0] = at;
            at += z;
            if (at > want) break;
        }
        s_last = c;
    }
    __syncthreads();
    // and the id in it, 16 in a row a thread
    const int p0 = s_last * AC_CHUNK;
    const double rest = want - s_d[0];
    if (mode == LAST_WITHOUT) mark(p0);
    share = left(p0, AC_PER * t, 1, y);
    upto = block_scan64(share, s_w, &all);
    const int me = first_past(share, upto, rest, s_i);
    if (t == me) {
        double at = upto - share;
        int id = -1;
#pragma unroll
        for (int i = 0; i < AC_PER; ++i) {
            const bool past = at > rest && id >= 0;
            at += y[i];
            if (y[i] > 0.0 && !past) id = p0 + AC_PER * t + i;
        }
        a.token[s] = id;
    }
}

size_t accept_rows_layout(AcceptArgs& a, void* base) {
    a.chunks = (a.V + AC_CHUNK - 1) / AC_CHUNK;
    Arena ar{base, 0};
    a.part = (AcceptPart*)ar.take((size_t)a.b.rows * a.chunks * sizeof(AcceptPart));
    a.csum = (double*)ar.take((size_t)a.b.n_seqs * a.chunks * sizeof(double));
    a.count = (int32_t*)ar.take((size_t)a.b.n_seqs * sizeof(int32_t));
    return ar.off;
}

hipError_t launch_accept_rows(const AcceptArgs& a, hipStream_t st) {
    if (a.b.rows < 0 || a.b.rows > 65535 || a.b.n_seqs > 65535 || a.b.max_rows > MJ_ROWS || a.V < 1)
        return hipErrorInvalidValue;
    if (a.b.rows > 0)
        hipLaunchKernelGGL(k_accept_stats, dim3(a.chunks, a.b.rows), dim3(256), 0, st, a);
    hipLaunchKernelGGL(k_accept_walk, dim3(a.chunks, a.b.n_seqs), dim3(256), 0, st, a);
    return hipGetLastError();
}
