// accept.hip -- the drafts of a batch of sequences checked against the target's probabilities, from given
// random numbers.
//
// p = softmax(logits / T) of a row.  A drafted token x below row r is accepted if u q(x) rest <= e(x),
// e = exp((logit - greatest) / T), rest the sum of e over the row less the drafts refused before (q: the
// draft's own probability, 1 where it is certain); the last row reached samples its token from what the
// refusals leave of p.  All in 64 bits: the sampled token is where a sum of V terms crosses a number, and
// V = 150000 terms off by fp32's 2^-24 each would move one sample in thirty to a neighbour.  (This chip's
// 64-bit fma runs at the rate of the unpacked 32-bit one, and the logits are read once: memory bounds it.)
#include "mj_abi_internal.h"
#include "mj_device.h"
#include "mj_paged.h"

#define AC_CHUNK 8192  // ids a block takes
#define AC_GREEDY 1e-5f

// exp(x) of x <= 0 in 64 bits: x = n ln 2 + r, |r| <= 0.35, and 11 terms of the series (r^12 / 12! is
// below 7e-15); 0 below -708 (and for NaN).
__device__ __forceinline__ double exp64(double x) {
    const double n = rint(x * 1.4426950408889634);
    double r = fma(-n, 0.69314718055994531, x);  // ln 2 in 64 bits, and what it lacks
    r = fma(-n, 2.3190468138462996e-17, r);
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
    return x >= -708.0 ? ldexp(p, (int)n) : 0.0;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, MJ_WAVE);
    return v;
}

// What a row's logits count as: a NaN as the least; an infinity shares the row with the others.
__device__ __forceinline__ float logit(float x) { return x == x ? x : -INFINITY; }
__device__ __forceinline__ double weight(float x, float m, double k) {  // k = 1 / T
    if (x == m) return m > -INFINITY ? 1.0 : 0.0;
    return exp64(((double)x - (double)m) * k);
}

// Sum of exp, greatest logit and its lowest place of AC_CHUNK ids of a row.
__global__ __launch_bounds__(256) void k_accept_stats(AcceptArgs a) {
    __shared__ float s_m[4];
    __shared__ int s_at[4];
    __shared__ double s_s[4];
    if (block_aborted(a.abort)) return;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, r = blockIdx.y, s = pg_seq(a.b, r);
    if (s >= a.b.n_seqs) return;
    const float T = a.temperature[s];
    const float* x = a.logits + r * a.ld;
    const int v0 = blockIdx.x * AC_CHUNK;
    float y[32], m = -INFINITY;
    int at = INT32_MAX;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const int v = v0 + 256 * i + t;
        y[i] = v < a.V ? logit(x[v]) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 32; ++i)
        if (y[i] > m) {
            m = y[i];
            at = v0 + 256 * i + t;
        }
    wave_argmax(m, at);
    if (lane == 0) {
        s_m[w] = m;
        s_at[w] = at;
    }
    __syncthreads();
    m = s_m[0];
    at = s_at[0];
    for (int i = 1; i < 4; ++i)
        if (s_m[i] > m || (s_m[i] == m && s_at[i] < at)) {
            m = s_m[i];
            at = s_at[i];
        }
    double sum = 0.0;
    if (T > AC_GREEDY) {
        const double k = 1.0 / (double)T;
#pragma unroll
        for (int i = 0; i < 32; ++i) sum += weight(y[i], m, k);
        sum = wave_sum64(sum);
        if (lane == 0) s_s[w] = sum;
        __syncthreads();
        sum = (s_s[0] + s_s[1]) + (s_s[2] + s_s[3]);
    }
    if (t == 0) a.part[(size_t)r * a.chunks + blockIdx.x] = AcceptPart{sum, m, at};
}

enum { LAST_P = 0, LAST_RESIDUAL = 1, LAST_WITHOUT = 2, LAST_TOKEN = 3 };

// One block a sequence: the rows' totals, every draft's weight under its parent, and the walk.
__global__ __launch_bounds__(256) void k_accept_walk(AcceptArgs a) {
    __shared__ double s_Z[MJ_ROWS], s_e[MJ_ROWS];
    __shared__ float s_m[MJ_ROWS], s_q[MJ_ROWS], s_u[MJ_ROWS];
    __shared__ int s_at[MJ_ROWS], s_par[MJ_ROWS], s_tok[MJ_ROWS];
    if (block_aborted(a.abort)) return;
    const int s = blockIdx.x, t = threadIdx.x, lane = t & 63, w = t >> 6;
    int r0;
    const int n = pg_rows(a.b, s, r0);
    if (n <= 0) {
        if (t == 0) {
            a.last[s] = AcceptLast{0.0, 0.0f, -1, LAST_TOKEN, 0};
            a.accepted[s] = 0;
            a.token[s] = -1;
        }
        return;
    }
    const float T = a.temperature[s];
    const bool greedy = !(T > AC_GREEDY);
    const double k = greedy ? 1.0 : 1.0 / (double)T;
    for (int r = w; r < n; r += 4) {
        float m = -INFINITY;
        int at = INT32_MAX;
        double Z = 0.0;
        for (int c0 = 0; c0 < a.chunks; c0 += 64) {
            const int c = c0 + lane;
            AcceptPart p{0.0, -INFINITY, INT32_MAX};
            if (c < a.chunks) p = a.part[(size_t)(r0 + r) * a.chunks + c];
            float cm = p.m;
            int ca = p.at;
            wave_argmax(cm, ca);
            const double z = wave_sum64(p.m > -INFINITY ? p.s * weight(p.m, cm, k) : 0.0);
            if (cm > m) {
                Z = Z * weight(m, cm, k) + z;
                m = cm;
                at = ca;
            } else {
                Z += z * weight(cm, m, k);
            }
        }
        if (lane == 0) {
            s_m[r] = m;
            s_at[r] = at;
            s_Z[r] = greedy ? (m > -INFINITY ? 1.0 : 0.0) : Z;
        }
    }
    if (t < n) {
        s_tok[t] = a.tokens[r0 + t];
        s_u[t] = a.u_accept[r0 + t];
        const uint64_t below = pg_anc(a.b, r0 + t, t) & ((1ull << t) - 1);
        s_par[t] = below ? 63 - __clzll(below) : -1;
    }
    __syncthreads();
    if (t < n) {
        const int par = s_par[t], tok = s_tok[t];
        double e = 0.0;
        float q = 1.0f;
        if (par >= 0 && (unsigned)tok < (unsigned)a.V) {
            const float x = logit(a.logits[(r0 + par) * a.ld + tok]);
            e = greedy ? (tok == s_at[par] && s_Z[par] > 0.0 ? 1.0 : 0.0) : weight(x, s_m[par], k);
            if (a.q) q = a.q[(r0 + par) * a.ldq + tok];
            // (the second of two equal siblings has nothing left)
            for (int i = par + 1; i < t; ++i)
                if (s_par[i] == par && s_tok[i] == tok) e = 0.0;
        }
        s_e[t] = e;
        s_q[t] = q;
    }
    __syncthreads();
    if (t != 0) return;
    int cur = 0, acc = 0, out = 0;
    double rest = s_Z[0];
    a.path[r0] = 0;
    for (int r = 1; r < n; ++r) {
        if (s_par[r] != cur) continue;
        const double e = s_e[r];
        if (e > 0.0 && s_q[r] > 0.0f && (double)s_u[r] * (double)s_q[r] * rest <= e) {
            cur = r;
            rest = s_Z[r];
            out = 0;
            a.path[r0 + ++acc] = r;
        } else {
            a.out_ids[s * MJ_ROWS + out++] = s_tok[r];
            rest -= e;
        }
    }
    for (int i = acc + 1; i < n; ++i) a.path[r0 + i] = -1;
    a.accepted[s] = acc;
    const bool none = !(s_Z[cur] > 0.0);
    if (none || greedy) a.token[s] = none ? -1 : s_at[cur];
    a.last[s] = AcceptLast{s_Z[cur], s_m[cur], none || greedy ? -1 : r0 + cur,
                           out == 0 ? LAST_P : a.q ? LAST_RESIDUAL : LAST_WITHOUT, out};
}

// Of the row that a sequence samples: what is left of id v's probability, times Z or not, whichever
// the mode's sums are of.
struct Left {
    const float *x, *q;
    float m;
    double k, inv;  // 1 / T, 1 / Z
    int mode;
    const uint32_t* gone;  // LAST_WITHOUT: bits of the chunk's refused ids
    int v0;
    __device__ __forceinline__ double of(int v) const {
        const double e = weight(logit(x[v]), m, k);
        if (mode == LAST_RESIDUAL) {
            const float y = q[v];
            return fmax(e * inv - (y > 0.0f ? (double)y : 0.0), 0.0);
        }
        if (mode == LAST_WITHOUT && (gone[(v - v0) >> 5] >> ((v - v0) & 31)) & 1) return 0.0;
        return e;
    }
};
// The whole block: bits of the refused ids in [v0, v0 + AC_CHUNK).
__device__ __forceinline__ void mark_gone(const AcceptArgs& a, int s, const AcceptLast& l, int v0, uint32_t* gone) {
    gone[threadIdx.x] = 0;
    __syncthreads();
    if (l.mode == LAST_WITHOUT && (int)threadIdx.x < l.n_out) {
        const int v = a.out_ids[s * MJ_ROWS + threadIdx.x] - v0;
        if ((unsigned)v < AC_CHUNK) atomicOr(&gone[v >> 5], 1u << (v & 31));
    }
    __syncthreads();
}

__global__ __launch_bounds__(256) void k_accept_sums(AcceptArgs a) {
    __shared__ uint32_t s_gone[AC_CHUNK / 32];
    __shared__ double s_s[4];
    if (block_aborted(a.abort)) return;
    const int s = blockIdx.y, t = threadIdx.x, v0 = blockIdx.x * AC_CHUNK;
    const AcceptLast l = a.last[s];
    if (l.row < 0) return;
    mark_gone(a, s, l, v0, s_gone);
    const Left left{a.logits + l.row * a.ld, a.q ? a.q + l.row * a.ldq : nullptr, l.m,
                    1.0 / (double)a.temperature[s], 1.0 / l.Z, l.mode, s_gone, v0};
    double sum = 0.0;
    for (int i = 0; i < 32; ++i) {
        const int v = v0 + 256 * i + t;
        if (v < a.V) sum += left.of(v);
    }
    sum = wave_sum64(sum);
    if ((t & 63) == 0) s_s[t >> 6] = sum;
    __syncthreads();
    if (t == 0) a.csum[(size_t)s * a.chunks + blockIdx.x] = (s_s[0] + s_s[1]) + (s_s[2] + s_s[3]);
}

// One block a sequence: the chunk where the sums cross u times all, then the id in it.
__global__ __launch_bounds__(256) void k_accept_pick(AcceptArgs a) {
    __shared__ uint32_t s_gone[AC_CHUNK / 32];
    __shared__ double s_s[256];
    __shared__ int s_last[256], s_pick;
    __shared__ double s_before;
    if (block_aborted(a.abort)) return;
    const int s = blockIdx.x, t = threadIdx.x;
    AcceptLast l = a.last[s];
    if (l.row < 0) return;
    const double k = 1.0 / (double)a.temperature[s];
    const double* sums = a.csum + (size_t)s * a.chunks;
    if (t == 0) {
        double total = 0.0;
        for (int c = 0; c < a.chunks; ++c) total += sums[c];
        // nothing left: the row's own probabilities
        s_last[0] = total > 0.0 ? l.mode : LAST_P;
    }
    __syncthreads();
    const bool plain = s_last[0] == LAST_P && l.mode != LAST_P;
    l.mode = s_last[0];
    __syncthreads();
    if (t == 0) {
        auto sum = [&](int c) {
            if (!plain) return sums[c];
            const AcceptPart p = a.part[(size_t)l.row * a.chunks + c];
            return p.m > -INFINITY ? p.s * weight(p.m, l.m, k) : 0.0;
        };
        double total = 0.0;
        for (int c = 0; c < a.chunks; ++c) total += sum(c);
        const double want = (double)a.u_sample[s] * total;
        int pick = -1;
        double before = 0.0, at = 0.0;
        for (int c = 0; c < a.chunks; ++c) {
            const double x = sum(c);
            if (x > 0.0) {
                pick = c;
                before = at;
                if (at + x > want) break;
            }
            at += x;
        }
        s_pick = pick;
        s_before = want - before;
    }
    __syncthreads();
    const int v0 = s_pick * AC_CHUNK;
    const double want = s_before;
    if (s_pick < 0) {
        if (t == 0) a.token[s] = -1;
        return;
    }
    mark_gone(a, s, l, v0, s_gone);
    const Left left{a.logits + l.row * a.ld, a.q ? a.q + l.row * a.ldq : nullptr, l.m, k, 1.0 / l.Z, l.mode,
                    s_gone, v0};
    // thread t: ids v0 + 32 t .. + 31
    double sum = 0.0;
    int last = -1;
    for (int i = 0; i < 32; ++i) {
        const int v = v0 + 32 * t + i;
        const double x = v < a.V ? left.of(v) : 0.0;
        sum += x;
        if (x > 0.0) last = v;
    }
    s_s[t] = sum;
    s_last[t] = last;
    __syncthreads();
    if (t != 0) return;
    double at = 0.0;
    int token = -1;
    for (int i = 0; i < 256; ++i) {
        if (s_last[i] < 0) continue;
        token = s_last[i];
        if (at + s_s[i] > want) {
            for (int v = v0 + 32 * i; v < min(a.V, v0 + 32 * i + 32); ++v) {
                const double x = left.of(v);
                at += x;
                if (x > 0.0 && at > want) {
                    token = v;
                    break;
                }
            }
            break;
        }
        at += s_s[i];
    }
    a.token[s] = token;
}

size_t accept_rows_layout(AcceptArgs& a, void* base) {
    a.chunks = (a.V + AC_CHUNK - 1) / AC_CHUNK;
    Arena ar{base, 0};
    a.part = (AcceptPart*)ar.take((size_t)a.b.rows * a.chunks * sizeof(AcceptPart));
    a.last = (AcceptLast*)ar.take((size_t)a.b.n_seqs * sizeof(AcceptLast));
    a.out_ids = (int32_t*)ar.take((size_t)a.b.n_seqs * MJ_ROWS * sizeof(int32_t));
    a.csum = (double*)ar.take((size_t)a.b.n_seqs * a.chunks * sizeof(double));
    return ar.off;
}

hipError_t launch_accept_rows(const AcceptArgs& a, hipStream_t st) {
    if (a.b.rows < 0 || a.b.rows > 65535 || a.b.n_seqs > 65535 || a.b.max_rows > MJ_ROWS || a.V < 1)
        return hipErrorInvalidValue;
    if (a.b.rows > 0)
        hipLaunchKernelGGL(k_accept_stats, dim3(a.chunks, a.b.rows), dim3(256), 0, st, a);
    hipLaunchKernelGGL(k_accept_walk, dim3(a.b.n_seqs), dim3(256), 0, st, a);
    hipLaunchKernelGGL(k_accept_sums, dim3(a.chunks, a.b.n_seqs), dim3(256), 0, st, a);
    hipLaunchKernelGGL(k_accept_pick, dim3(a.b.n_seqs), dim3(256), 0, st, a);
    return hipGetLastError();
}
