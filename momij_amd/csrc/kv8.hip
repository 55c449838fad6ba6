// kv8.hip -- the 8-bit KV cache: appending normed and rotated rows to the fp16 ring, sealing blocks
// into pages and back, choosing blocks by a cheap score, evicting them by accumulated weight.
// (Attention over the cache: kv8_attn.hip.)
#include "mj_device.h"
#include "mj_kv8.h"

#define HD 128

typedef int i4v __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------------ append
// A 256-thread block takes 32 of a row's nQ + 2 nKV vectors, eight lanes a vector, 16 dims a lane:
// parts pa and pa + X of 8 dims each, X = half / 8 parts apart, so that both dims of a rotated pair
// sit in one lane.  y = x / sqrt(mean x^2 + eps) * w, then (y_i, y_{i+half}) turned by the angle
// position * frequency_i.  The angle is formed in turns in 64 bits and reduced to half a turn before
// it is rounded to 32 (at position 131071 an angle formed in 32 bits is off by up to 4e-3).  The
// block's angles are formed once, in LDS, while its rows are on their way.
__global__ __launch_bounds__(256) void k_qkv_append(Kv8AppendArgs a) {
    __shared__ float2 cs[MJ_ROPE_F];
    __shared__ int s_abort;
    const int t = threadIdx.x, jb = t & 7, r = blockIdx.y;
    const int vec = blockIdx.x * 32 + (t >> 3), nv = a.nQ + 2 * a.nKV;
    const int vc = vec < nv ? vec : nv - 1;
    const int X = a.half >= 16 ? a.half / 8 : 8;
    const int pa = (jb & (X - 1)) | ((jb & ~(X - 1)) << 1), pb = pa + X;
    const uint16_t* src = a.qkv + (size_t)r * a.ld + (size_t)vc * HD;
    const bool isq = vc < a.nQ, isv = vc >= a.nQ + a.nKV;
    const uint16_t* nw = isq ? a.qw : a.kw;
    u4v va = *(const u4v*)(src + 8 * pa), vb = *(const u4v*)(src + 8 * pb);
    const u4v wa = *(const u4v*)(nw + 8 * pa), wb = *(const u4v*)(nw + 8 * pb);
    const int ab = a.abort ? *a.abort : 0;
    if (t == 0) s_abort = ab;
    if (t < a.half) {
        const double turn = (double)(a.L + a.depth[r]) * a.turns[t];
        float s, c;
        sincospif(2.0f * (float)(turn - rint(turn)), &s, &c);
        cs[t] = make_float2(c, s);
    }
    __syncthreads();
    if (s_abort) return;
    if (!isv) {
        float xa[8], xb[8], ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            xa[i] = h2f((uint16_t)(va[i >> 1] >> (16 * (i & 1))));
            xb[i] = h2f((uint16_t)(vb[i >> 1] >> (16 * (i & 1))));
            ss = fmaf(xa[i], xa[i], ss);
            ss = fmaf(xb[i], xb[i], ss);
        }
#pragma unroll
        for (int m = 1; m < 8; m <<= 1) ss += __shfl_xor(ss, m, MJ_WAVE);
        const float scl = 1.0f / sqrtf(ss / (float)HD + a.eps);
        const bool rot = 8 * pa < a.half;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            xa[i] = xa[i] * scl * h2f((uint16_t)(wa[i >> 1] >> (16 * (i & 1))));
            xb[i] = xb[i] * scl * h2f((uint16_t)(wb[i >> 1] >> (16 * (i & 1))));
            if (rot) {
                const float2 c = cs[8 * pa + i];
                const float ya = fmaf(xa[i], c.x, -(xb[i] * c.y));
                xb[i] = fmaf(xb[i], c.x, xa[i] * c.y);
                xa[i] = ya;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            va[j] = pack2(f2h(xa[2 * j]), f2h(xa[2 * j + 1]));
            vb[j] = pack2(f2h(xb[2 * j]), f2h(xb[2 * j + 1]));
        }
    }
    if (vec >= nv) return;
    uint16_t* dst;
    if (isq) {
        dst = a.q_out + ((size_t)r * a.nQ + vec) * HD;
    } else {
        int64_t slot = a.slot0 + r;
        slot -= slot >= a.ring.C ? a.ring.C : 0;
        const int g = vec - a.nQ - (isv ? a.nKV : 0);
        dst = (isv ? a.ring.v : a.ring.k) + ((size_t)g * a.ring.C + slot) * HD;
    }
    *(u4v*)(dst + 8 * pa) = va;
    *(u4v*)(dst + 8 * pb) = vb;
}

hipError_t launch_qkv_append(const Kv8AppendArgs& a, hipStream_t st) {
    if (a.M < 1 || a.M > MJ_ROWS || a.half > MJ_ROPE_F || (a.half & (a.half - 1)) || a.half == 8)
        return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_qkv_append, dim3((a.nQ + 2 * a.nKV + 31) / 32, a.M), dim3(256), 0, st, a);
    return hipGetLastError();
}

// -------------------------------------------------------------------------------------- seal
__device__ __forceinline__ int page_of(const Kv8Pool& p, int g, int i) {
    const int pg = p.table[(size_t)g * p.stride + i];
    return (unsigned)pg < (unsigned)p.n_pages ? pg : -1;
}
__device__ __forceinline__ size_t ring_row(const Kv8Ring& r, int g, int64_t slot0, int64_t i) {
    int64_t s = slot0 + i;
    s -= s >= r.C ? r.C : 0;
    return ((size_t)g * r.C + s) * HD;
}
__device__ __forceinline__ float absmax_finite(float m, float x) {
    const float ax = fabsf(x);
    return ax < INFINITY && ax > m ? ax : m;  // (a NaN compares false)
}
// code of x under 127 / greatest magnitude: nearest whole number, an infinity at +-127, a NaN 0
__device__ __forceinline__ int code8(float x, float r) {
    const float c = fminf(fmaxf(rintf(x * r), -127.0f), 127.0f);
    return x == x && r > 0.0f ? (int)c : 0;
}

// A 256-thread block seals K (blockIdx.z 0) or V (1) of one block of one head: 16 KB in, 8 KB of
// codes out.  Thread t holds dims 8 (t % 16) .. + 7 of tokens t / 16 + 16 i.  K codes go straight to
// their 8-byte places; V codes are turned by way of LDS, as a page has four tokens of a dim side by
// side.
__global__ __launch_bounds__(256) void k_kv8_seal(Kv8Pool p, Kv8Ring ring, int64_t slot0, int at,
                                                  const int* abort) {
    __shared__ float red[4];
    __shared__ __align__(16) uint8_t tile[KV8_B][HD + 4];
    __shared__ int8_t lim[2][16][HD];
    __shared__ int s_abort;
    const int t = threadIdx.x, dg = t & 15, k0 = t >> 4;
    const int i = blockIdx.x, g = blockIdx.y;
    const bool isv = blockIdx.z != 0;
    const uint16_t* src = isv ? ring.v : ring.k;
    u4v raw[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        raw[j] = *(const u4v*)(src + ring_row(ring, g, slot0, (int64_t)KV8_B * i + k0 + 16 * j) +
                               8 * dg);
    const int ab = abort ? *abort : 0;
    if (t == 0) s_abort = ab;
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e)
            m = absmax_finite(m, h2f((uint16_t)(raw[j][e >> 1] >> (16 * (e & 1)))));
    m = wave_max(m);
    if ((t & 63) == 0) red[t >> 6] = m;
    const int pg = page_of(p, g, at + i);
    __syncthreads();
    if (s_abort || pg < 0) return;  // whole block
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float r = m > 0.0f ? 127.0f / m : 0.0f;
    if (t == 0) (isv ? p.vs : p.ks)[pg] = m / 127.0f;
    uint8_t* dst = (isv ? p.v : p.k) + (size_t)pg * KV8_PAGE_BYTES;
    int hi[8], lo[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int c = code8(h2f((uint16_t)(raw[j][e >> 1] >> (16 * (e & 1)))), r);
            hi[e] = j == 0 ? c : max(hi[e], c);
            lo[e] = j == 0 ? c : min(lo[e], c);
            w[e >> 2] |= (uint32_t)(c + 128) << (8 * (e & 3));
        }
        const int key = k0 + 16 * j;
        if (!isv) {
            *(uint2*)(dst + 2048 * j + 1024 * (dg >> 3) + 256 * ((dg >> 1) & 3) + 16 * k0 +
                      8 * (dg & 1)) = make_uint2(w[0], w[1]);
        } else {
            *(uint32_t*)&tile[key][8 * dg] = w[0];
            *(uint32_t*)&tile[key][8 * dg + 4] = w[1];
        }
    }
    if (!isv) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            lim[0][k0][8 * dg + e] = (int8_t)hi[e];
            lim[1][k0][8 * dg + e] = (int8_t)lo[e];
        }
    }
    __syncthreads();
    if (!isv) {  // thread t: greatest (t < 128) or least code of dim t % 128
        const int which = t >> 7, d = t & 127;
        int v = lim[which][0][d];
#pragma unroll
        for (int k = 1; k < 16; ++k) v = which ? min(v, (int)lim[1][k][d]) : max(v, (int)lim[0][k][d]);
        p.bounds[(size_t)pg * (2 * HD) + t] = (int8_t)v;
    } else {
#pragma unroll
        for (int c = 0; c < 2; ++c) {  // 16 bytes of a page: dim d, tokens 4 lq + b % 4 + 16 (b / 4)
            const int ch = t + 256 * c, d = 16 * (ch >> 6) + (ch & 15), lq = (ch >> 4) & 3;
            u4v o;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t w = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b) w |= (uint32_t)tile[16 * q + 4 * lq + b][d] << (8 * b);
                o[q] = w;
            }
            *(u4v*)(dst + 16 * ch) = o;
        }
    }
}

// The way back: half(code * scale) into the ring's rows; V by way of LDS again.
__global__ __launch_bounds__(256) void k_kv8_unseal(Kv8Pool p, Kv8Ring ring, int64_t slot0, int at,
                                                    const int* abort) {
    __shared__ __align__(16) uint8_t tile[KV8_B][HD + 4];
    __shared__ int s_abort;
    const int t = threadIdx.x, dg = t & 15, k0 = t >> 4;
    const int i = blockIdx.x, g = blockIdx.y;
    const bool isv = blockIdx.z != 0;
    const int pg = page_of(p, g, at + i);
    const int ab = abort ? *abort : 0;
    if (t == 0) s_abort = ab;
    __syncthreads();
    if (s_abort || pg < 0) return;  // whole block
    const uint8_t* src = (isv ? p.v : p.k) + (size_t)pg * KV8_PAGE_BYTES;
    const float s = (isv ? p.vs : p.ks)[pg];
    if (isv) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int ch = t + 256 * c, d = 16 * (ch >> 6) + (ch & 15), lq = (ch >> 4) & 3;
            const u4v o = *(const u4v*)(src + 16 * ch);
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int b = 0; b < 4; ++b) tile[16 * q + 4 * lq + b][d] = (uint8_t)(o[q] >> (8 * b));
        }
        __syncthreads();
    }
    uint16_t* out = isv ? ring.v : ring.k;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t w[2];
        const int key = k0 + 16 * j;
        if (!isv) {
            const uint2 v = *(const uint2*)(src + 2048 * j + 1024 * (dg >> 3) + 256 * ((dg >> 1) & 3) +
                                            16 * k0 + 8 * (dg & 1));
            w[0] = v.x;
            w[1] = v.y;
        } else {
            w[0] = *(const uint32_t*)&tile[key][8 * dg];
            w[1] = *(const uint32_t*)&tile[key][8 * dg + 4];
        }
        u4v o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c0 = (int)((w[e >> 1] >> (16 * (e & 1))) & 255u) - 128;
            const int c1 = (int)((w[e >> 1] >> (16 * (e & 1) + 8)) & 255u) - 128;
            o[e] = pack2(f2h((float)c0 * s), f2h((float)c1 * s));
        }
        *(u4v*)(out + ring_row(ring, g, slot0, (int64_t)KV8_B * i + key) + 8 * dg) = o;
    }
}

hipError_t launch_kv8_seal(const Kv8Pool& p, const Kv8Ring& r, int64_t slot0, int count, int at,
                           const int* abort, hipStream_t st) {
    hipLaunchKernelGGL(k_kv8_seal, dim3(count, p.nKV, 2), dim3(256), 0, st, p, r, slot0, at, abort);
    return hipGetLastError();
}
hipError_t launch_kv8_unseal(const Kv8Pool& p, const Kv8Ring& r, int64_t slot0, int count, int at,
                             const int* abort, hipStream_t st) {
    hipLaunchKernelGGL(k_kv8_unseal, dim3(count, p.nKV, 2), dim3(256), 0, st, p, r, slot0, at, abort);
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------ select
// Order-preserving key of a float: greater float, greater key; -0 as +0, a NaN below -inf.
__device__ __forceinline__ uint32_t order_key(float f) {
    const uint32_t b = __float_as_uint(f + 0.0f);
    return f != f ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// Scores of 64 blocks of one head for the rows of blockIdx.z's share, a wave 16 blocks:
//   u = sum_d max(c_d hi_d, c_d lo_d) = sum_d c+_d hi_d + c-_d lo_d,  c+ = max(c, 0), c- = min(c, 0),
// on v_mfma_i32_16x16x64_i8 (blocks as rows, query heads as columns), exact in whole numbers.  A
// row's heads take P columns (the next power of two, at most 16; more heads in further products), so
// that their maximum is found by xor moves.  Reads 256 bytes a block where attention reads 16 KB.
__global__ __launch_bounds__(256) void k_kv8_score(Kv8SelectArgs a, int P, int tiles_z) {
    const int t = threadIdx.x, lane = t & 63, ln = lane & 15, lq = lane >> 4;
    const int g = blockIdx.y, b0 = blockIdx.x * 64 + 16 * (t >> 6);
    const int idx = b0 + ln, nQ = a.p.nKV * a.G;
    const int pg = idx < a.n ? page_of(a.p, g, idx) : -1;
    if (aborted(a.abort)) return;
    i4v hi[2], lo[2];
    {
        const int8_t* b = a.p.bounds + (size_t)(pg < 0 ? 0 : pg) * (2 * HD) + 16 * lq;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            hi[j] = *(const i4v*)(b + 64 * j);
            lo[j] = *(const i4v*)(b + HD + 64 * j);
        }
    }
    const float ks_l = pg < 0 ? 0.0f : a.p.ks[pg];
    float ks[4];
    bool have[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        ks[r] = __shfl(ks_l, 4 * lq + r, MJ_WAVE);
        have[r] = __shfl(pg, 4 * lq + r, MJ_WAVE) >= 0;
    }
    const int rpt = 16 / P, tiles = (a.M + rpt - 1) / rpt;
    const int t0 = blockIdx.z * tiles_z, t1 = min(t0 + tiles_z, tiles);
    for (int rt = t0; rt < t1; ++rt) {
        const int row = rt * rpt + ln / P;
        float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        for (int h0 = 0; h0 < a.G; h0 += 16) {
            const int head = h0 + ln % P;
            const bool on = row < a.M && head < a.G;
            const uint16_t* q = a.q + (size_t)(on ? row : 0) * a.ldq +
                                (size_t)(g * a.G + (on ? head : 0)) * HD + 16 * lq;
            u4v raw[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) raw[j] = *(const u4v*)(q + 64 * (j >> 1) + 8 * (j & 1));
            float m = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    m = absmax_finite(m, h2f((uint16_t)(raw[j][e >> 1] >> (16 * (e & 1)))));
            m = fmaxf(m, __shfl_xor(m, 16, MJ_WAVE));
            m = fmaxf(m, __shfl_xor(m, 32, MJ_WAVE));
            const float r = m > 0.0f ? 127.0f / m : 0.0f, sq = m / 127.0f;
            i4v up[2], dn[2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t pu = 0, pd = 0;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const int e = 4 * w + b;
                        const int c = code8(
                            h2f((uint16_t)(raw[2 * j + (e >> 3)][(e & 7) >> 1] >> (16 * (e & 1)))), r);
                        pu |= (uint32_t)(max(c, 0) & 255) << (8 * b);
                        pd |= (uint32_t)(min(c, 0) & 255) << (8 * b);
                    }
                    up[j][w] = (int)pu;
                    dn[j][w] = (int)pd;
                }
            i4v u = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                u = __builtin_amdgcn_mfma_i32_16x16x64_i8(hi[j], up[j], u, 0, 0, 0);
                u = __builtin_amdgcn_mfma_i32_16x16x64_i8(lo[j], dn[j], u, 0, 0, 0);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float sc = (float)u[k] * ks[k] * sq;
                best[k] = on && have[k] && sc > best[k] ? sc : best[k];  // (not a NaN)
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            for (int o = 1; o < P; o <<= 1) best[k] = fmaxf(best[k], __shfl_xor(best[k], o, MJ_WAVE));
        if (ln % P == 0 && row < a.M) {
            float* s = a.scores + ((size_t)row * a.p.nKV + g) * a.n;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (b0 + 4 * lq + k < a.n) s[b0 + 4 * lq + k] = best[k];
        }
    }
}

// The k greatest of n keys (0 < k <= n), the lower index first among equal ones: the threshold key
// and how many of the keys equal to it belong to them.  Radix selection, eight bits a round from the
// top; whole block of NT threads, the same in every thread.
template <int NT, typename F>
__device__ __forceinline__ void kth_key(F key, int n, int k, uint32_t& thr, int& take) {
    __shared__ int hist[256];
    __shared__ int s_dig, s_left;
    const int t = threadIdx.x;
    uint32_t prefix = 0;
    for (int sh = 24; sh >= 0; sh -= 8) {
        for (int i = t; i < 256; i += NT) hist[i] = 0;
        __syncthreads();
        for (int i = t; i < n; i += NT) {
            const uint32_t u = key(i);
            if (sh == 24 || (u >> (sh + 8)) == (prefix >> (sh + 8))) atomicAdd(&hist[(u >> sh) & 255], 1);
        }
        __syncthreads();
        if (t < 64) {
            // lane t: digits 255 - 4 t .. 252 - 4 t; the digit whose running count reaches k
            int c[4], tot = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                c[j] = hist[255 - 4 * t - j];
                tot += c[j];
            }
            int run = tot;
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(run, o, MJ_WAVE);
                if (t >= o) run += v;
            }
            int before = run - tot;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (before < k && before + c[j] >= k) {
                    s_dig = 255 - 4 * t - j;
                    s_left = k - before;
                }
                before += c[j];
            }
        }
        __syncthreads();
        prefix |= (uint32_t)s_dig << sh;
        k = s_left;
        __syncthreads();
    }
    thr = prefix;
    take = k;
}

// In increasing index order, out(i, place, chosen): place among the chosen or among the others.
template <int NT, typename F, typename O>
__device__ __forceinline__ void split_by_key(F key, int n, uint32_t thr, int take, O out) {
    __shared__ int s_eq[NT / 64], s_in[NT / 64];
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    const uint64_t below = (1ull << lane) - 1;
    int eq0 = 0, in0 = 0;  // equal and chosen ones of the rounds before
    for (int i0 = 0; i0 < n; i0 += NT) {
        const int i = i0 + t;
        const uint32_t u = i < n ? key(i) : 0;
        const bool eq = i < n && u == thr;
        const uint64_t beq = __ballot(eq);
        if (lane == 0) s_eq[wv] = __popcll(beq);
        __syncthreads();
        int eqb = eq0, eqt = 0;
        for (int w = 0; w < NT / 64; ++w) {
            eqb += w < wv ? s_eq[w] : 0;
            eqt += s_eq[w];
        }
        const bool in = i < n && (u > thr || (eq && eqb + __popcll(beq & below) < take));
        const uint64_t bin = __ballot(in);
        if (lane == 0) s_in[wv] = __popcll(bin);
        __syncthreads();
        int inb = in0, intot = 0;
        for (int w = 0; w < NT / 64; ++w) {
            inb += w < wv ? s_in[w] : 0;
            intot += s_in[w];
        }
        const int place = inb + __popcll(bin & below);
        if (i < n) out(i, in ? place : i - place, in);
        eq0 += eqt;
        in0 += intot;
        __syncthreads();
    }
}

// One block a row and head: the n_sel greatest scores, the first and last blocks above all others.
template <int NT>
__global__ __launch_bounds__(NT) void k_kv8_topk(Kv8SelectArgs a) {
    const size_t rg = blockIdx.x;
    if (block_aborted(a.abort)) return;
    const float* s = a.scores + rg * a.n;
    int32_t* sel = a.sel + rg * a.n_sel;
    auto key = [&](int i) -> uint32_t {
        return i < a.first || i >= a.n - a.last ? 0xFFFFFFFFu : order_key(s[i]);
    };
    const int k = min(a.n_sel, a.n);
    if (k > 0) {
        uint32_t thr;
        int take;
        kth_key<NT>(key, a.n, k, thr, take);
        split_by_key<NT>(key, a.n, thr, take, [&](int i, int place, bool in) {
            if (in) sel[place] = i;
        });
    }
    for (int i = k + threadIdx.x; i < a.n_sel; i += NT) sel[i] = -1;
}

hipError_t launch_kv8_select(const Kv8SelectArgs& a, hipStream_t st) {
    if (a.n > 0) {
        int P = 1;
        while (P < a.G && P < 16) P *= 2;
        const int rpt = 16 / P, tiles = (a.M + rpt - 1) / rpt, nb = (a.n + 63) / 64;
        // the rows' tiles over further blocks while the launch is small
        int z = 1;
        while (z < tiles && nb * a.p.nKV * z < 512) z *= 2;
        const int per = (tiles + z - 1) / z;
        hipLaunchKernelGGL(k_kv8_score, dim3(nb, a.p.nKV, (tiles + per - 1) / per), dim3(256), 0, st, a,
                           P, per);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(k_kv8_topk<1024>, dim3(a.M * a.p.nKV), dim3(1024), 0, st, a);
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------- evict
// One block a head: the `keep` greatest masses, the first and last blocks above all others; the
// table and the masses split in two, each part in its old order.
template <int NT>
__global__ __launch_bounds__(NT) void k_kv8_evict(Kv8Pool p, int n, int keep, int first, int last,
                                                  const float* __restrict__ mass_in,
                                                  int32_t* __restrict__ table_out,
                                                  float* __restrict__ mass_out, const int* abort) {
    if (block_aborted(abort)) return;
    const size_t row = (size_t)blockIdx.x * p.stride;
    const float* m = mass_in + row;
    auto key = [&](int i) -> uint32_t {
        return i < first || i >= n - last ? 0xFFFFFFFFu : order_key(m[i]);
    };
    uint32_t thr = 0xFFFFFFFFu;  // keep 0: nothing stays
    int take = 0;
    if (keep > 0) kth_key<NT>(key, n, keep, thr, take);
    split_by_key<NT>(key, n, thr, take, [&](int i, int place, bool in) {
        const int at = in ? place : keep + place;
        table_out[row + at] = p.table[row + i];
        mass_out[row + at] = in ? m[i] : 0.0f;
    });
    for (int i = n + threadIdx.x; i < p.stride; i += NT) {
        table_out[row + i] = p.table[row + i];
        mass_out[row + i] = 0.0f;
    }
}

hipError_t launch_kv8_evict(const Kv8Pool& p, int n, int keep, int first, int last,
                            const float* mass_in, int32_t* table_out, float* mass_out,
                            const int* abort, hipStream_t st) {
    hipLaunchKernelGGL(k_kv8_evict<1024>, dim3(p.nKV), dim3(1024), 0, st, p, n, keep, first, last,
                       mass_in, table_out, mass_out, abort);
    return hipGetLastError();
}
