// kv8.hip -- the 8-bit KV cache: appending normed and rotated rows to the fp16 ring, sealing blocks
// into pages and back, choosing blocks by a cheap score, evicting them by accumulated weight.
// (Attention over the cache: kv8_attn.hip.)
#include <type_traits>

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
// block's angles are formed once, in LDS, while its rows are on their way.  One row of 24 vectors 2.6 us,
// 64 rows 3.6 us: a launch, a round of requests and the angles, not the 0.8 MB.
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
// code of x under r = 127 / greatest magnitude (0: all codes 0): nearest whole number, an infinity at
// +-127, a NaN 0
__device__ __forceinline__ int code8(float x, float r) {
    float v = x * r;
    v = v == v ? v : 0.0f;
    return (int)rintf(__builtin_amdgcn_fmed3f(v, -127.0f, 127.0f));
}
__device__ __forceinline__ uint32_t bytes4(int a, int b, int c, int d) {  // the low bytes, a lowest
    const uint32_t ab = __builtin_amdgcn_perm((uint32_t)b, (uint32_t)a, 0x0C0C0400u);
    const uint32_t cd = __builtin_amdgcn_perm((uint32_t)d, (uint32_t)c, 0x0C0C0400u);
    return ab | (cd << 16);
}

// Wave-wide steps by lane moves (an LDS shuffle costs some 100 cycles a step, and a block that does
// little else waits for each): inclusive sums, and the least and greatest in every lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_scan(int v) {
    v = dpp_add<0x111, 0xF>(v);  // from 1, 2, 4, 8 lanes below in the row
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);  // row 0's total to row 1, row 2's to row 3
    return dpp_add<0x143, 0xC>(v);  // rows 0 and 1's to rows 2 and 3
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_mov(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xF, 0xF, false);
}
template <bool MIN>
__device__ __forceinline__ uint32_t wave_ext(uint32_t v) {
    auto ext = [](uint32_t a, uint32_t b) { return MIN ? min(a, b) : max(a, b); };
    v = ext(v, dpp_mov<0xB1>(v));   // xor 1
    v = ext(v, dpp_mov<0x4E>(v));   // xor 2
    v = ext(v, dpp_mov<0x141>(v));  // eight lanes mirrored
    v = ext(v, dpp_mov<0x140>(v));  // sixteen
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = ext(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return ext(b[0], b[1]);
}

// A 256-thread block seals K (blockIdx.z 0) or V (1) of one block of one head: 16 KB in, 8 KB of
// codes out.  Thread t holds dims 8 (t % 16) .. + 7 of tokens t / 16 + 16 i.  K codes go straight to
// their 8-byte places; V codes are turned by way of LDS, as a page has four tokens of a dim side by
// side.  Bound by memory: 2048 blocks of 4 heads, 402 MB, in about 80 us (5 TB/s; a copy reaches 5.2); the
// ring's rows, done with here, pass by the caches (87 us else, the codes' lines pushed out).
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
        raw[j] = __builtin_nontemporal_load(
            (const u4v*)(src + ring_row(ring, g, slot0, (int64_t)KV8_B * i + k0 + 16 * j) + 8 * dg));
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
        int c[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            c[e] = code8(h2f((uint16_t)(raw[j][e >> 1] >> (16 * (e & 1)))), r);
            hi[e] = j == 0 ? c[e] : max(hi[e], c[e]);
            lo[e] = j == 0 ? c[e] : min(lo[e], c[e]);
        }
        const uint32_t w[2] = {bytes4(c[0], c[1], c[2], c[3]) ^ 0x80808080u,
                               bytes4(c[4], c[5], c[6], c[7]) ^ 0x80808080u};
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

// The way back: half(code * scale) into the ring's rows; V by way of LDS again.  The same 402 MB in 59
// us, part of the codes still in the last cache (63 us with the rows kept in the caches).
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
        __builtin_nontemporal_store(
            o, (u4v*)(out + ring_row(ring, g, slot0, (int64_t)KV8_B * i + key) + 8 * dg));
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

// max over 16 consecutive lanes, in all of them
__device__ __forceinline__ float max16(float v) {
    auto step = [](float x, uint32_t y) { return fmaxf(x, __uint_as_float(y)); };
    v = step(v, dpp_mov<0xB1>(__float_as_uint(v)));
    v = step(v, dpp_mov<0x4E>(__float_as_uint(v)));
    v = step(v, dpp_mov<0x141>(__float_as_uint(v)));
    return step(v, dpp_mov<0x140>(__float_as_uint(v)));
}

// A query vector's 8-bit codes as operands: lane (ln, lq) holds dims 64 j + 16 lq + 0 .. 15 of column
// ln's vector q; up = max(c, 0), dn = min(c, 0); returns the scale.
__device__ __forceinline__ float query_codes(const uint16_t* q, i4v up[2], i4v dn[2]) {
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
    const float r = m > 0.0f ? 127.0f / m : 0.0f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            int c[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int e = 4 * w + b;
                c[b] = code8(h2f((uint16_t)(raw[2 * j + (e >> 3)][(e & 7) >> 1] >> (16 * (e & 1)))), r);
            }
            const uint32_t pc = bytes4(c[0], c[1], c[2], c[3]);
            const uint32_t sign = (pc >> 7) & 0x01010101u, neg = (sign << 8) - sign;  // bytes < 0
            up[j][w] = (int)(pc & ~neg);
            dn[j][w] = (int)(pc & neg);
        }
    return m / 127.0f;
}

// u = sum_d max(c_d hi_d, c_d lo_d) = sum_d up_d hi_d + dn_d lo_d of 16 blocks (rows) and 16 query
// vectors (columns), exact in whole numbers.
__device__ __forceinline__ i4v bound_sums(const i4v hi[2], const i4v lo[2], const i4v up[2],
                                          const i4v dn[2]) {
    i4v u = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        u = __builtin_amdgcn_mfma_i32_16x16x64_i8(hi[j], up[j], u, 0, 0, 0);
        u = __builtin_amdgcn_mfma_i32_16x16x64_i8(lo[j], dn[j], u, 0, 0, 0);
    }
    return u;
}
__device__ __forceinline__ void load_bounds(const Kv8Pool& p, int pg, i4v hi[2], i4v lo[2]) {
    const int8_t* b = p.bounds + (size_t)max(pg, 0) * (2 * HD) + 16 * ((threadIdx.x & 63) >> 4);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        hi[j] = *(const i4v*)(b + 64 * j);
        lo[j] = *(const i4v*)(b + HD + 64 * j);
    }
}

// Scores of 64 blocks of one head for the rows of blockIdx.z's share, a wave 16 blocks:
//   u = sum_d max(c_d hi_d, c_d lo_d) = sum_d c+_d hi_d + c-_d lo_d,  c+ = max(c, 0), c- = min(c, 0),
// on v_mfma_i32_16x16x64_i8 (blocks as rows, query heads as columns), exact in whole numbers.  A
// row's heads take P columns (the next power of two, at most 16; more heads in further products), so
// that their maximum is found by xor moves.  Reads 256 bytes a block where attention reads 16 KB: 2047
// blocks of 4 heads for one row, 2.1 MB, 5.2 us, a launch and two requests that wait for each other
// (the page's number, its bounds); 2000 blocks for 64 rows 17 us (the query codes, formed by every
// block again).
__global__ __launch_bounds__(256) void k_kv8_score(Kv8SelectArgs a, int P, int tiles_z) {
    const int t = threadIdx.x, lane = t & 63, ln = lane & 15, lq = lane >> 4;
    const int g = blockIdx.y, b0 = blockIdx.x * 64 + 16 * (t >> 6);
    const int idx = b0 + ln, nQ = a.p.nKV * a.G;
    const int pg = idx < a.n ? page_of(a.p, g, idx) : -1;
    const int ab = a.abort ? *a.abort : 0;  // decides at the end, off the chain table -> bounds
    i4v hi[2], lo[2];
    load_bounds(a.p, pg, hi, lo);
    const float ks_l = a.p.ks[max(pg, 0)];
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
            i4v up[2], dn[2];
            const float sq = query_codes(q, up, dn);
            const i4v u = bound_sums(hi, lo, up, dn);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float sc = (float)u[k] * ks[k] * sq;
                best[k] = on && have[k] && sc > best[k] ? sc : best[k];  // (not a NaN)
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            for (int o = 1; o < P; o <<= 1) best[k] = fmaxf(best[k], __shfl_xor(best[k], o, MJ_WAVE));
        if (ab == 0 && ln % P == 0 && row < a.M) {
            float* s = a.scores + ((size_t)row * a.p.nKV + g) * a.n;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (b0 + 4 * lq + k < a.n) s[b0 + 4 * lq + k] = best[k];
        }
    }
}

// The k greatest of the keys that a block's threads hold in registers, the lower index first among
// equal ones: thr and take such that key > thr, or key == thr and among the first `take` of those.
// Thread (w, lane) holds R keys, of indices (w R + r) 64 + lane; ON marks those that compete (k of
// them at least, k > 0).  The range of the keys is cut into 1024 equal bins, the bin that holds the
// k-th found, and so on inside it until it holds 64 keys or fewer, which one wave ranks: one round
// for scores that spread at all (a radix round of eight bits a time took four, most keys meeting in
// one bin of the first).
template <int NT, int R>
__device__ __forceinline__ void kth_of(const uint32_t key[R], const bool on[R], int k, uint32_t& thr,
                                       int& take) {
    constexpr int NW = NT / 64, LB = NT == 1024 ? 10 : 8;  // a thread a bin
    static_assert(NT == 1 << LB, "");
    __shared__ int hist[NT], s_tot[NW], s_pick[3], s_n;
    __shared__ uint32_t s_lo[NW], s_hi[NW], s_cand[64];
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6, lw = lane & (NW - 1);
    uint32_t lo = 0xFFFFFFFFu, hi = 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (on[r]) {
            lo = min(lo, key[r]);
            hi = max(hi, key[r]);
        }
    lo = wave_ext<true>(lo);
    hi = wave_ext<false>(hi);
    if (lane == 0) {
        s_lo[wv] = lo;
        s_hi[wv] = hi;
    }
    hist[t] = 0;
    if (t == 0) s_n = 0;
    __syncthreads();
    lo = wave_ext<true>(s_lo[lw]);
    hi = wave_ext<false>(s_hi[lw]);
    for (;;) {
        const int bits = hi > lo ? 32 - __clz((int)(hi - lo)) : 0, sh = bits > LB ? bits - LB : 0;
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (on[r] && key[r] >= lo && key[r] <= hi) atomicAdd(&hist[(key[r] - lo) >> sh], 1);
        __syncthreads();
        const int c = hist[NT - 1 - t];  // bins from the top
        const int run = wave_scan(c);
        if (lane == 63) s_tot[wv] = run;
        __syncthreads();
        const int tot = wave_scan(lane < NW ? s_tot[lw] : 0);
        const int before = run - c + (wv ? __builtin_amdgcn_readlane(tot, wv - 1) : 0);
        if (before < k && before + c >= k) {
            s_pick[0] = NT - 1 - t;
            s_pick[1] = before;
            s_pick[2] = c;
        }
        hist[NT - 1 - t] = 0;
        __syncthreads();
        lo += (uint32_t)s_pick[0] << sh;
        hi = min(hi, lo + ((1u << sh) - 1));
        k -= s_pick[1];
        const int in = s_pick[2];
        if (sh == 0) {  // one key is left
            thr = lo;
            take = k;
            return;
        }
        if (in == k) {  // the whole bin: the keys from lo on
            thr = lo > 0 ? lo - 1 : 0;
            take = lo > 0 ? 0 : 0x7FFFFFFF;
            return;
        }
        if (in > 64) continue;  // (nobody writes s_pick before the next two barriers)
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (on[r] && key[r] >= lo && key[r] <= hi) s_cand[atomicAdd(&s_n, 1)] = key[r];
        __syncthreads();
        // every wave ranks them for itself
        const uint32_t mine = lane < in ? s_cand[lane] : 0;
        int above = 0, same = 0;
        for (int i = 0; i < in; ++i) {
            const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)mine, i);
            above += o > mine;
            same += o == mine;
        }
        const int at = __builtin_ctzll(__ballot(lane < in && above < k && k <= above + same));
        thr = (uint32_t)__builtin_amdgcn_readlane((int)mine, at);
        take = k - __builtin_amdgcn_readlane(above, at);
        return;
    }
}

// The keys of kth_of's layout split in two, each part in increasing index order: out(i, place, chosen),
// place among the chosen (sure: without competing) or among the others; n keys in all.
template <int NT, int R, typename O>
__device__ __forceinline__ void split_keys(const uint32_t key[R], const bool on[R], const bool sure[R],
                                           int n, uint32_t thr, int take, O out) {
    constexpr int NW = NT / 64;
    __shared__ int s_eq[NW], s_gt[NW];
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6, lw = lane & (NW - 1);
    const uint64_t below = (1ull << lane) - 1;
    int eq = 0, gt = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        eq += __popcll(__ballot(on[r] && key[r] == thr));
        gt += __popcll(__ballot(sure[r] || (on[r] && key[r] > thr)));
    }
    if (lane == 0) {
        s_eq[wv] = eq;
        s_gt[wv] = gt;
    }
    __syncthreads();
    eq = wave_scan(lane < NW ? s_eq[lw] : 0);
    gt = wave_scan(lane < NW ? s_gt[lw] : 0);
    eq = wv ? __builtin_amdgcn_readlane(eq, wv - 1) : 0;  // those of the waves before
    gt = wv ? __builtin_amdgcn_readlane(gt, wv - 1) : 0;
    int in = gt + min(eq, take);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = (wv * R + r) * 64 + lane;
        const uint64_t e = __ballot(on[r] && key[r] == thr);
        const bool chosen = sure[r] || (on[r] && (key[r] > thr || (key[r] == thr &&
                                                                   eq + __popcll(e & below) < take)));
        const uint64_t b = __ballot(chosen);
        const int place = in + __popcll(b & below);
        if (i < n) out(i, r, chosen ? place : i - place, chosen);
        eq += __popcll(e);
        in += __popcll(b);
    }
}

// k of n keys (0 <= k <= n), those of the first and last indices for certain.  key(i, r) requests the
// key of index i < n, the thread's r-th (of no keys: -1); abort: thread 0's reading decides for the
// block, which returns false with nothing done.
template <int NT, int R, typename F, typename O>
__device__ __forceinline__ bool pick_keys(F key, int n, int k, int first, int last, int abort, O out) {
    __shared__ int s_abort;
    const int t = threadIdx.x;
    uint32_t kr[R], thr = 0xFFFFFFFFu;  // (no key of a float)
    bool on[R], sure[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = ((t >> 6) * R + r) * 64 + (t & 63);
        sure[r] = i < n && (i < first || i >= n - last || k == n);
        on[r] = i < n && !sure[r];
        kr[r] = key(min(i, n - 1), r);
    }
    if (t == 0) s_abort = abort;
    __syncthreads();
    if (s_abort) return false;
    int take = 0;
    const int left = k == n ? 0 : k - first - last;  // (first + last <= k < n: they do not overlap)
    if (left > 0) kth_of<NT, R>(kr, on, left, thr, take);
    split_keys<NT, R>(kr, on, sure, n, thr, take, out);
    return true;
}

// One block a row and head: scores formed in LDS, then the n_sel greatest, for up to CHOOSE_MAX blocks
// (their 256 bytes each come through one CU, which has only so many lines under way: of 8 rows 250
// blocks take 10 us and 500 13, in two launches 12.5 and 12.5 and the gap between them, so about there
// the two meet; 1000 19 and 13.5).
#define CHOOSE_MAX 512
__global__ __launch_bounds__(1024) void k_kv8_choose(Kv8SelectArgs a) {
    __shared__ float s_sc[CHOOSE_MAX];
    __shared__ __align__(16) i4v s_q[4][4][64];
    __shared__ float s_sq[4][16];
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6, ln = lane & 15, lq = lane >> 4;
    const int g = blockIdx.x, row = blockIdx.y, groups = (a.G + 15) / 16;
    const int ab = a.abort ? *a.abort : 0;
    constexpr int X = CHOOSE_MAX / 256;
    int pg[X];
#pragma unroll
    for (int x = 0; x < X; ++x) {
        const int idx = 16 * (wv + 16 * x) + ln;
        pg[x] = idx < a.n ? page_of(a.p, g, idx) : -1;
    }
    i4v hi[X][2], lo[X][2];
    float ksl[X];
#pragma unroll
    for (int x = 0; x < X; ++x) {
        if (16 * (wv + 16 * x) >= a.n) break;  // uniform
        load_bounds(a.p, pg[x], hi[x], lo[x]);
        ksl[x] = a.p.ks[max(pg[x], 0)];
    }
    if (wv < groups) {  // 16 heads a wave; a head past the group's last takes that one again
        const int head = min(16 * wv + ln, a.G - 1);
        i4v up[2], dn[2];
        const float sq =
            query_codes(a.q + (size_t)row * a.ldq + (size_t)(g * a.G + head) * HD + 16 * lq, up, dn);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            s_q[wv][j][lane] = up[j];
            s_q[wv][2 + j][lane] = dn[j];
        }
        if (lq == 0) s_sq[wv][ln] = sq;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < X; ++x) {
        const int b0 = 16 * (wv + 16 * x);
        if (b0 >= a.n) break;
        float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, ks[4];
        bool have[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            ks[k] = __shfl(ksl[x], 4 * lq + k, MJ_WAVE);
            have[k] = __shfl(pg[x], 4 * lq + k, MJ_WAVE) >= 0;
        }
        for (int h = 0; h < groups; ++h) {
            const i4v up[2] = {s_q[h][0][lane], s_q[h][1][lane]};
            const i4v dn[2] = {s_q[h][2][lane], s_q[h][3][lane]};
            const i4v u = bound_sums(hi[x], lo[x], up, dn);
            const float sq = s_sq[h][ln];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float sc = (float)u[k] * ks[k] * sq;
                best[k] = have[k] && sc > best[k] ? sc : best[k];  // (not a NaN)
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            best[k] = max16(best[k]);
            if (ln == 0) s_sc[b0 + 4 * lq + k] = best[k];
        }
    }
    __syncthreads();
    int32_t* sel = a.sel + ((size_t)row * a.p.nKV + g) * a.n_sel;
    const int k = min(a.n_sel, a.n);
    if (!pick_keys<1024, 1>([&](int i, int) { return order_key(s_sc[max(i, 0)]); }, a.n, k, a.first,
                            a.last, ab, [&](int i, int, int place, bool in) {
                                if (in) sel[place] = i;
                            }))
        return;
    for (int i = k + t; i < a.n_sel; i += 1024) sel[i] = -1;
}

// The same over keys in memory, any number of them (0 < k <= n), by radix selection, eight bits a round
// from the top; whole block of NT threads, thr and take the same in every thread.
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

// One block a row and head: the n_sel greatest scores; R keys a thread in registers, or R = 0: in
// memory (lists past 16384).  2047 scores 5.2 us: a launch, a request and seven barriers or more.
template <int NT, int R>
__global__ __launch_bounds__(NT) void k_kv8_topk(Kv8SelectArgs a) {
    const size_t rg = blockIdx.x;
    const float* s = a.scores + rg * a.n;
    int32_t* sel = a.sel + rg * a.n_sel;
    const int k = min(a.n_sel, a.n);
    if constexpr (R > 0) {
        const int ab = a.abort ? *a.abort : 0;
        if (!pick_keys<NT, R>([&](int i, int) { return order_key(s[i]); }, a.n, k, a.first, a.last, ab,
                              [&](int i, int, int place, bool in) {
                                  if (in) sel[place] = i;
                              }))
            return;
    } else {
        if (block_aborted(a.abort)) return;
        auto key = [&](int i) -> uint32_t {
            return i < a.first || i >= a.n - a.last ? 0xFFFFFFFFu : order_key(s[i]);
        };
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
    if (a.n <= CHOOSE_MAX) {
        hipLaunchKernelGGL(k_kv8_choose, dim3(a.p.nKV, a.M), dim3(1024), 0, st, a);
        return hipGetLastError();
    }
    int P = 1;
    while (P < a.G && P < 16) P *= 2;
    const int rpt = 16 / P, tiles = (a.M + rpt - 1) / rpt, nb = (a.n + 63) / 64;
    // the rows' tiles over further blocks while the launch is small
    int z = 1;
    while (z < tiles && nb * a.p.nKV * z < 512) z *= 2;
    const int per = (tiles + z - 1) / z;
    hipLaunchKernelGGL(k_kv8_score, dim3(nb, a.p.nKV, (tiles + per - 1) / per), dim3(256), 0, st, a, P,
                       per);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const dim3 flat(a.M * a.p.nKV);
    if (a.n <= 1024) hipLaunchKernelGGL((k_kv8_topk<256, 4>), flat, dim3(256), 0, st, a);
    else if (a.n <= 4096) hipLaunchKernelGGL((k_kv8_topk<1024, 4>), flat, dim3(1024), 0, st, a);
    else if (a.n <= 16384) hipLaunchKernelGGL((k_kv8_topk<1024, 16>), flat, dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((k_kv8_topk<1024, 0>), flat, dim3(1024), 0, st, a);
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------- evict
// One block a head: the `keep` greatest masses, the first and last blocks above all others; the
// table and the masses split in two, each part in its old order.  R as above.  65 blocks a head 3.5 us,
// 2047 7 us, bound as the choice of scores is.
template <int NT, int R>
__global__ __launch_bounds__(NT) void k_kv8_evict(Kv8Pool p, int n, int keep, int first, int last,
                                                  const float* __restrict__ mass_in,
                                                  int32_t* __restrict__ table_out,
                                                  float* __restrict__ mass_out, const int* abort) {
    const size_t row = (size_t)blockIdx.x * p.stride;
    const float* m = mass_in + row;
    const int32_t* tab = p.table + row;
    if constexpr (R > 0) {
        const int ab = abort ? *abort : 0;
        float mr[R];
        int32_t tr[R];
        auto key = [&](int i, int r) {  // (of no blocks: unused)
            mr[r] = m[max(i, 0)];
            tr[r] = tab[max(i, 0)];
            return order_key(mr[r]);
        };
        if (!pick_keys<NT, R>(key, n, keep, first, last, ab, [&](int i, int r, int place, bool in) {
                const int at = in ? place : keep + place;
                table_out[row + at] = tr[r];
                mass_out[row + at] = in ? mr[r] : 0.0f;
            }))
            return;
    } else {
        if (block_aborted(abort)) return;
        auto key = [&](int i) -> uint32_t {
            return i < first || i >= n - last ? 0xFFFFFFFFu : order_key(m[i]);
        };
        uint32_t thr = 0xFFFFFFFFu;  // keep 0: nothing stays
        int take = 0;
        if (keep > 0) kth_key<NT>(key, n, keep, thr, take);
        split_by_key<NT>(key, n, thr, take, [&](int i, int place, bool in) {
            const int at = in ? place : keep + place;
            table_out[row + at] = tab[i];
            mass_out[row + at] = in ? m[i] : 0.0f;
        });
    }
    for (int i = n + threadIdx.x; i < p.stride; i += NT) {
        table_out[row + i] = tab[i];
        mass_out[row + i] = 0.0f;
    }
}

hipError_t launch_kv8_evict(const Kv8Pool& p, int n, int keep, int first, int last,
                            const float* mass_in, int32_t* table_out, float* mass_out,
                            const int* abort, hipStream_t st) {
    auto go = [&](auto kernel, int threads) {
        hipLaunchKernelGGL(kernel, dim3(p.nKV), dim3(threads), 0, st, p, n, keep, first, last, mass_in,
                           table_out, mass_out, abort);
    };
    if (n <= 256) go(k_kv8_evict<256, 1>, 256);
    else if (n <= 1024) go(k_kv8_evict<256, 4>, 256);
    else if (n <= 4096) go(k_kv8_evict<1024, 4>, 1024);
    else if (n <= 16384) go(k_kv8_evict<1024, 16>, 1024);
    else go(k_kv8_evict<1024, 0>, 1024);
    return hipGetLastError();
}
