// kv8_attn.hip -- attention over the 8-bit KV cache: sealed pages, then the fp16 ring's rows.
//
// softmax(q k^T / sqrt(128)) v in one pass over the keys with a running maximum and sum.  A unit is
// one page or 64 rows of the ring; a part is a run of units that one block takes; the parts of a row
// and head are joined by k_kv8_combine.  Scores are kept in log2 units (scale * log2 e).
#include <algorithm>

#include "mj_device.h"
#include "mj_kv8.h"

#define HD 128
#define LOG2E 1.44269504088896341f

// max / sum over lanes i, i ^ 16, i ^ 32, i ^ 48 (the same bits in every lane)
__device__ __forceinline__ float x4_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float x4_sum(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Four codes (bytes, code + 128) to four halves, exactly: a byte under the exponent of 1024 is 1024 +
// code + 128, and 1152 is taken off.
__device__ __forceinline__ void codes4(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const h2v off = {(_Float16)1152.0f, (_Float16)1152.0f};
    const uint32_t a = __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u);
    const uint32_t b = __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u);
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2v, a) - off);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2v, b) - off);
}
// 16 codes to the two 8-half operands they make
__device__ __forceinline__ void codes16(const u4v w, u4v& a, u4v& b) {
    uint32_t x, y;
    codes4(w.x, x, y);
    a.x = x;
    a.y = y;
    codes4(w.y, x, y);
    a.z = x;
    a.w = y;
    codes4(w.z, x, y);
    b.x = x;
    b.y = y;
    codes4(w.w, x, y);
    b.z = x;
    b.w = y;
}

__device__ __forceinline__ int unit_page(const Kv8AttnArgs& a, int g, int row, int u) {
    int i = u;
    if (a.sel) {
        i = a.sel[((size_t)row * a.p.nKV + g) * a.n_sel + u];
        if ((unsigned)i >= (unsigned)a.n) return -1;
    }
    const int pg = a.p.table[(size_t)g * a.p.stride + i];
    return (unsigned)pg < (unsigned)a.p.n_pages ? pg : -1;
}

// The state of one tile of 16 query vectors.  Lane (ln, lq): query vector ln's maximum and sum (lq's
// share of it), and outputs of vectors 4 lq + r, dims 16 dt + ln.
struct Tile {
    float m, l;
    f4 o[8];
};

// One unit's scores of a tile: D lane (ln, lq) of K Q^T = vector ln against tokens 16 kt + 4 lq + r.
// K operand s holds dims 64 (s / 2) + 16 lq + 8 (s % 2) + 0 .. 7, as Q's does.
template <bool RING>
__device__ __forceinline__ void tile_unit(Tile& T, const u4v q[4], const u4v* Kf, const u4v* Vf,
                                          int lane, float ksc, float vsc, uint64_t committed,
                                          uint64_t own, float2* rec) {
    const int ln = lane & 15, lq = lane >> 4;
    f4 S[4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
        S[kt] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < 4; ++s)
            S[kt] = mfma16x16x32(as_h8(Kf[(4 * kt + s) * 64 + lane]), as_h8(q[s]), S[kt]);
    }
    float m = -INFINITY;
    const uint64_t ok = committed | own;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float s = S[kt][r] * ksc;
            if (RING) s = (ok >> (16 * kt + 4 * lq + r)) & 1 ? s : -INFINITY;
            S[kt][r] = s;
            m = fmaxf(m, s);
        }
    m = fmaxf(T.m, x4_max(m));
    // nothing seen yet: any finite reference (a masked score still gives 0, a NaN stays one)
    const float ref = m == -INFINITY ? 0.0f : m;
    const float alpha = __builtin_amdgcn_exp2f(T.m - ref);
    T.m = m;
    float l = 0.0f;
    u4v pa[2];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
        float p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            p[r] = __builtin_amdgcn_exp2f(S[kt][r] - ref);
            l += p[r];
        }
        pa[kt >> 1][2 * (kt & 1)] = pack2(f2h(p[0]), f2h(p[1]));
        pa[kt >> 1][2 * (kt & 1) + 1] = pack2(f2h(p[2]), f2h(p[3]));
    }
    T.l = fmaf(T.l, alpha, l);
    if (rec) {
        const float lu = x4_sum(l);
        if (lq == 0) rec[ln] = make_float2(m, lu);
    }
    float al[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) al[r] = __shfl(alpha, 4 * lq + r, MJ_WAVE);
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
        f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 2; ++j)
            o = mfma16x16x32(as_h8(pa[j]), as_h8(Vf[(2 * dt + j) * 64 + lane]), o);
#pragma unroll
        for (int r = 0; r < 4; ++r) T.o[dt][r] = fmaf(o[r], vsc, T.o[dt][r] * al[r]);
    }
}

// Infinities and NaN among the V rows of the pass (a tree row's siblings must not see them: 0 times
// an infinity is a NaN) are left out of the products (staged as 0) and added here, for the rows that
// do attend to them; bad: the ring rows that hold any.
__device__ __forceinline__ void add_bad_rows(Tile& T, const u4v q[4], const u4v* Kf, int lane, float ksc,
                                          uint64_t ok, uint64_t bad, const uint16_t* vrow0,
                                          int slot0, int C) {
    const int ln = lane & 15, lq = lane >> 4;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
        if (!((bad >> (16 * kt)) & 0xFFFFu)) continue;
        f4 S = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < 4; ++s)
            S = mfma16x16x32(as_h8(Kf[(4 * kt + s) * 64 + lane]), as_h8(q[s]), S);
        const float ref = T.m == -INFINITY ? 0.0f : T.m;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int key = 16 * kt + 4 * lq + r;
            // -1: not attended
            const float p = (ok >> key) & 1 ? __builtin_amdgcn_exp2f(S[r] * ksc - ref) : -1.0f;
            for (int kq = 0; kq < 4; ++kq) {
                const int k = 16 * kt + 4 * kq + r;
                if (!((bad >> k) & 1)) continue;  // uniform
                int sl = slot0 + k;
                sl -= sl >= C ? C : 0;
                const uint16_t* vr = vrow0 + (size_t)sl * HD + ln;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float pv = __shfl(p, 16 * kq + 4 * lq + x, MJ_WAVE);
#pragma unroll
                    for (int dt = 0; dt < 8; ++dt) {
                        const float v = h2f(vr[16 * dt]);
                        if (!(fabsf(v) < INFINITY) && !(pv < 0.0f)) T.o[dt][x] += pv * v;
                    }
                }
            }
        }
    }
}

__device__ __forceinline__ u4v finite8(u4v v, bool& bad) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool b0 = (v[j] & 0x7C00u) == 0x7C00u, b1 = (v[j] & 0x7C000000u) == 0x7C000000u;
        bad |= b0 | b1;
        v[j] = (b0 ? 0u : v[j] & 0xFFFFu) | (b1 ? 0u : v[j] & 0xFFFF0000u);
    }
    return v;
}

// A 256-thread block takes part blockIdx.x of KV head blockIdx.z for 4 T tiles of query vectors
// (vector r * G + j: head j of the group, row r; where rows list their own blocks, the vectors of row
// blockIdx.y), T a wave.  Units are staged in LDS as the halves the matrix instructions take: K
// operand (kt, s) and V operand (dt, j), 1 KB each, a lane's 16 bytes at 16 * lane.
template <int T>
__global__ __launch_bounds__(256) void k_kv8_attn(Kv8AttnArgs a) {
    __shared__ __align__(16) u4v Kf[16 * 64];
    __shared__ __align__(16) u4v Vf[16 * 64];
    __shared__ int s_abort;
    __shared__ uint32_t s_bad[2][2];  // ring rows with an infinity or NaN in V, units in turn
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6, ln = lane & 15, lq = lane >> 4;
    const int part = blockIdx.x, g = blockIdx.z;
    const int row_y = a.sel ? blockIdx.y : 0;
    const int v0 = a.sel ? row_y * a.G : (int)blockIdx.y * 64 * T;    // first vector of the block
    const int vend = a.sel ? v0 + a.G : a.M * a.G;
    const int nv = a.M * a.G, nQ = a.p.nKV * a.G, C = (int)a.ring.C;
    const int ab = a.abort ? *a.abort : 0;
    if (t == 0) s_abort = ab;
    if (t < 4) s_bad[t >> 1][t & 1] = 0;
    Tile tl[T];
    u4v q[T][4];
    uint64_t anc[T];
#pragma unroll
    for (int i = 0; i < T; ++i) {
        const int v = v0 + 16 * (wv * T + i) + ln;
        const bool on = v < vend;
        const int r = on ? v / a.G : 0, h = on ? g * a.G + v - r * a.G : 0;
        const uint16_t* qp = a.q + (size_t)r * a.ldq + (size_t)h * HD;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            q[i][s] = *(const u4v*)(qp + 64 * (s >> 1) + 16 * lq + 8 * (s & 1));
            if (!on) q[i][s] = (u4v){0u, 0u, 0u, 0u};
        }
        anc[i] = on ? a.anc[r] : 0;
        tl[i].m = -INFINITY;
        tl[i].l = 0.0f;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) tl[i].o[dt] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    }
    __syncthreads();
    if (s_abort) return;
    const float sc2 = LOG2E * 0.08838834764831845f;  // log2 e / sqrt(128)
    const int u1 = min((part + 1) * a.upp, a.units);
    for (int u = part * a.upp; u < u1; ++u) {
        const bool ringu = u >= a.n_list;
        float ksc = sc2, vsc = 1.0f;
        int pg = 0;
        uint64_t committed = 0;
        int base = 0, slot_b = 0;  // ring row of the unit's first token, its slot
        if (!ringu) {
            pg = unit_page(a, g, row_y, u);
            if (pg < 0) continue;  // whole block
            ksc = a.p.ks[pg] * sc2;
            vsc = a.p.vs[pg];
            const u4v* kp = (const u4v*)(a.p.k + (size_t)pg * KV8_PAGE_BYTES);
            const u4v* vp = (const u4v*)(a.p.v + (size_t)pg * KV8_PAGE_BYTES);
            u4v kr[2], vr[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                kr[c] = kp[t + 256 * c];
                vr[c] = vp[t + 256 * c];
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int ch = t + 256 * c, f = ch >> 6;
                codes16(kr[c], Kf[(2 * f) * 64 + lane], Kf[(2 * f + 1) * 64 + lane]);
                codes16(vr[c], Vf[(2 * f) * 64 + lane], Vf[(2 * f + 1) * 64 + lane]);
            }
        } else {
            base = 64 * (u - a.n_list);
            const int rows = a.R + a.M;
            slot_b = a.slot0 + base;
            slot_b -= slot_b >= C ? C : 0;
            auto slot = [&](int k) {  // of row `base + k`, a row past the last taken as the last
                int s = a.slot0 + min(base + k, rows - 1);
                s -= s >= C ? C : 0;
                return ((size_t)g * C + s) * HD;
            };
            if (t < 2) s_bad[(u & 1) ^ 1][t] = 0;  // nobody reads or sets the other one's now
            if (a.R > base) committed = a.R - base >= 64 ? ~0ull : (1ull << (a.R - base)) - 1;
            u4v kr[4], vr[4];
            const int kg = t & 15, vd = t >> 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = t + 256 * i;
                kr[i] = *(const u4v*)(a.ring.k + slot(c >> 4) + 8 * (c & 15));
                vr[i] = *(const u4v*)(a.ring.v + slot(4 * kg + i) + 8 * vd);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = t + 256 * i, k = c >> 4, dg = c & 15;
                const bool on = base + k < rows;
                Kf[(4 * (k >> 4) + 2 * (dg >> 3) + (dg & 1)) * 64 + 16 * ((dg >> 1) & 3) + (k & 15)] =
                    on ? kr[i] : (u4v){0u, 0u, 0u, 0u};
                if (base + 4 * kg + i >= rows) vr[i] = (u4v){0u, 0u, 0u, 0u};
                bool bad = false;
                vr[i] = finite8(vr[i], bad);
                if (bad) atomicOr(&s_bad[u & 1][kg >> 3], 1u << ((4 * kg + i) & 31));
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int sh = 16 * (e & 1);
                const uint32_t x = pack2(vr[0][e >> 1] >> sh, vr[1][e >> 1] >> sh);
                const uint32_t y = pack2(vr[2][e >> 1] >> sh, vr[3][e >> 1] >> sh);
                const int d = 8 * vd + e, aa = kg >> 2;
                uint2* p = (uint2*)&Vf[(2 * (d >> 4) + (aa >> 1)) * 64 + 16 * (kg & 3) + (d & 15)];
                p[aa & 1] = make_uint2(x, y);
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < T; ++i) {
            const int tv = v0 + 16 * (wv * T + i);
            if (tv >= vend) continue;  // uniform
            if (!ringu) {
                float2* rec = a.rec ? a.rec + ((size_t)g * a.n + u) * nv + tv : nullptr;
                if (rec && tv + ln >= vend) rec = a.rec + (size_t)a.p.nKV * a.n * nv;  // (spare row)
                tile_unit<false>(tl[i], q[i], Kf, Vf, lane, ksc, vsc, 0, 0, rec);
            } else {
                const int d0 = base - a.R;  // own row of the unit's first token
                const uint64_t own = d0 >= 64 ? 0 : d0 >= 0 ? anc[i] >> d0 : d0 > -64 ? anc[i] << -d0 : 0;
                const bool on = tv + ln < vend;
                const uint64_t ok = on ? committed | own : 0;
                tile_unit<true>(tl[i], q[i], Kf, Vf, lane, ksc, vsc, ok, 0, nullptr);
                const uint64_t bad = s_bad[u & 1][0] | ((uint64_t)s_bad[u & 1][1] << 32);
                if (bad)
                    add_bad_rows(tl[i], q[i], Kf, lane, ksc, ok, bad,
                                 a.ring.v + (size_t)g * C * HD, slot_b, C);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < T; ++i) {
        const int tv = v0 + 16 * (wv * T + i);
        if (tv >= vend) continue;
        const float l = x4_sum(tl[i].l);
        const size_t pb = ((size_t)part * a.p.nKV + g) * nv + tv;
        if (lq == 0 && tv + ln < vend) a.ml[pb + ln] = make_float2(tl[i].m, l);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (tv + 4 * lq + r < vend) {
                float* op = a.opart + (pb + 4 * lq + r) * HD + ln;
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) op[16 * dt] = tl[i].o[dt][r];
            }
    }
}

// One 256-thread block a row and head: wave w takes parts w, w + 4, .. in turn (lane = two dims), the
// four sums are added in wave order.  A part that saw no key has maximum -inf and weight 0.
__global__ __launch_bounds__(256) void k_kv8_combine(Kv8AttnArgs a) {
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    const int nQ = a.p.nKV * a.G, nv = a.M * a.G;
    const int r = blockIdx.x / nQ, h = blockIdx.x % nQ, g = h / a.G, v = r * a.G + h % a.G;
    __shared__ float s_o[4][HD];
    __shared__ float s_l[4];
    __shared__ int s_abort;
    const int ab = a.abort ? *a.abort : 0;
    if (t == 0) s_abort = ab;
    const size_t step = (size_t)a.p.nKV * nv, at = (size_t)g * nv + v;
    float mx = -INFINITY;
    for (int c = lane; c < a.parts; c += 64) mx = fmaxf(mx, a.ml[at + c * step].x);
    mx = wave_max(mx);
    const float ref = mx == -INFINITY ? 0.0f : mx;
    float o0 = 0.0f, o1 = 0.0f, l = 0.0f;
    for (int c = wv; c < a.parts; c += 4) {
        const float2 ml = a.ml[at + c * step];
        const float2 o = *(const float2*)(a.opart + (at + c * step) * HD + 2 * lane);
        const float w = __builtin_amdgcn_exp2f(ml.x - ref);
        l = fmaf(ml.y, w, l);
        o0 = fmaf(o.x, w, o0);
        o1 = fmaf(o.y, w, o1);
    }
    s_o[wv][2 * lane] = o0;
    s_o[wv][2 * lane + 1] = o1;
    if (lane == 0) s_l[wv] = l;
    __syncthreads();
    if (s_abort) return;
    if (t >= 16) return;
    l = ((s_l[0] + s_l[1]) + s_l[2]) + s_l[3];
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key at all: zeros
    if (t == 0 && a.stat) a.stat[at] = make_float2(ref, inv);
    u4v ov;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int d = 8 * t + 2 * j;
        const float x = (((s_o[0][d] + s_o[1][d]) + s_o[2][d]) + s_o[3][d]) * inv;
        const float y = (((s_o[0][d + 1] + s_o[1][d + 1]) + s_o[2][d + 1]) + s_o[3][d + 1]) * inv;
        ov[j] = pack2(f2h(x), f2h(y));
    }
    if (a.out) *(u4v*)(a.out + (size_t)r * a.ldo + (size_t)h * HD + 8 * t) = ov;
    if (a.out_perm) {
        const int K = nQ * HD;
        emit_qx(ov, t, a.out_perm + (size_t)r * K, a.out_sum + (size_t)r * (K / 64), h * HD + 8 * t);
    }
}

// mass_out = mass_in + sum over the head's query vectors of the block's share of their softmax, a wave
// a block.
__global__ __launch_bounds__(256) void k_kv8_mass(Kv8AttnArgs a) {
    const int lane = threadIdx.x & 63, g = blockIdx.y, nv = a.M * a.G;
    const int i = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= a.n || aborted(a.abort)) return;
    const size_t at = (size_t)g * a.p.stride + i;
    const int pg = a.p.table[at];
    float s = 0.0f;
    if ((unsigned)pg < (unsigned)a.p.n_pages)
        for (int v = lane; v < nv; v += 64) {
            const float2 rc = a.rec[((size_t)g * a.n + i) * nv + v], st = a.stat[(size_t)g * nv + v];
            s = fmaf(rc.y * st.y, __builtin_amdgcn_exp2f((rc.x == -INFINITY ? 0.0f : rc.x) - st.x), s);
        }
    s = wave_sum(s);
    if (lane == 0) a.mass_out[at] = (a.mass_in ? a.mass_in[at] : 0.0f) + s;
}

size_t kv8_attn_plan(Kv8AttnArgs& a, bool mass, void* base) {
    a.n_list = a.n_sel > 0 ? a.n_sel : a.n;
    a.units = a.n_list + (a.R + a.M + KV8_B - 1) / KV8_B;
    const int nv = a.M * a.G;
    const int vb = a.n_sel > 0 ? a.G : nv;           // vectors a block column takes
    a.tiles = (vb + 15) / 16 > 4 ? 2 : 1;  // tiles a wave
    const int cols = a.n_sel > 0 ? a.M : (vb + 64 * a.tiles - 1) / (64 * a.tiles);
    int parts = std::max(1, 512 / (cols * a.p.nKV));
    parts = std::min(parts, a.units);
    a.upp = (a.units + parts - 1) / parts;
    a.parts = (a.units + a.upp - 1) / a.upp;
    size_t off = 0;
    auto take = [&](size_t bytes) {
        off = (off + 255) & ~(size_t)255;
        void* p = base ? (char*)base + off : nullptr;
        off += bytes;
        return p;
    };
    const size_t vecs = (size_t)a.p.nKV * nv;
    a.opart = (float*)take(vecs * a.parts * HD * 4);
    a.ml = (float2*)take(vecs * a.parts * 8);
    a.rec = mass ? (float2*)take((vecs * a.n + 16) * 8) : nullptr;
    a.stat = mass ? (float2*)take(vecs * 8) : nullptr;
    return off;
}

hipError_t launch_kv8_attn(const Kv8AttnArgs& a, hipStream_t st) {
    if (a.M < 1 || a.M > MJ_ROWS || a.ring.C >= ((int64_t)1 << 30) || a.units < 1)
        return hipErrorInvalidValue;
    const int nv = a.M * a.G, vb = a.n_sel > 0 ? a.G : nv;
    const int cols = a.n_sel > 0 ? a.M : (vb + 64 * a.tiles - 1) / (64 * a.tiles);
    const dim3 grid(a.parts, cols, a.p.nKV);
    if (a.tiles == 1) hipLaunchKernelGGL(k_kv8_attn<1>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_kv8_attn<2>, grid, dim3(256), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_kv8_combine, dim3(a.M * a.p.nKV * a.G), dim3(256), 0, st, a);
    e = hipGetLastError();
    if (e != hipSuccess || !a.rec) return e;
    hipLaunchKernelGGL(k_kv8_mass, dim3((a.n + 3) / 4, a.p.nKV), dim3(256), 0, st, a);
    return hipGetLastError();
}
