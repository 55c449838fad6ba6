// kv8_attn.hip -- attention over the 8-bit KV cache: sealed pages, then the fp16 ring's rows.
//
// softmax(q k^T / sqrt(128)) v in one pass over the keys with a running maximum and sum.  A unit is
// one page or 64 rows of the ring; a part is a run of units that one block takes; the parts of a row
// and head are joined by k_kv8_combine.  Scores are kept in log2 units (scale * log2 e).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "mj_device.h"
#include "mj_kv8.h"

#define HD 128
#define SC2 (1.44269504088896341f * 0.08838834764831845f)  // log2 e / sqrt(128)

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

__device__ __forceinline__ float lane_of(float v, int i) {  // lane i's value (i uniform)
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i));
}

__device__ __forceinline__ int page_of_list(const Kv8AttnArgs& a, int g, int i) {
    const int pg = a.p.table[(size_t)g * a.p.stride + i];
    return (unsigned)pg < (unsigned)a.p.n_pages ? pg : -1;
}
__device__ __forceinline__ int unit_page(const Kv8AttnArgs& a, int g, int row, int u) {
    if (!a.sel) return page_of_list(a, g, u);
    const int i = a.sel[((size_t)row * a.p.nKV + g) * a.n_sel + u];
    return (unsigned)i < (unsigned)a.n ? page_of_list(a, g, i) : -1;
}

// The state of one tile of 16 query vectors.  Lane (ln, lq): query vector ln's maximum and sum (lq's
// share of it), and outputs of vectors 4 lq + r, dims 16 dt + ln.
struct Tile {
    float m, l;
    f4 o[8];
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) o[dt] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    }
};

typedef float f2v __attribute__((ext_vector_type(2)));

// What a unit's codes stand for: ksc, the factor of its raw scores to log2 units; lv, log2 of its V
// scale (at least LV_MIN, that of a block of the least fp16 number; a block of zeros has none) less
// LV_TOP; ilv, 1 / V scale.
struct Scales {
    float ksc, lv, ilv;
};
#define LV_MIN -31.0f
#define LV_TOP 3.0f
__device__ __forceinline__ float log2_scale(float vs) {  // (a NaN stays one)
    const float l = __builtin_amdgcn_logf(vs);
    return l < LV_MIN ? LV_MIN : l;
}

// Softmax of one unit's scores against the running state.  S: lane (ln, lq) holds vector ln against
// tokens 16 kt + 4 lq + r, without the scale ksc >= 0; masked ones -inf.  The weights come out times
// the unit's V scale, w = exp2(s + lv - m + LIFT), so the products with V accumulate in the state without a
// step between; m is the running reference of s + lv.  It follows the maximum only where that is more
// than 2^SLACK above it: outputs are rescaled once or twice a part, not at every unit.  w is rounded to
// fp16, as the two A operands of the product with V (their k slot 8 lq + u is token 32 j + 4 lq + u,
// then 32 j + 16 + 4 lq + u - 4): half a step, 2^-11 of a weight.  It is lifted by 2^LIFT before, as
// high as fp16 goes (SLACK + LIFT = 15): fp16's steps widen below 2^-14, which is 2^-23 of the reference,
// so a weight times V scale is off by at most 2^-34 of the part's greatest one (unlifted by 2^-25: of
// pages with V scales 2^26 apart the smaller one's values were lost).  The factor is the same in outputs
// and sums and leaves with the division.  The sum takes the weights before the rounding.  lu: the unit's
// sum of exp2(s - m + LIFT), this lane's share.
#define SLACK 6.0f
#define LIFT 9.0f
// Scores past FAR, whose steps in fp32 are an eighth and more: s + lv would lose lv, and a weight's one
// fma differs from the rounded s by up to thousands (weights of infinity or 0).  There m is at least the
// rounded s itself, and move_ref takes it off the rounded scores, exactly for those near it, in the
// branch that it has for moving.  A weight is then up to 2^(lv + LIFT): below 2^15.1 for a sealed block
// (scale 65504 / 127 at most), which is what LV_TOP is for.
#define FAR 1048576.0f

// The reference moved, for T tiles at once (one branch; the weights of one tile can then be formed
// under the products of another); c: what makes exp2(fma(S, ksc, c)) of vector ln's scores its weights.
template <int T>
__device__ __forceinline__ void move_ref(Tile* tl, f4 (*S)[4], Scales u, float* c) {
    float x[T], m[T], ref[T];
    bool rare = false;
#pragma unroll
    for (int i = 0; i < T; ++i) {
        x[i] = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            x[i] = fmaxf(fmaxf(x[i], S[i][kt][0]), S[i][kt][1]);
            x[i] = fmaxf(fmaxf(x[i], S[i][kt][2]), S[i][kt][3]);
        }
        x[i] = x4_max(x[i]);
        m[i] = fmaf(x[i], u.ksc, u.lv);
        rare |= (m[i] > tl[i].m + SLACK) | (fabsf(m[i]) > FAR);
        ref[i] = tl[i].m;
    }
    if (__any(rare)) {
        const int lq = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int i = 0; i < T; ++i) {
            const float s = product(x[i], u.ksc);
            const bool far = fabsf(m[i]) > FAR && s > -INFINITY;  // (-inf: every score is masked)
            const float mn = fmaxf(tl[i].m, far ? s : m[i]);
            // (both may be -inf)
            const float alpha = tl[i].m == mn ? 1.0f : __builtin_amdgcn_exp2f(tl[i].m - mn);
            tl[i].m = mn;
            tl[i].l *= alpha;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float al = __shfl(alpha, 4 * lq + r, MJ_WAVE);
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) tl[i].o[dt][r] *= al;
            }
            ref[i] = far ? 0.0f : mn;
            if (!__any(far)) continue;
            const float inv = 1.0f / u.ksc;  // (far scores have no ksc of 0)
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    S[i][kt][r] = far ? (product(S[i][kt][r], u.ksc) - mn) * inv : S[i][kt][r];
        }
    }
#pragma unroll
    for (int i = 0; i < T; ++i)
        // no key seen: any finite reference (a masked score still gives 0, a NaN stays one)
        c[i] = u.lv + LIFT - (ref[i] == -INFINITY ? 0.0f : ref[i]);
}
__device__ __forceinline__ void weights(Tile& T, const f4 S[4], Scales u, float c, u4v pa[2], float& lu) {
    lu = 0.0f;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f2v p = {__builtin_amdgcn_exp2f(fmaf(S[kt][2 * h], u.ksc, c)),
                           __builtin_amdgcn_exp2f(fmaf(S[kt][2 * h + 1], u.ksc, c))};
            lu += p.x;
            lu += p.y;
            pa[kt >> 1][2 * (kt & 1) + h] =
                __builtin_bit_cast(uint32_t, __builtin_convertvector(p, h2v));
        }
    lu *= u.ilv;
    T.l += lu;
}

// Infinities and NaN among the V rows of the pass (a tree row's siblings must not see them: 0 times
// an infinity is a NaN) are left out of the products (staged as 0) and added here to the outputs of
// the vectors that attend to them, whatever their weights (which are above 0, if not in fp32).  bad:
// the unit's rows that hold any, ok: those that vector ln attends.
__device__ __forceinline__ void add_bad_rows(Tile& T, int lane, uint64_t ok, uint64_t bad,
                                             const uint16_t* vrow0, int slot0, int C) {
    const int ln = lane & 15, lq = lane >> 4;
#pragma unroll 1
    for (; bad; bad &= bad - 1) {
        const int k = __builtin_ctzll(bad);
        const uint32_t att = (uint32_t)__ballot((ok >> k) & 1) >> (4 * lq);  // of vectors 4 lq + x
        int sl = slot0 + k;
        sl -= sl >= C ? C : 0;
        const uint16_t* vr = vrow0 + (size_t)sl * HD + ln;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            const float v = h2f(vr[16 * dt]);
            const float e = fabsf(v) < INFINITY ? 0.0f : v;
#pragma unroll
            for (int x = 0; x < 4; ++x) T.o[dt][x] += (att >> x) & 1 ? e : 0.0f;
        }
    }
}

// Query vector v of KV head g (head j of the group, row r: v = r * G + j) as the B operand: operand s
// holds dims 64 (s / 2) + 16 lq + 8 (s % 2) + 0 .. 7, as the K operands do.  Lanes without a vector
// (on false) take the head's first, unused.
__device__ __forceinline__ void load_q(const Kv8AttnArgs& a, int g, int v, bool on, u4v q[4]) {
    const int lq = (threadIdx.x & 63) >> 4;
    const int r = on ? v / a.G : 0, h = on ? g * a.G + v - r * a.G : g * a.G;
    const uint16_t* qp = a.q + (size_t)r * a.ldq + (size_t)h * HD;
#pragma unroll
    for (int s = 0; s < 4; ++s) q[s] = *(const u4v*)(qp + 64 * (s >> 1) + 16 * lq + 8 * (s & 1));
}

// 64 rows of the ring, base .. base + 63 of the call's open rows, as the operands of a unit in LDS: K
// operand (kt, s) and V operand (dt, j), 1 KB each, a lane's 16 bytes at 16 * lane.  V is turned four
// tokens by eight dims at a time.  Rows past the last are zeros; bad: the rows with an infinity or
// NaN in V (set here, cleared before).
template <int NT>
__device__ __forceinline__ void stage_ring(const Kv8AttnArgs& a, int g, int base, u4v* Kf, u4v* Vf,
                                           uint32_t* bad) {
    const int t = threadIdx.x, rows = a.R + a.M, C = (int)a.ring.C;
    auto slot = [&](int k) {  // of row `base + k`, a row past the last taken as the last
        int s = a.slot0 + min(base + k, rows - 1);
        s -= s >= C ? C : 0;
        return ((size_t)g * C + s) * HD;
    };
    constexpr int NK = 1024 / NT, NV = 256 / NT > 0 ? 256 / NT : 1;
    u4v kr[NK], vr[NV][4];
#pragma unroll
    for (int i = 0; i < NK; ++i) {
        const int c = t + NT * i;
        kr[i] = *(const u4v*)(a.ring.k + slot(c >> 4) + 8 * (c & 15));
    }
    const bool vt = NT <= 256 || t < 256;
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = (t + NT * n) & 255;
            vr[n][i] = *(const u4v*)(a.ring.v + slot(4 * (c & 15) + i) + 8 * (c >> 4));
        }
#pragma unroll
    for (int i = 0; i < NK; ++i) {
        const int c = t + NT * i, k = c >> 4, dg = c & 15;
        Kf[(4 * (k >> 4) + 2 * (dg >> 3) + (dg & 1)) * 64 + 16 * ((dg >> 1) & 3) + (k & 15)] =
            base + k < rows ? kr[i] : (u4v){0u, 0u, 0u, 0u};
    }
    if (!vt) return;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int c = t + NT * n, kg = c & 15, vd = c >> 4, aa = kg >> 2;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (base + 4 * kg + i >= rows) vr[n][i] = (u4v){0u, 0u, 0u, 0u};
            bool b = false;
            vr[n][i] = finite8(vr[n][i], b);
            if (b) atomicOr(&bad[kg >> 3], 1u << ((4 * kg + i) & 31));
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int sh = 16 * (e & 1), d = 8 * vd + e;
            const uint32_t x = pack2(vr[n][0][e >> 1] >> sh, vr[n][1][e >> 1] >> sh);
            const uint32_t y = pack2(vr[n][2][e >> 1] >> sh, vr[n][3][e >> 1] >> sh);
            uint2* p = (uint2*)&Vf[(2 * (d >> 4) + (aa >> 1)) * 64 + 16 * (kg & 3) + (d & 15)];
            p[aa & 1] = make_uint2(x, y);
        }
    }
}

// The rows of a ring unit that vector v attends.
__device__ __forceinline__ uint64_t ring_mask(const Kv8AttnArgs& a, int base, int v, bool on) {
    const uint64_t anc = a.anc[on ? v / a.G : 0];
    uint64_t committed = 0;
    if (a.R > base) committed = a.R - base >= 64 ? ~0ull : (1ull << (a.R - base)) - 1;
    const int d0 = base - a.R;  // own row of the unit's first token
    const uint64_t own = d0 >= 64 ? 0 : d0 >= 0 ? anc >> d0 : d0 > -64 ? anc << -d0 : 0;
    return on ? committed | own : 0;
}

// A tile against a ring unit staged in LDS; ok: the rows that vector ln attends.
__device__ __forceinline__ void ring_unit(Tile& tl, const u4v q[4], const u4v* Kf, const u4v* Vf,
                                          int lane, uint64_t ok) {
    const uint64_t okl = ok >> (4 * (lane >> 4));  // token 16 kt + 4 lq + r: bit 16 kt + r
    f4 S[1][4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
        const uint32_t w = (uint32_t)(okl >> (32 * (kt >> 1))) >> (16 * (kt & 1));
        S[0][kt] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < 4; ++s)
            S[0][kt] = mfma16x16x32(as_h8(Kf[(4 * kt + s) * 64 + lane]), as_h8(q[s]), S[0][kt]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            S[0][kt][r] = (w >> r) & 1 ? S[0][kt][r] : -INFINITY;
        __builtin_amdgcn_sched_barrier(0);  // (all operands ahead of the products: 100 registers more)
    }
    const Scales u{SC2, -LV_TOP, 1.0f};
    u4v pa[2];
    float c, lu;
    move_ref<1>(&tl, S, u, &c);
    weights(tl, S[0], u, c, pa, lu);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            tl.o[dt] = mfma16x16x32(as_h8(pa[j]), as_h8(Vf[(2 * dt + j) * 64 + lane]), tl.o[dt]);
            if (dt % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
}

__device__ __forceinline__ void write_part(const Kv8AttnArgs& a, int part, int g, int tv, int vend,
                                           const Tile& T) {
    const int lane = threadIdx.x & 63, ln = lane & 15, lq = lane >> 4, nv = a.M * a.G;
    const float l = x4_sum(T.l);
    const size_t pb = ((size_t)part * a.p.nKV + g) * nv + tv;
    if (lq == 0 && tv + ln < vend) a.ml[pb + ln] = make_float2(T.m, l);
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (tv + 4 * lq + r < vend) {
            float* op = a.opart + (pb + 4 * lq + r) * HD + ln;
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) op[16 * dt] = T.o[dt][r];
        }
}

// The query vectors v0 .. vend - 1 of a block of `per` at most, column blockIdx.y; with lists of their
// own, of one row.
__device__ __forceinline__ void block_vectors(const Kv8AttnArgs& a, int per, int& row, int& v0,
                                              int& vend) {
    const int cols = a.sel ? (a.G + per - 1) / per : 1;
    row = a.sel ? blockIdx.y / cols : 0;
    v0 = a.sel ? row * a.G + per * (blockIdx.y % cols) : per * (int)blockIdx.y;
    vend = min(a.sel ? row * a.G + a.G : a.M * a.G, v0 + per);
}

// A part of the ring: units part * upr on, upr of them (64 rows each of the call's open ones), one at a
// time; the block of NW waves stages a unit and takes the query vectors v0 .. vend - 1 a tile a wave,
// in further rounds where they are more.  lds: 32 KB.
template <int NW>
__device__ __forceinline__ void ring_part(const Kv8AttnArgs& a, int part, int g, int v0, int vend,
                                          u4v* lds, uint32_t* s_bad, int* s_abort) {
    const int t = threadIdx.x, lane = t & 63, ln = lane & 15, C = (int)a.ring.C;
    const int u0 = part * a.upr, u1 = min(u0 + a.upr, a.ring_units);
    const int ab = a.abort ? *a.abort : 0;  // thread 0's reading decides for the block
    u4v* Kf = lds;
    u4v* Vf = Kf + 1024;
    auto stage = [&](int u) {
        if (t < 2) s_bad[t] = 0;
        __syncthreads();
        stage_ring<64 * NW>(a, g, KV8_B * u, Kf, Vf, s_bad);
        if (t == 0) *s_abort = ab;
        __syncthreads();
        return *s_abort != 0;
    };
    auto take = [&](int u, int tv, const u4v* q, Tile& tl) {
        const uint64_t bad = s_bad[0] | ((uint64_t)s_bad[1] << 32);
        const uint64_t ok = ring_mask(a, KV8_B * u, tv + ln, tv + ln < vend);
        ring_unit(tl, q, Kf, Vf, lane, ok);
        if (bad) {
            int sb = a.slot0 + KV8_B * u;
            sb -= sb >= C ? C : 0;
            add_bad_rows(tl, lane, ok, bad, a.ring.v + (size_t)g * C * HD, sb, C);
        }
    };
    if (a.upr == 1) {  // staged once (one loop for both forms cost a short context 0.8 us)
        if (stage(u0)) return;
        for (int tv = v0 + 16 * (t >> 6); tv < vend; tv += 16 * NW) {
            u4v q[4];
            load_q(a, g, tv + ln, tv + ln < vend, q);
            Tile tl;
            tl.clear();
            take(u0, tv, q, tl);
            write_part(a, part, g, tv, vend, tl);
        }
        return;
    }
    for (int r0 = v0; r0 < vend; r0 += 16 * NW) {
        const int tv = r0 + 16 * (t >> 6);
        u4v q[4];
        load_q(a, g, tv + ln, tv + ln < vend, q);
        Tile tl;
        tl.clear();
        for (int u = u0; u < u1; ++u) {
            __syncthreads();  // everyone is done with the unit before
            if (stage(u)) return;
            if (tv < vend) take(u, tv, q, tl);
        }
        if (tv < vend) write_part(a, part, g, tv, vend, tl);
    }
}

// A tile's products with a unit in LDS: all K operands are requested before the first product and all V
// operands before the softmax (left to itself the compiler waits for each read in turn).
template <int T>
__device__ __forceinline__ void staged_unit(Tile* tl, const u4v (*q)[4], const u4v* Kf, const u4v* Vf,
                                            int lane, Scales u, float2* const* rec) {
    f4 S[T][4];
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) S[i][kt] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    {
        u4v k[16];
#pragma unroll
        for (int f = 0; f < 16; ++f) k[f] = Kf[f * 64 + lane];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int i = 0; i < T; ++i)
                    S[i][kt] = mfma16x16x32(as_h8(k[4 * kt + s]), as_h8(q[i][s]), S[i][kt]);
    }
    u4v v[16];
#pragma unroll
    for (int f = 0; f < 16; ++f) v[f] = Vf[f * 64 + lane];
    __builtin_amdgcn_sched_barrier(0);
    float c[T];
    move_ref<T>(tl, S, u, c);
    u4v pa[T][2];
#pragma unroll
    for (int i = 0; i < T; ++i) {
        float lu;
        weights(tl[i], S[i], u, c[i], pa[i], lu);
        if (rec[i]) {
            lu = x4_sum(lu);
            if (lane < 16) *rec[i] = make_float2(tl[i].m, lu);
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int dt = 0; dt < 8; ++dt)
#pragma unroll
            for (int i = 0; i < T; ++i)
                tl[i].o[dt] = mfma16x16x32(as_h8(pa[i][j]), as_h8(v[2 * dt + j]), tl[i].o[dt]);
}

// Pages shared: a block of NW waves takes a run of pages for NW T tiles of query vectors, T a wave.  A
// page is turned to halves once, by the whole block, and read from LDS by its waves; two pages are in
// LDS and one in registers on its way, one barrier a page.  The first blocks take the ring's
// parts; rows with lists of their own (a.sel) as below.  64 rows of 16 heads over 65500 tokens: 47 us,
// 0.73 PFLOP/s, the matrix units busy 38% of the time and the VALU 51% (the softmax, the codes), one
// after the other, as all waves run the same phase between two barriers.  17 rows over 32000 tokens with
// masses 17.6 us: eight pages a block, each a barrier and a chain of products, softmax and products that
// its few waves do not cover (a second page on its way, half the LDS reads, or the next page's scores
// under a page's softmax change nothing).
template <int T, int NW, bool MASS>
__global__ __launch_bounds__(64 * NW) void k_kv8_attn_shared(Kv8AttnArgs a) {
    constexpr int NT = 64 * NW, NR = 512 / NT;
    extern __shared__ __align__(16) u4v lds[];  // two pages: K operands, V operands
    __shared__ int s_abort;
    __shared__ uint32_t s_bad[2];
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6, ln = lane & 15;
    const int part = blockIdx.x, g = blockIdx.z, nv = a.M * a.G;
    int row, v0, vend;
    block_vectors(a, 16 * NW * T, row, v0, vend);
    if (part < a.ring_parts) {
        ring_part<NW>(a, part, g, v0, vend, lds, s_bad, &s_abort);
        return;
    }
    const int ab = a.abort ? *a.abort : 0;
    Tile tl[T];
    u4v q[T][4];
    const bool idle = v0 + 16 * wv * T >= vend;  // the wave has no vector: it stages only
    const int u0 = (part - a.ring_parts) * a.upp, u1 = min(u0 + a.upp, a.n_list);
    u4v kr[NR], vr[NR];
    auto request = [&](int pg) {
        const u4v* kp = (const u4v*)(a.p.k + (size_t)pg * KV8_PAGE_BYTES);
        const u4v* vp = (const u4v*)(a.p.v + (size_t)pg * KV8_PAGE_BYTES);
#pragma unroll
        for (int c = 0; c < NR; ++c) {
            kr[c] = kp[t + NT * c];
            vr[c] = vp[t + NT * c];
        }
    };
    auto stage = [&](int b) {
        u4v* Kf = lds + b * 2048;
        u4v* Vf = Kf + 1024;
#pragma unroll
        for (int c = 0; c < NR; ++c) {
            const int f = (t + NT * c) >> 6;
            codes16(kr[c], Kf[(2 * f) * 64 + lane], Kf[(2 * f + 1) * 64 + lane]);
            codes16(vr[c], Vf[(2 * f) * 64 + lane], Vf[(2 * f + 1) * 64 + lane]);
        }
    };
    for (int ub = u0; ub < u1; ub += 64) {
        const int pl = ub + lane < u1 ? unit_page(a, g, row, ub + lane) : -1;
        if (ub == u0) {
#pragma unroll
            for (int i = 0; i < T; ++i) {
                const int v = v0 + 16 * (wv * T + i) + ln;
                load_q(a, g, v, v < vend, q[i]);
                tl[i].clear();
            }
        }
        uint64_t todo = __ballot(pl >= 0);  // the same in every wave
        int cur = todo ? __builtin_ctzll(todo) : -1, nxt = -1, b = 0;
        if (cur >= 0) {
            request(__builtin_amdgcn_readlane(pl, cur));
            todo &= todo - 1;
            nxt = todo ? __builtin_ctzll(todo) : -1;
        }
        const float ksl = (pl >= 0 ? a.p.ks[pl] : 0.0f) * SC2;
        const float lg = log2_scale(pl >= 0 ? a.p.vs[pl] : 0.0f), lvl = lg - LV_TOP;
        const float ill = __builtin_amdgcn_exp2f(-lg);
        if (t == 0) s_abort = ab;
        if (ub != u0) __syncthreads();  // the batch before is done with
        if (cur >= 0) stage(0);
        if (nxt >= 0) request(__builtin_amdgcn_readlane(pl, nxt));
        for (bool first = true; cur >= 0; first = false) {
            todo &= todo - 1;
            const int n2 = todo ? __builtin_ctzll(todo) : -1;
            __syncthreads();  // page cur is staged; everyone is done with the one before
            if (first && s_abort) return;
            if (nxt >= 0) {
                stage(b ^ 1);
                if (n2 >= 0) request(__builtin_amdgcn_readlane(pl, n2));
            }
            if (!idle) {
                const u4v* Kf = lds + b * 2048;
                float2* rec[T];
#pragma unroll
                for (int i = 0; i < T; ++i) {
                    const int v = v0 + 16 * (wv * T + i) + ln;
                    rec[i] = !MASS      ? nullptr
                             : v < vend ? a.rec + ((size_t)g * a.n + ub + cur) * nv + v
                                        : a.rec + (size_t)a.p.nKV * a.n * nv + ln;  // a spare row
                }
                staged_unit<T>(tl, q, Kf, Kf + 1024, lane,
                               Scales{lane_of(ksl, cur), lane_of(lvl, cur), lane_of(ill, cur)}, rec);
            }
            cur = nxt;
            nxt = n2;
            b ^= 1;
        }
    }
#pragma unroll
    for (int i = 0; i < T; ++i) {
        const int tv = v0 + 16 * (wv * T + i);
        if (tv < vend) write_part(a, part, g, tv, vend, tl[i]);
    }
}

// Pages of P waves' own: every P waves of the block take pages for themselves, T tiles of query vectors
// each, straight into registers: a page's bytes lie in the order of the operands, so a lane's 16 bytes
// are two of them, turned to halves once for all T tiles.  (The P waves ask for a page at about the
// same time; it comes from memory once.)  A wave's next K goes out behind its scores, its next V behind
// its output products; the page numbers and scales of 64 pages come with one request a lane each.  The
// waves are joined in LDS.  The first blocks take the ring's parts.  Where rows list their own blocks
// (a.sel), blockIdx.y is a row and a share of its heads.  Bound by memory: one row over 131000 tokens
// of 4 heads, 134 MB, in 23 us (5.8 TB/s).
template <int T, int P, int NW, bool MASS>
__global__ __launch_bounds__(64 * NW) void k_kv8_attn_own(Kv8AttnArgs a) {
    constexpr int NT = 64 * NW, NG = NW / P;
    extern __shared__ __align__(16) u4v lds[];
    __shared__ int s_abort;
    __shared__ uint32_t s_bad[2];
    __shared__ float s_m[T][NW][16], s_l[NW][16];
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6, ln = lane & 15, lq = lane >> 4;
    const int part = blockIdx.x, g = blockIdx.z, nv = a.M * a.G, pr = wv % P;
    int row, v0, vend;
    block_vectors(a, 16 * T * P, row, v0, vend);
    if (part < a.ring_parts) {
        ring_part<NW>(a, part, g, v0, vend, lds, s_bad, &s_abort);
        return;
    }
    const int vw = v0 + 16 * T * pr;  // the wave's vectors
    const int ab = a.abort ? *a.abort : 0;
    Tile tl[T];
    u4v q[T][4];
    const int up = (part - a.ring_parts) * a.upp;
    const int u0 = up + wv / P, u1 = P > 1 && vw >= vend ? 0 : min(up + a.upp, a.n_list);
    for (int ub = u0; ub < u1 || ub == u0; ub += 64 * NG) {
        const int ul = ub + NG * lane;  // lane's unit
        const int pl = ul < u1 ? unit_page(a, g, row, ul) : -1;
        if (ub == u0) {
#pragma unroll
            for (int i = 0; i < T; ++i) {
                load_q(a, g, vw + 16 * i + ln, vw + 16 * i + ln < vend, q[i]);
                tl[i].clear();
            }
        }
        uint64_t todo = __ballot(pl >= 0);
        u4v kr[8], vr[8];
        auto request_k = [&](int i) {
            const u4v* p = (const u4v*)(a.p.k + (size_t)__builtin_amdgcn_readlane(pl, i) * KV8_PAGE_BYTES);
#pragma unroll
            for (int f = 0; f < 8; ++f) kr[f] = p[64 * f + lane];
        };
        auto request_v = [&](int i) {
            const u4v* p = (const u4v*)(a.p.v + (size_t)__builtin_amdgcn_readlane(pl, i) * KV8_PAGE_BYTES);
#pragma unroll
            for (int f = 0; f < 8; ++f) vr[f] = p[64 * f + lane];
        };
        int i0 = todo ? __builtin_ctzll(todo) : -1;
        if (i0 >= 0) {
            request_k(i0);
            request_v(i0);
        }
        const float ksl = (pl >= 0 ? a.p.ks[pl] : 0.0f) * SC2;
        const float lg = log2_scale(pl >= 0 ? a.p.vs[pl] : 0.0f), lvl = lg - LV_TOP;
        const float ill = __builtin_amdgcn_exp2f(-lg);
        auto step = [&](int i, int nx, auto more) {  // page i; page nx requested behind it
            const Scales sc{lane_of(ksl, i), lane_of(lvl, i), lane_of(ill, i)};
            f4 S[T][4];
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
                for (int x = 0; x < T; ++x) S[x][kt] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    u4v k0, k1;
                    codes16(kr[2 * kt + j], k0, k1);
#pragma unroll
                    for (int x = 0; x < T; ++x)
                        S[x][kt] = mfma16x16x32(as_h8(k0), as_h8(q[x][2 * j]), S[x][kt]);
#pragma unroll
                    for (int x = 0; x < T; ++x)
                        S[x][kt] = mfma16x16x32(as_h8(k1), as_h8(q[x][2 * j + 1]), S[x][kt]);
                }
            }
            if constexpr (more.value) request_k(nx);
            float c[T];
            move_ref<T>(tl, S, sc, c);
            u4v pa[T][2];
#pragma unroll
            for (int x = 0; x < T; ++x) {
                float lu;
                weights(tl[x], S[x], sc, c[x], pa[x], lu);
                if constexpr (MASS) {
                    const int v = vw + 16 * x + ln;
                    lu = x4_sum(lu);
                    if (lq == 0 && v < vend)
                        a.rec[((size_t)g * a.n + ub + NG * i) * nv + v] = make_float2(tl[x].m, lu);
                }
            }
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) {
                u4v w0, w1;
                codes16(vr[dt], w0, w1);
#pragma unroll
                for (int x = 0; x < T; ++x)
                    tl[x].o[dt] = mfma16x16x32(as_h8(pa[x][0]), as_h8(w0), tl[x].o[dt]);
#pragma unroll
                for (int x = 0; x < T; ++x)
                    tl[x].o[dt] = mfma16x16x32(as_h8(pa[x][1]), as_h8(w1), tl[x].o[dt]);
            }
            if constexpr (more.value) request_v(nx);
        };
        // the last page apart: a request that is not used would be waited for at the join
        while (todo) {
            const int i = i0;
            todo &= todo - 1;
            if (!todo) break;
            i0 = __builtin_ctzll(todo);
            step(i, i0, std::true_type{});
        }
        if (i0 >= 0) step(i0, 0, std::false_type{});
    }
    // ---- the waves joined, a tile of each of the P together at a time: each wave scales its outputs to
    // its tile's maximum and puts them side by side in LDS (a lane's four vectors of a dim in 16
    // bytes), then a thread adds up one dim of four vectors, wave by wave.  (Every thread weighing
    // every wave's outputs read three times as much LDS: 1.7 us a tile.)
    f4* so = (f4*)lds;  // [NW][4][128]: vectors 4 y .. + 3 of dim d
#pragma unroll
    for (int x = 0; x < T; ++x)
        if (lq == 0) s_m[x][wv][ln] = tl[x].m;
    if (t == 0) s_abort = ab;
    __syncthreads();
    if (s_abort) return;
    auto put = [&](Tile& tt, int x) {
        const float l = x4_sum(tt.l);
        float m = s_m[x][pr][ln];
#pragma unroll
        for (int w = 1; w < NG; ++w) m = fmaxf(m, s_m[x][w * P + pr][ln]);
        const float f = __builtin_amdgcn_exp2f(tt.m - (m == -INFINITY ? 0.0f : m));
        if (lq == 0) s_l[wv][ln] = l * f;
        f4 fr;
#pragma unroll
        for (int r = 0; r < 4; ++r) fr[r] = __shfl(f, 4 * lq + r, MJ_WAVE);
        if (vw + 16 * x + 4 * lq < vend)
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) {
                f4 o = tt.o[dt];
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] *= fr[r];
                so[(wv * 4 + lq) * 128 + 16 * dt + ln] = o;
            }
    };
#pragma unroll 1
    for (int x = 0; x < T; ++x) {
        if (v0 + 16 * x >= vend) break;  // whole block
        if (x) __syncthreads();
        if (x == 0) put(tl[0], 0);
        if constexpr (T > 1)
            if (x == 1) put(tl[1], 1);
        __syncthreads();
        const size_t pb = ((size_t)part * a.p.nKV + g) * nv;
        if (t < 16 * P) {
            const int p = t >> 4, v = v0 + 16 * (T * p + x) + (t & 15);
            float l = 0.0f, m = s_m[x][p][t & 15];
#pragma unroll
            for (int w = 0; w < NG; ++w) {
                l += s_l[w * P + p][t & 15];
                m = fmaxf(m, s_m[x][w * P + p][t & 15]);
            }
            if (v < vend) a.ml[pb + v] = make_float2(m, l);
        }
#pragma unroll
        for (int e0 = 0; e0 < 512 * P; e0 += NT) {
            const int e = e0 + t, p = e >> 9, v = v0 + 16 * (T * p + x) + 4 * ((e >> 7) & 3), d = e & 127;
            if (v >= vend) continue;
            const f4* src = so + p * 512 + (e & 511);
            f4 o = src[0];
#pragma unroll
            for (int w = 1; w < NG; ++w) {
                const f4 y = src[w * P * 512];
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] += y[k];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (v + k < vend) a.opart[(pb + v + k) * HD + d] = o[k];
        }
    }
}

// mass_out = mass_in + sum over the head's query vectors of the block's share of their softmax: a wave
// takes one of a head's blocks.  The vectors' final maxima and sums are formed again here from the
// parts' (a launch that waited for them took 4 us more), once for NW blocks: vectors x parts x blocks /
// NW reads.  17 rows, 500 blocks of 4 heads: with the join 6.5 us; 64 rows, 1023 blocks 20.4 us (7.6
// without masses).
template <int NW>
__device__ __forceinline__ void mass_blocks(const Kv8AttnArgs& a, int blk) {
    __shared__ float2 s_w[2][NW][64];
    __shared__ int s_stop;
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6, nv = a.M * a.G, per = (a.n + NW - 1) / NW;
    const int g = blk / per, i = (blk - g * per) * NW + wv, ic = min(i, a.n - 1);
    const int ab = a.abort ? *a.abort : 0;
    if (t == 0) s_stop = ab;
    const size_t step = (size_t)a.p.nKV * nv, at = (size_t)g * a.p.stride + ic;
    const bool there = page_of_list(a, g, ic) >= 0;
    const float before = a.mass_in ? a.mass_in[at] : 0.0f;
    float s = 0.0f;
    for (int v0 = 0; v0 < nv; v0 += 64) {  // a lane a vector, a wave every NW-th part
        const int vc = min(v0 + lane, nv - 1);
        const float2 rc = a.rec[((size_t)g * a.n + ic) * nv + vc];
        const float2* ml = a.ml + (size_t)g * nv + vc;
        float m = -INFINITY, l = 0.0f;
        for (int c0 = wv; c0 < a.parts; c0 += 16 * NW) {
            float2 x[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = ml[(size_t)min(c0 + NW * j, a.parts - 1) * step];
            float mn = m;
#pragma unroll
            for (int j = 0; j < 16; ++j) mn = fmaxf(mn, x[j].x);
            const float ref = mn == -INFINITY ? 0.0f : mn;
            l *= __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
            for (int j = 0; j < 16; ++j)
                l = c0 + NW * j < a.parts ? fmaf(x[j].y, __builtin_amdgcn_exp2f(x[j].x - ref), l) : l;
            m = mn;
        }
        s_w[v0 / 64 & 1][wv][lane] = make_float2(m, l);
        __syncthreads();  // (the next write of this buffer is behind the next barrier)
        const float2* w = &s_w[v0 / 64 & 1][0][lane];
        float mx = w[0].x;
#pragma unroll
        for (int k = 1; k < NW; ++k) mx = fmaxf(mx, w[64 * k].x);
        mx = mx == -INFINITY ? 0.0f : mx;
        float ls = 0.0f;
#pragma unroll
        for (int k = 0; k < NW; ++k) ls = fmaf(w[64 * k].y, __builtin_amdgcn_exp2f(w[64 * k].x - mx), ls);
        const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
        const float share =
            rc.y * inv * __builtin_amdgcn_exp2f((rc.x == -INFINITY ? 0.0f : rc.x) - mx);
        s += v0 + lane < nv ? share : 0.0f;
    }
    if (s_stop) return;
    s = wave_sum(there ? s : 0.0f);
    if (lane == 0 && i < a.n) a.mass_out[at] = before + s;
}

// One block a row and head.  NG groups of 32 lanes (a lane four dims) take every NG-th part, eight
// requested at a time, each to its own running maximum; the groups are then joined in order.  A part
// that saw no key has maximum -inf and weight 0.  Blocks past the rows' form the masses.  One row of 16
// heads over 30 to 64 parts 3.4 to 5.3 us, a launch and a round of requests; 64 rows over 63 parts (33
// MB) 7.6 us.
template <int NG, bool MASS>
__global__ __launch_bounds__(32 * NG) void k_kv8_combine(Kv8AttnArgs a) {
    const int t = threadIdx.x, gr = t >> 5, d4 = t & 31;
    const int nQ = a.p.nKV * a.G, nv = a.M * a.G;
    if (MASS && (int)blockIdx.x >= a.M * nQ) {
        if constexpr (MASS) mass_blocks<NG / 2>(a, blockIdx.x - a.M * nQ);
        return;
    }
    const int r = blockIdx.x / nQ, h = blockIdx.x % nQ, g = h / a.G, v = r * a.G + h % a.G;
    __shared__ f4 s_o[NG][32];
    __shared__ float s_m[NG], s_l[NG];
    __shared__ int s_abort;
    const int ab = a.abort ? *a.abort : 0;
    if (t == 0) s_abort = ab;
    const size_t step = (size_t)a.p.nKV * nv, at = (size_t)g * nv + v;
    float m = -INFINITY, l = 0.0f;
    f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c0 = gr; c0 < a.parts; c0 += 8 * NG) {
        float2 ml[8];
        f4 x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const size_t c = at + (size_t)min(c0 + NG * j, a.parts - 1) * step;
            ml[j] = a.ml[c];
            x[j] = *(const f4*)(a.opart + c * HD + 4 * d4);
        }
        float mn = m;
#pragma unroll
        for (int j = 0; j < 8; ++j) mn = fmaxf(mn, ml[j].x);  // (a repeated last part changes nothing)
        const float ref = mn == -INFINITY ? 0.0f : mn;
        const float f = __builtin_amdgcn_exp2f(m - ref);
        l *= f;
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] *= f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (c0 + NG * j >= a.parts) break;
            const float w = __builtin_amdgcn_exp2f(ml[j].x - ref);
            l = fmaf(ml[j].y, w, l);
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = fmaf(x[j][k], w, o[k]);
        }
        m = mn;
    }
    s_o[gr][d4] = o;
    if (d4 == 0) {
        s_m[gr] = m;
        s_l[gr] = l;
    }
    __syncthreads();
    if (s_abort || t >= 16) return;
    float mx = s_m[0];
#pragma unroll
    for (int j = 1; j < NG; ++j) mx = fmaxf(mx, s_m[j]);
    const float ref = mx == -INFINITY ? 0.0f : mx;
    float y[8] = {};
    l = 0.0f;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
        const float w = __builtin_amdgcn_exp2f(s_m[j] - ref);
        l = fmaf(s_l[j], w, l);
        const f4 p0 = s_o[j][2 * t], p1 = s_o[j][2 * t + 1];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            y[k] = fmaf(p0[k], w, y[k]);
            y[4 + k] = fmaf(p1[k], w, y[4 + k]);
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key at all: zeros
    u4v ov;
#pragma unroll
    for (int j = 0; j < 4; ++j) ov[j] = pack2(f2h(y[2 * j] * inv), f2h(y[2 * j + 1] * inv));
    if (a.out) *(u4v*)(a.out + (size_t)r * a.ldo + (size_t)h * HD + 8 * t) = ov;
    if (a.out_perm) {
        const int K = nQ * HD;
        emit_qx(ov, t, a.out_perm + (size_t)r * K, a.out_sum + (size_t)r * (K / 64), h * HD + 8 * t);
    }
}

#define NWAVES 8
#define CHIP 256       // blocks of the attention launch, one a CU
#define RING_MOST 128  // parts of a ring
size_t kv8_attn_plan(Kv8AttnArgs& a, bool mass, void* base) {
    a.n_list = a.n_sel > 0 ? a.n_sel : a.n;
    a.ring_units = (a.R + a.M + KV8_B - 1) / KV8_B;
    const int nv = a.M * a.G;
    const int tiles = ((a.n_sel > 0 ? a.G : nv) + 15) / 16;  // that share their units
    const int rows = a.n_sel > 0 ? a.M : 1;
    // Shared pages: each is turned to halves by a whole block, a page or two a block where there are few
    // (one row at 2000 tokens 5.3 us, 7.2 where a wave takes a page alone; 8 rows at 9600 8.0 and 11.8).
    // Pages of a wave's own, for one or two tiles: they stream (one row at 131000 tokens 23 us; 8 rows
    // at 65000 17.4, 19.9 shared); of two waves together, for three or four, later (9 rows at 131000
    // tokens 31.6 us, 35.9 shared; at 65000 19.7 and 20.6; at 32000 14.8 and 14.3).  More share (17
    // rows at 131000 47 us, 51 by four waves together).  Two tiles a wave past eight in all, where the
    // block's LDS reads bound it (64 rows at 65000 tokens 46 us, 60 with one; at 9600 20.6 and 18.8).
    // Rows with lists of their own take pages each (join included: one row of 64 listed blocks 10.6 us
    // shared and 10.9, of 128 11.7 and 11.2; 9 rows of 8 9.5 and 10.4, of 16 10.4 and 10.6, of 32 13.2
    // and 10.9; 64 rows of one 19.1 and 17.5).
    const int64_t visits = (int64_t)a.n_list * a.p.nKV;
    const int64_t most = tiles == 1 ? 300 : tiles == 2 ? 2500 : tiles <= 4 ? 3500 : INT64_MAX;
    a.shared = visits * rows * ((tiles + NWAVES - 1) / NWAVES) <= most;
    a.pair = !a.shared && tiles > 2 ? 2 : 1;
    a.tiles = a.shared ? (tiles > NWAVES && visits > 1400 ? 2 : 1) : std::min(tiles, 2);
    const int per = a.shared ? a.tiles * NWAVES : a.tiles * a.pair;
    a.cols = rows * ((tiles + per - 1) / per);
    // one block a CU, those of the ring (small, first in the grid) among them: a block more than the
    // chip holds would run alone at the end.  A ring of many units leaves the pages half the chip, and
    // one of more than 8192 rows takes several units a part (the parts' outputs grow with them).
    const int share = CHIP / (a.cols * a.p.nKV), ring_most = std::max(share, RING_MOST);
    a.upr = (a.ring_units + ring_most - 1) / ring_most;
    a.ring_parts = (a.ring_units + a.upr - 1) / a.upr;
    int parts = std::max({1, share / 2, share - a.ring_parts});
    parts = std::min(parts, a.shared ? a.n_list : (a.n_list + NWAVES / a.pair - 1) / (NWAVES / a.pair));
    a.upp = parts ? (a.n_list + parts - 1) / parts : 0;
    a.parts = a.ring_parts + (parts ? (a.n_list + a.upp - 1) / a.upp : 0);
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
    return off;
}

// A plan's parts: at most a list's blocks and CHIP / (cols nKV), and of the ring its units and ring_most.
// A column has at most 16 tiles, so vectors times page parts stay below 256 CHIP, or one part each.
size_t kv8_attn_bound(int nKV, int64_t vecs, int n_list, int64_t ring_rows, int n_mass) {
    const int64_t share = std::max(1, CHIP / nKV);
    const int64_t units = (ring_rows + KV8_B - 1) / KV8_B;
    const int64_t pages = std::min(vecs * std::min<int64_t>(n_list, share), std::max<int64_t>(vecs, 256 * CHIP));
    const int64_t ring = vecs * std::min(units, std::max<int64_t>(share, RING_MOST));
    return (size_t)(pages + ring) * (HD * 4 + 8) + (n_mass ? ((size_t)vecs * n_mass + 16) * 8 : 0) + 1024;
}

#define ATTN_LDS 65536  // two pages as halves; the waves' outputs side by side; a ring unit

// The LDS past 64 KB is asked for once a kernel and device.
template <auto KERNEL>
static hipError_t launch_one(const Kv8AttnArgs& a, hipStream_t st) {
    static std::atomic<uint64_t> raised{0};
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (!(raised.load(std::memory_order_relaxed) & bit)) {
        e = hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, ATTN_LDS);
        if (e != hipSuccess) return e;
        raised.fetch_or(bit, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL(KERNEL, dim3(a.parts, a.cols, a.p.nKV), dim3(64 * NWAVES), ATTN_LDS, st, a);
    return hipGetLastError();
}
template <bool MASS>
static hipError_t launch_pages(const Kv8AttnArgs& a, hipStream_t st) {
    if (a.shared)
        return a.tiles == 1 ? launch_one<k_kv8_attn_shared<1, NWAVES, MASS>>(a, st)
                            : launch_one<k_kv8_attn_shared<2, NWAVES, MASS>>(a, st);
    if (a.pair == 2) return launch_one<k_kv8_attn_own<2, 2, NWAVES, MASS>>(a, st);
    return a.tiles == 1 ? launch_one<k_kv8_attn_own<1, 1, NWAVES, MASS>>(a, st)
                        : launch_one<k_kv8_attn_own<2, 1, NWAVES, MASS>>(a, st);
}

template <bool MASS>
static hipError_t launch_attn_pass(const Kv8AttnArgs& a, hipStream_t st) {
    const hipError_t e = launch_pages<MASS>(a, st);
    if (e != hipSuccess) return e;
    // the join: a block a row and head, then (masses) one for every NG / 2 blocks of a head
    auto join = [&](auto kernel, int ng) {
        const int masses = MASS ? (a.n + ng / 2 - 1) / (ng / 2) * a.p.nKV : 0;
        hipLaunchKernelGGL(kernel, dim3(a.M * a.p.nKV * a.G + masses), dim3(32 * ng), 0, st, a);
    };
    // more than 64 parts, a round of 8 groups' requests: 32 groups (4 rows of 8 heads over 250 parts 6.3
    // us, 11.8 by 8 groups; 1 row of 16 heads over 60 parts 4.9 us, 4.0 by 8)
    if (a.parts > 64) join(k_kv8_combine<32, MASS>, 32);
    else join(k_kv8_combine<8, MASS>, 8);
    return hipGetLastError();
}

hipError_t launch_kv8_attn(const Kv8AttnArgs& a, hipStream_t st) {
    if (a.M < 1 || a.M > MJ_ROWS || a.ring.C >= ((int64_t)1 << 30) || a.parts < 1)
        return hipErrorInvalidValue;
    return a.rec ? launch_attn_pass<true>(a, st) : launch_attn_pass<false>(a, st);
}
