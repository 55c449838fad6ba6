// paged.hip -- the pages of many sequences: appending a batch's normed and rotated rows, making room
// (with a copy of shared pages), sharing, giving back, and moving accepted rows together.
// (Attention over the pages: paged_attn.hip.)
#include <algorithm>

#include "mj_device.h"
#include "mj_paged.h"

#define HD 128

// ------------------------------------------------------------------------------------ append
// As k_qkv_append (a 256-thread block takes 32 of a row's nQ + 2 nKV vectors, eight lanes a vector, 16 dims
// a lane, both dims of a rotated pair in one lane; angles in turns in 64 bits), with the row's sequence,
// length and depth from the device: every wave counts the sequences that end at or before the row, 64 a
// step, so the position is two dependent rounds of requests away and the row's data are on their way
// meanwhile.  A token's V goes to 128 places 16 bytes apart (eight tokens of a dim lie together).  A row takes
// 3.8 us, 64 chains of up to 9 rows 6.3.
__global__ __launch_bounds__(256) void k_paged_append(PgAppendArgs a) {
    __shared__ float2 cs[MJ_ROPE_F];
    __shared__ int s_abort;
    const int t = threadIdx.x, jb = t & 7, r = blockIdx.y;
    const int vec = blockIdx.x * 32 + (t >> 3), nv = a.nQ + 2 * a.p.nKV;
    const int vc = vec < nv ? vec : nv - 1;
    const int X = a.half >= 16 ? a.half / 8 : 8;
    const int pa = (jb & (X - 1)) | ((jb & ~(X - 1)) << 1), pb = pa + X;
    const uint16_t* src = a.qkv + (size_t)r * a.ld + (size_t)vc * HD;
    const bool isq = vc < a.nQ, isv = vc >= a.nQ + a.p.nKV;
    const uint16_t* nw = isq ? a.qw : a.kw;
    u4v va = *(const u4v*)(src + 8 * pa), vb = *(const u4v*)(src + 8 * pb);
    u4v wa{}, wb{};
    if (nw) {
        wa = *(const u4v*)(nw + 8 * pa);
        wb = *(const u4v*)(nw + 8 * pb);
    }
    const int ab = abort_word(a.abort);
    if (t == 0) s_abort = ab;
    const int s = pg_seq(a.b, r);
    int r0 = 0, m = 0, L = 0, word = PG_UNKNOWN;
    if (s < a.b.n_seqs) {
        m = pg_rows(a.b, s, r0);
        L = pg_len(a.p, s);
        word = pg_word(a.p, s);
    }
    const int local = r - r0;
    const bool row = local >= 0 && local < m;
    // (the page on its way before the angles, its count before the norm)
    const int slot = L + local, pg = row ? pg_page(a.p, s, slot >> a.p.shift) : -1, tok = slot & (a.p.page - 1);
    if (t < a.half && row) {
        const int64_t pos = (int64_t)L + pg_depth(pg_anc(a.b, r, local), local);
        const double turn = (double)pos * a.turns[t];
        float sn, c;
        sincospif(2.0f * (float)(turn - rint(turn)), &sn, &c);
        cs[t] = make_float2(c, sn);
    }
    __syncthreads();
    if (s_abort || !row) return;
    const int named = word == PG_UNKNOWN && pg >= 0 ? a.p.refs[pg] : 0;
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
        for (int k = 1; k < 8; k <<= 1) ss += __shfl_xor(ss, k, MJ_WAVE);
        const float scl = 1.0f / sqrtf(ss / (float)HD + a.eps);
        const bool rot = 8 * pa < a.half;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (nw) {
                xa[i] = xa[i] * scl * h2f((uint16_t)(wa[i >> 1] >> (16 * (i & 1))));
                xb[i] = xb[i] * scl * h2f((uint16_t)(wb[i >> 1] >> (16 * (i & 1))));
            }
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
    if (isq) {
        uint16_t* dst = a.q_out + ((size_t)r * a.nQ + vec) * HD;
        *(u4v*)(dst + 8 * pa) = va;
        *(u4v*)(dst + 8 * pb) = vb;
        return;
    }
    if (pg < 0 || !pg_own(word, named)) return;
    const int g = vec - a.nQ - (isv ? a.p.nKV : 0);
    const size_t at = a.layer * a.p.layer_halves() + ((size_t)pg * a.p.nKV + g) * a.p.head_halves();
    if (!isv) {
        *(u4v*)(a.p.k + at + pg_k_at(tok, 8 * pa)) = va;
        *(u4v*)(a.p.k + at + pg_k_at(tok, 8 * pb)) = vb;
        return;
    }
    uint16_t *da = a.p.v + at + pg_v_at(tok, 8 * pa), *db = a.p.v + at + pg_v_at(tok, 8 * pb);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        da[8 * i] = (uint16_t)(va[i >> 1] >> (16 * (i & 1)));
        db[8 * i] = (uint16_t)(vb[i >> 1] >> (16 * (i & 1)));
    }
}

hipError_t launch_paged_append(const PgAppendArgs& a, hipStream_t st) {
    if (a.b.rows < 1 || a.b.rows > 65535 || a.half > MJ_ROPE_F || (a.half & (a.half - 1)) || a.half == 8)
        return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_paged_append, dim3((a.nQ + 2 * a.p.nKV + 31) / 32, a.b.rows), dim3(256), 0, st, a);
    return hipGetLastError();
}

// -------------------------------------------------------------------------------------- pages
// A sequence's entries from `first` on given back: one reference less each, the entry empty.
__device__ __forceinline__ void give_back(const PgPool& p, int s, int first) {
    int32_t* row = p.table + (size_t)s * p.stride;
    for (int j = first + (int)threadIdx.x; j < p.stride; j += (int)blockDim.x) {
        const int pg = row[j];
        if ((unsigned)pg < (unsigned)p.n_pages) atomicSub(&p.refs[pg], 1);
        if (pg != -1) row[j] = -1;
    }
}

__global__ __launch_bounds__(256) void k_pages_truncate(PgPool p, const int32_t* len, const int* abort) {
    __shared__ int s_abort;
    const int ab = abort_word(abort);
    const int s = blockIdx.x, want = len[s], L = pg_len(p, s), n = min(want, L);
    if (threadIdx.x == 0) s_abort = ab;
    __syncthreads();
    if (s_abort || want < 0) return;
    if (threadIdx.x == 0) {
        p.lens[s] = n;
        if (p.served && n < L) p.served[s] = PG_UNKNOWN;
    }
    give_back(p, s, (n + p.page - 1) >> p.shift);
}

// A branch takes its source's place in the table: its own entries are given back, the source's committed
// ones named once more.  Counts only change by atomics, so the order of the blocks does not matter; a
// source that is itself a destination would be read while it is written, and is not taken.
__global__ __launch_bounds__(256) void k_pages_fork(PgPool p, const int32_t* from, const int* abort) {
    __shared__ int s_abort;
    const int ab = abort_word(abort);
    const int s = blockIdx.x, f = from[s];
    if (threadIdx.x == 0) s_abort = ab;
    __syncthreads();
    if (s_abort) return;
    if ((unsigned)f >= (unsigned)p.n_seqs || f == s) return;
    const int ff = from[f];
    if ((unsigned)ff < (unsigned)p.n_seqs && ff != f) return;
    const int L = pg_len(p, f), n = (L + p.page - 1) >> p.shift;
    int32_t* dst = p.table + (size_t)s * p.stride;
    const int32_t* src = p.table + (size_t)f * p.stride;
    for (int j = threadIdx.x; j < p.stride; j += 256) {
        const int old = dst[j];
        int pg = j < n ? src[j] : -1;
        if ((unsigned)pg >= (unsigned)p.n_pages) pg = -1;
        if ((unsigned)old < (unsigned)p.n_pages) atomicSub(&p.refs[old], 1);
        if (pg >= 0) atomicAdd(&p.refs[pg], 1);
        dst[j] = pg;
    }
    if (threadIdx.x == 0) {
        p.lens[s] = L;
        if (p.served) p.served[s] = PG_UNKNOWN;
    }
}

// Inclusive sum over a block of 1024 threads; *total: of all of them.
__device__ __forceinline__ int block_scan(int v, int* wsum, int* total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(v, o, MJ_WAVE);
        v += lane >= o ? x : 0;
    }
    __syncthreads();  // (the sums of a scan before are read)
    if (lane == 63) wsum[w] = v;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int x = wsum[i];
        before += i < w ? x : 0;
        all += x;
    }
    *total = all;
    return before + v;
}

// Room for the batch's rows, one block: a thread a sequence counts the blocks that it lacks, a scan gives
// each its place among them, and the pool's counts are gone through for as many free pages, 16 a thread
// and round, so that the k-th lacking block takes the k-th free page.  Bound by requests one after another (a
// sequence's rows and length, its table, the counts of these pages) and three scans: 5 us for 4 sequences, 6 for
// 64; the counts of the first 16384 pages come meanwhile.
__global__ __launch_bounds__(1024) void k_pages_reserve(PgPool p, PgRows b, int32_t* out, const int* abort) {
    __shared__ int wsum[16];
    __shared__ int ids[PG_NEED * PG_MAX_SEQS];
    __shared__ int s_abort;
    const int s = threadIdx.x;
    const int ab = abort_word(abort);
    int4 next[4];  // counts of 16 pages, requested a round ahead
    auto request = [&](int base) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int at = base + 16 * s + 4 * k;
            next[k] = make_int4(1, 1, 1, 1);
            if (at + 3 < p.n_pages) {
                next[k] = *(const int4*)(p.refs + at);
            } else {
                if (at < p.n_pages) next[k].x = p.refs[at];
                if (at + 1 < p.n_pages) next[k].y = p.refs[at + 1];
                if (at + 2 < p.n_pages) next[k].z = p.refs[at + 2];
            }
        }
    };
    request(0);
    int old[PG_NEED], refs[PG_NEED], need = 0, count = 0, first = 0, L = 0, m = 0;
    bool fits = false;
    if (s < p.n_seqs) {
        int r0;
        m = pg_rows(b, s, r0);
        L = pg_len(p, s);
        first = L >> p.shift;
        const int last = (L + m - 1) >> p.shift;
        fits = m > 0 && last < p.stride;
#pragma unroll
        for (int i = 0; i < PG_NEED; ++i) old[i] = fits && first + i <= last ? pg_page(p, s, first + i) : -1;
#pragma unroll
        for (int i = 0; i < PG_NEED; ++i) refs[i] = old[i] >= 0 ? p.refs[old[i]] : 0;
#pragma unroll
        for (int i = 0; i < PG_NEED; ++i) {
            if (fits && first + i <= last && refs[i] != 1) {
                need |= 1 << i;
                ++count;
            }
            // (a page that others name too: one reference less, below)
            if (refs[i] <= 1) old[i] = -1;
        }
    }
    if (s == 0) s_abort = ab;
    __syncthreads();
    if (s_abort) {  // nobody is served (the copies that follow go by these records)
        if (s < p.n_seqs) {
            *(int4*)(out + 4 * s) = make_int4(0, 0, -1, -1);
            if (p.served && m > 0) p.served[s] = PG_REFUSED;
        }
        return;
    }
    int want, found = 0;
    const int upto = block_scan(count, wsum, &want);
    for (int base = 0; base < p.n_pages && found < want; base += 1024 * 16) {
        int free = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int4 c = next[k];
            free |= ((c.x == 0) | (c.y == 0) << 1 | (c.z == 0) << 2 | (c.w == 0) << 3) << (4 * k);
        }
        request(base + 1024 * 16);
        int total;
        int at = found + block_scan(__popc(free), wsum, &total) - __popc(free);
        for (; free && at < want; free &= free - 1, ++at) ids[at] = base + 16 * s + __builtin_ctz(free);
        found += total;
    }
    __syncthreads();  // ids, and every count of the pool has been read
    if (s >= p.n_seqs) return;
    const bool served = fits && (upto <= found || count == 0);
    int4 res = make_int4(served ? 1 : 0, served ? count : 0, -1, -1);
    if (served) {
        int at = upto - count;
#pragma unroll
        for (int i = 0; i < PG_NEED; ++i)
            if ((need >> i) & 1) {
                const int pg = ids[at++];
                p.table[(size_t)s * p.stride + first + i] = pg;
                p.refs[pg] = 1;
                if (old[i] >= 0) {
                    atomicSub(&p.refs[old[i]], 1);
                    if (i == 0 && (L & (p.page - 1))) {
                        res.z = old[i];
                        res.w = pg;
                    }
                }
            }
    }
    *(int4*)(out + 4 * s) = res;
    if (p.served && m > 0) p.served[s] = served ? PG_SERVED : PG_REFUSED;
}

// The committed tokens of the pages that were shared, copied to their new ones: block (layer and K or
// V, head, some of the sequences), 16 bytes a thread and piece, four pieces under way (all heads in one block, a
// piece at a time: one branch of 24 layers 7.2 us, so 5); groups of eight tokens behind the last committed one
// stay.  A piece of K holds eight dims of a token (group (piece / 4) % 4 of its unit), one of V eight tokens of
// a dim (group (piece / 16) % 4).  In most steps few sequences or none have a page to copy: of many, a block
// looks through 64 records at once, and the launch has no more blocks than find their place in a few us.
// (An abort does not stop it: the table names the new pages already.)
#define COPY_BLOCKS 16384
__global__ __launch_bounds__(256) void k_pages_copy(PgPool p, const int32_t* moved) {
    const int t = threadIdx.x, lane = t & 63, step = gridDim.z;
    const bool isv = blockIdx.x & 1;
    uint16_t* base = (isv ? p.v : p.k) + (blockIdx.x >> 1) * p.layer_halves() + blockIdx.y * p.head_halves();
    const size_t page_halves = p.nKV * p.head_halves();
    for (int s0 = blockIdx.z; s0 < p.n_seqs; s0 += 64 * step) {
        const int mine = s0 + lane * step;
        int from = -1, to = -1, len = 0;
        if (mine < p.n_seqs) {
            const int2 m = *(const int2*)(moved + 4 * mine + 2);
            from = m.x;
            to = m.y;
            len = pg_len(p, mine);
        }
        const bool has = (unsigned)from < (unsigned)p.n_pages && (unsigned)to < (unsigned)p.n_pages;
        for (uint64_t todo = __ballot(has); todo; todo &= todo - 1) {
            const int l = __builtin_ctzll(todo);
            const int fill = __builtin_amdgcn_readlane(len, l) & (p.page - 1);
            const u4v* src = (const u4v*)(base + __builtin_amdgcn_readlane(from, l) * page_halves);
            u4v* dst = (u4v*)(base + __builtin_amdgcn_readlane(to, l) * page_halves);
            const int n = ((fill + 31) >> 5) * 512;  // (512 pieces a unit)
            for (int i = t; i < n; i += 1024) {
                u4v x[4];
                bool on[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int at = i + 256 * k;
                    const int token = 32 * (at >> 9) + 8 * (isv ? (at >> 4) & 3 : (at >> 2) & 3);
                    on[k] = token < fill;
                    if (on[k]) x[k] = src[at];
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (on[k]) dst[i + 256 * k] = x[k];
            }
        }
    }
}

// The rows of an accepted path moved to consecutive places: block (layer and K or V, sequence, four heads).
// A thread takes 16 bytes of K, or one dim of V, of a head's row; 64 of these rows a turn, all read before any
// is written.  64 sequences of up to 17 rows and 24 layers take 15.8 us, of which looking up who has
// room is 0.3.  (A head a block: 17 us; a head a turn, with the places looked up for each: 26 us.)
#define COMMIT_HEADS 4
// How many rows of a sequence are kept, if they were all written (pg_stored).
__device__ __forceinline__ int kept_rows(int s, int m, const int32_t* accepted) {
    return m > 0 ? max(0, min(accepted[s], m - 1) + 1) : 0;
}
__global__ __launch_bounds__(256) void k_pages_commit(PgPool p, PgRows b, const int32_t* accepted,
                                                      const int32_t* path, int32_t* lens_out,
                                                      const int* abort) {
    __shared__ int64_t s_from[MJ_ROWS], s_to[MJ_ROWS];
    __shared__ int s_n, s_abort, s_stored;
    const int s = blockIdx.y, t = threadIdx.x;
    const bool isv = blockIdx.x & 1;
    const int ab = abort_word(abort);
    int r0;
    const int m = pg_rows(b, s, r0), L = pg_len(p, s);
    const int kept = kept_rows(s, m, accepted);
    if (t < 64) {  // rows that move, in order: where they lie in their page's first head, and where they go
        int from = t;
        if (path && t < kept) from = path[r0 + t];
        bool move = path && t < kept && from != t && from >= 0 && from < m;
        int64_t src = 0, dst = 0;
        if (move) {
            const int a = L + from, c = L + t, pa = pg_page(p, s, a >> p.shift), pc = pg_page(p, s, c >> p.shift);
            const int ta = a & (p.page - 1), tc = c & (p.page - 1);
            move = pa >= 0 && pc >= 0;
            src = (int64_t)((size_t)pa * p.nKV * p.head_halves()) + (isv ? pg_v_at(ta, 0) : pg_k_at(ta, 0));
            dst = (int64_t)((size_t)pc * p.nKV * p.head_halves()) + (isv ? pg_v_at(tc, 0) : pg_k_at(tc, 0));
        }
        const uint64_t which = __ballot(move);
        const int at = __popcll(which & ((1ull << t) - 1));
        if (move) {
            s_from[at] = src;
            s_to[at] = dst;
        }
        if (t == 0) {
            s_n = __popcll(which);
            s_abort = ab;
        }
    } else if (t < 128) {  // (the second wave's requests beside the first one's)
        const bool stored = pg_stored(p, s, L, m);
        if (t == 64) s_stored = stored;
    }
    __syncthreads();
    if (s_abort) return;
    if (blockIdx.x == 0 && blockIdx.z == 0 && t == 0 && lens_out) lens_out[s] = s_stored ? min(L + kept, p.room()) : L;
    const int n = s_stored ? s_n : 0;
    if (n == 0) return;
    uint16_t* base = (isv ? p.v : p.k) + (blockIdx.x >> 1) * p.layer_halves();
    const int h0 = COMMIT_HEADS * blockIdx.z, h1 = min(h0 + COMMIT_HEADS, p.nKV), turn = 64 / n;
    for (int g0 = h0; g0 < h1; g0 += turn) {
        const int rows = n * min(turn, h1 - g0);
        auto at = [&](int j, const int64_t* place) __attribute__((always_inline)) {
            const int g = j / n;
            return base + (size_t)(g0 + g) * p.head_halves() + place[j - g * n];
        };
        if (!isv) {
            const int d = pg_k_at(0, 8 * (t & 15));
            u4v x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = 16 * i + (t >> 4);
                if (j < rows) x[i] = *(const u4v*)(at(j, s_from) + d);
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = 16 * i + (t >> 4);
                if (j < rows) *(u4v*)(at(j, s_to) + d) = x[i];
            }
        } else {
            const int d = pg_v_at(0, t & 127), j0 = __builtin_amdgcn_readfirstlane(t >> 7);
            uint16_t x[32];
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (2 * i + j0 < rows) x[i] = at(2 * i + j0, s_from)[d];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (2 * i + j0 < rows) at(2 * i + j0, s_to)[d] = x[i];
        }
    }
}

// The lengths alone, after every block of the launch before has read them.
__global__ __launch_bounds__(256) void k_pages_lens(PgPool p, PgRows b, const int32_t* accepted,
                                                    const int* abort) {
    if (aborted(abort)) return;
    const int s = blockIdx.x * 256 + threadIdx.x;
    if (s >= p.n_seqs) return;
    int r0;
    const int m = pg_rows(b, s, r0), L = pg_len(p, s);
    p.lens[s] = pg_stored(p, s, L, m) ? min(L + kept_rows(s, m, accepted), p.room()) : L;
}

hipError_t launch_pages_fork(const PgPool& p, const int32_t* from, const int* abort, hipStream_t st) {
    hipLaunchKernelGGL(k_pages_fork, dim3(p.n_seqs), dim3(256), 0, st, p, from, abort);
    return hipGetLastError();
}

hipError_t launch_pages_truncate(const PgPool& p, const int32_t* len, const int* abort, hipStream_t st) {
    hipLaunchKernelGGL(k_pages_truncate, dim3(p.n_seqs), dim3(256), 0, st, p, len, abort);
    return hipGetLastError();
}

hipError_t launch_pages_reserve(const PgPool& p, const PgRows& b, int32_t* out, const int* abort,
                                hipStream_t st) {
    if (p.n_seqs > PG_MAX_SEQS || b.max_rows > MJ_ROWS || p.page < 32) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_pages_reserve, dim3(1), dim3(1024), 0, st, p, b, out, abort);
    const int z = std::max(1, std::min(p.n_seqs, COPY_BLOCKS / (2 * p.n_layers * p.nKV)));
    hipLaunchKernelGGL(k_pages_copy, dim3(2 * p.n_layers, p.nKV, z), dim3(256), 0, st, p, out);
    return hipGetLastError();
}

hipError_t launch_pages_commit(const PgPool& p, const PgRows& b, const int32_t* accepted,
                               const int32_t* path, int32_t* lens_out, const int* abort,
                               hipStream_t st) {
    if (b.max_rows > MJ_ROWS) return hipErrorInvalidValue;
    const bool here = lens_out == p.lens;
    if (path || !here) {
        const dim3 grid(path ? 2 * p.n_layers : 1, p.n_seqs, path ? (p.nKV + COMMIT_HEADS - 1) / COMMIT_HEADS : 1);
        hipLaunchKernelGGL(k_pages_commit, grid, dim3(256), 0, st, p, b, accepted, path, here ? nullptr : lens_out,
                           abort);
    }
    if (here)
        hipLaunchKernelGGL(k_pages_lens, dim3((p.n_seqs + 255) / 256), dim3(256), 0, st, p, b, accepted,
                           abort);
    return hipGetLastError();
}
