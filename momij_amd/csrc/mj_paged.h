// mj_paged.h -- launchers of the pages of many sequences (paged.hip, paged_attn.hip) and of their
// drafts' acceptance (accept.hip) for the C entries (paged.cpp).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mj_internal.h"

#define PG_UNIT 32          // tokens of a unit: the keys of one step of attention
#define PG_UNIT_HALVES 4096  // halves of K or of V in a unit of one head
#define PG_MAX_SEQS 1024
#define PG_MAX_LAYERS 4096
#define PG_NEED 3           // blocks that MJ_ROWS rows touch at most (pages of 32 and more)
#define PG_REFUSED 0        // of a sequence: the last call for room had none for its rows
#define PG_SERVED 1         // it had
#define PG_UNKNOWN -1       // nobody asked since its pages were another's too, or cut

struct PgPool {
    uint16_t* k;  // [n_layers][n_pages][nKV][page * 128]
    uint16_t* v;
    int32_t* table;  // [n_seqs][stride]
    int32_t* lens;   // [n_seqs]
    int32_t* refs;   // [n_pages]
    int32_t* served;  // [n_seqs] or nullptr: PG_REFUSED, PG_SERVED, others
    int nKV, n_pages, page, shift, n_seqs, stride, n_layers;  // page = 1 << shift tokens
    __host__ __device__ size_t head_halves() const { return (size_t)page * 128; }
    __host__ __device__ size_t layer_halves() const { return (size_t)n_pages * nKV * page * 128; }
    __host__ __device__ int room() const { return stride << shift; }  // tokens a table row can hold
};

// The rows of a pass: sequence s has start[s] .. start[s + 1] - 1 of them.
struct PgRows {
    const int32_t* start;
    const uint64_t* anc;  // [rows] rows of its sequence that a row sees (nullptr: a chain)
    int rows, max_rows, n_seqs;
};

struct PgAppendArgs {
    PgPool p;
    PgRows b;
    const uint16_t* qkv;
    int64_t ld;
    const uint16_t* qw;  // nullable: queries (keys) are not normed
    const uint16_t* kw;
    uint16_t* q_out;
    int layer, nQ, half;
    float eps;
    const int* abort;
    double turns[MJ_ROPE_F];  // frequency i in turns a position
};
hipError_t launch_paged_append(const PgAppendArgs& a, hipStream_t st);

hipError_t launch_pages_fork(const PgPool& p, const int32_t* from, const int* abort, hipStream_t st);
hipError_t launch_pages_truncate(const PgPool& p, const int32_t* len, const int* abort,
                                 hipStream_t st);
hipError_t launch_pages_reserve(const PgPool& p, const PgRows& b, int32_t* out, const int* abort,
                                hipStream_t st);
hipError_t launch_pages_commit(const PgPool& p, const PgRows& b, const int32_t* accepted,
                               const int32_t* path, int32_t* lens_out, const int* abort,
                               hipStream_t st);

#define PG_MAX_BLOCKS 512  // of an attention launch
struct PgAttnArgs {
    PgPool p;
    PgRows b;
    const uint16_t* q;
    int64_t ldq;
    uint16_t* out;
    int64_t ldo;
    int layer, G, window;
    // set by paged_attn_plan: blocks of the launch, query vectors a column group, units
    // a block at least, and the workspace
    int blocks, cols, least, extra;
    int64_t* off;   // [n_seqs + 2]: units before each sequence, units in all, units a block
    float* po;      // [blocks][2][cols][128] partial outputs of a block's first and last segment
    float2* pml;    // [blocks][2][cols] {reference, sum}
    const int* abort;
};
// Fills the plan fields and returns the workspace bytes; base (nullable) is where it lies.
size_t paged_attn_plan(PgAttnArgs& a, void* base);
hipError_t launch_paged_attn(const PgAttnArgs& a, hipStream_t st);

// A chunk's share of a row's probabilities: sum of exp((x - m) / T), its greatest logit and where.
struct AcceptPart {
    double s;
    float m;
    int at;
};
// A sequence's last row, for the launch that samples from what is left of it (row -1: nothing to do).
struct AcceptLast {
    double Z;          // its sum
    uint64_t refused;  // drafts below it, by row of the sequence
    float m;           // its greatest logit
    int first, row;    // of the sequence, and the row
    int count;         // blocks that have stored their chunk's sum
};
struct AcceptArgs {
    PgRows b;
    const float* logits;
    int64_t ld;
    int V;
    const int32_t* tokens;
    const float* q;  // nullable
    int64_t ldq;
    const float* temperature;
    const float* u_accept;
    const float* u_sample;
    int32_t* accepted;
    int32_t* path;
    int32_t* token;
    // workspace
    AcceptPart* part;  // [rows][chunks]
    double* csum;      // [n_seqs][chunks] what is left of the last row's probabilities
    AcceptLast* last;  // [n_seqs]
    int chunks;        // of a row
    const int* abort;
};
size_t accept_rows_layout(AcceptArgs& a, void* base);
hipError_t launch_accept_rows(const AcceptArgs& a, hipStream_t st);

// Rows of sequence s (at most max_rows), the first of them r0; whatever `start` holds, they lie in the
// batch's arrays.
__device__ __forceinline__ int pg_rows(const PgRows& b, int s, int& r0) {
    const int lo = min(max(b.start[s], 0), b.rows), hi = min(max(b.start[s + 1], lo), b.rows);
    r0 = lo;
    return min(hi - lo, b.max_rows);
}
__device__ __forceinline__ int pg_len(const PgPool& p, int s) { return min(max(p.lens[s], 0), p.room()); }
// The page of block j of sequence s, or -1.
__device__ __forceinline__ int pg_page(const PgPool& p, int s, int j) {
    if ((unsigned)j >= (unsigned)p.stride) return -1;
    const int pg = p.table[(size_t)s * p.stride + j];
    return (unsigned)pg < (unsigned)p.n_pages ? pg : -1;
}
// Whether rows of a sequence may be written to a page of its table.  Where it was served: from its length on its
// pages hold nothing that is another's (those that others named were left then; a branch made since has
// the tokens before that length only, and its own call for room gives it other pages; a branch's and a cut
// sequence's word is PG_UNKNOWN).  Where it is not known, the page's count tells.
__device__ __forceinline__ int pg_word(const PgPool& p, int s) {
    const int word = p.served ? p.served[s] : PG_UNKNOWN;
    return word == PG_SERVED || word == PG_REFUSED ? word : PG_UNKNOWN;
}
__device__ __forceinline__ bool pg_own(int word, int refs) {  // refs: of the page, or the greatest of several
    return word == PG_SERVED || (word == PG_UNKNOWN && refs <= 1);
}
// Whether all of m rows from the length L on could be written.  (No branches: one after another the requests of three
// blocks took 1.5 us.)
__device__ __forceinline__ bool pg_stored(const PgPool& p, int s, int L, int m) {
    const int word = pg_word(p, s), first = L >> p.shift, n = m > 0 ? ((L + m - 1) >> p.shift) - first + 1 : 0;
    const int32_t* row = p.table + (size_t)s * p.stride;
    int pg[PG_NEED], refs[PG_NEED];
#pragma unroll
    for (int i = 0; i < PG_NEED; ++i) pg[i] = row[min(first + i, p.stride - 1)];
    bool all = first + n <= p.stride;
    int most = 0;
#pragma unroll
    for (int i = 0; i < PG_NEED; ++i) {
        const bool there = (unsigned)pg[i] < (unsigned)p.n_pages;
        all &= there | (i >= n);
        pg[i] = there ? pg[i] : 0;
    }
#pragma unroll
    for (int i = 0; i < PG_NEED; ++i) refs[i] = p.refs[pg[i]];
#pragma unroll
    for (int i = 0; i < PG_NEED; ++i) most = max(most, i < n ? refs[i] : 0);
    return all & pg_own(word, most);
}
// The sequence that row r belongs to (n_seqs: none), by one round of loads of a whole wave.
__device__ __forceinline__ int pg_seq(const PgRows& b, int r) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int s = lane; s - lane < b.n_seqs; s += 64)
        n += __popcll(__ballot(s < b.n_seqs && b.start[s + 1] <= r));
    return n;
}
__device__ __forceinline__ uint64_t pg_anc(const PgRows& b, int row, int local) {
    return b.anc ? b.anc[row] : (2ull << local) - 1;
}
__device__ __forceinline__ int pg_depth(uint64_t anc, int local) { return __popcll(anc & ((1ull << local) - 1)); }
// Where token t and dims d .. d + 7 (K) or dim d (V) lie in a head's page.
__device__ __forceinline__ int pg_k_at(int t, int d) {
    return (t >> 5) * PG_UNIT_HALVES + 2048 * ((t >> 2) & 1) + 512 * (d >> 5) + 128 * ((d >> 3) & 3) +
           32 * ((t >> 3) & 3) + 8 * (t & 3) + (d & 7);
}
__device__ __forceinline__ int pg_v_at(int t, int d) {
    return (t >> 5) * PG_UNIT_HALVES + 512 * (d >> 4) + 128 * ((t >> 3) & 3) + 8 * (d & 15) + (t & 7);
}
