// mj_kv8.h -- launchers of the 8-bit KV cache (kv8.hip, kv8_attn.hip) for its C entries (kv8.cpp).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mj_internal.h"

#define KV8_B 64            // tokens a block (MJ_KV8_BLOCK)
#define KV8_PAGE_BYTES 8192  // codes of K or of V in a page

struct Kv8Pool {
    uint8_t* k;
    uint8_t* v;
    float* ks;
    float* vs;
    int8_t* bounds;
    const int32_t* table;
    int nKV, n_pages, stride;
};
struct Kv8Ring {
    uint16_t* k;
    uint16_t* v;
    int64_t C;
};

// Queries and keys of a pass: turns[i] = frequency i in turns a position.
struct Kv8AppendArgs {
    const uint16_t* qkv;
    int64_t ld;
    const uint16_t* qw;
    const uint16_t* kw;
    Kv8Ring ring;
    uint16_t* q_out;
    int64_t L, slot0;  // slot0 = L % C
    int M, nQ, nKV, half;
    float eps;
    const int* abort;
    double turns[MJ_ROPE_F];
    uint8_t depth[MJ_ROWS];
};
hipError_t launch_qkv_append(const Kv8AppendArgs& a, hipStream_t st);

hipError_t launch_kv8_seal(const Kv8Pool& p, const Kv8Ring& r, int64_t slot0, int count, int at,
                           const int* abort, hipStream_t st);
hipError_t launch_kv8_unseal(const Kv8Pool& p, const Kv8Ring& r, int64_t slot0, int count, int at,
                             const int* abort, hipStream_t st);

struct Kv8SelectArgs {
    Kv8Pool p;
    const uint16_t* q;
    int64_t ldq;
    int M, G, n, n_sel, first, last;
    float* scores;  // [M][nKV][n]
    int32_t* sel;   // [M][nKV][n_sel]
    const int* abort;
};
hipError_t launch_kv8_select(const Kv8SelectArgs& a, hipStream_t st);
hipError_t launch_kv8_evict(const Kv8Pool& p, int n, int keep, int first, int last,
                            const float* mass_in, int32_t* table_out, float* mass_out,
                            const int* abort, hipStream_t st);

struct Kv8AttnArgs {
    Kv8Pool p;
    Kv8Ring ring;
    const uint16_t* q;
    int64_t ldq;
    const int32_t* sel;  // [M][nKV][n_sel] or nullptr
    int n, n_sel;        // blocks; listed blocks a row
    int slot0, R, M, G;  // first ring position's slot, committed ring rows, rows, heads a group
    uint16_t* out;       // plain [M][ldo] (nullable)
    int64_t ldo;
    uint16_t* out_perm;  // or the same in qx order [M][nKV * G * 128] with its block sums
    float2* out_sum;
    const float* mass_in;
    float* mass_out;
    // set by kv8_attn_plan: ring_parts of upr units (64 rows) of the ring each, then parts of upp
    // listed blocks each, parts in all; shared: which kernel; tiles: of 16 query vectors, a wave; pair: waves that
    // take their pages together; cols: block columns (groups of tiles, rows with lists of their own)
    int n_list, upp, parts, ring_units, upr, ring_parts, tiles, pair, cols;
    bool shared;
    float* opart;   // [parts][nKV][nv][128] sums of exp2(s - m) v, times a constant
    float2* ml;     // [parts][nKV][nv] {m, sum}: the sum times the same
    float2* rec;    // [nKV][n][nv] {m, sum} of each block where masses are wanted, likewise
    const int* abort;
    uint64_t anc[MJ_ROWS];  // of pass row r: bit a set for its ancestors and itself
};
// Fills the plan fields for the sizes given and returns the workspace bytes; base (nullable) is
// where the workspace lies.
size_t kv8_attn_plan(Kv8AttnArgs& a, bool mass, void* base);
// Bytes that no plan of up to vecs query vectors (of all heads), n_list blocks a list, ring_rows open
// and new rows and n_mass blocks with masses passes.
size_t kv8_attn_bound(int nKV, int64_t vecs, int n_list, int64_t ring_rows, int n_mass);
hipError_t launch_kv8_attn(const Kv8AttnArgs& a, hipStream_t st);
