/*
 * momij_hip.h -- C ABI of the MI355X (gfx950) speculative-decode verify step.
 *
 * Plain C: device pointers are `void*` / typed scalars, sizes are ints.  No HIP or torch types
 * cross this boundary.  Every call is asynchronous on the context's stream unless it says it
 * synchronises; a context is not re-entrant (the reference engine is single-request too,
 * README.md:32, Server.swift:677-700); distinct contexts may be driven from distinct threads.
 * Calls that take host arrays (an attention block, greedy acceptance, a penalty history) are refused
 * with MJ_HIP_ERROR while their stream is being captured into a graph: a replay would run on the
 * captured call's.
 * The caller owns every tensor it allocates (weights, activations, outputs); the library owns
 * only its scratch and, for a model, the KV cache.
 *
 * Reference paths below are relative to penta2himajin/momij, swift/Sources/MomijCore/.
 * Tensor layouts follow MLX (WeightStore.swift:48-92): 2-bit affine weights as uint32 words
 * packing 16 codes LSB-first, [rows][K/16]; fp16 scales and biases [rows][K/gs]; up||gate
 * packed with the up rows first.
 */
#ifndef MOMIJ_HIP_H
#define MOMIJ_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MJ_ABI_VERSION 1
#define MJ_MAX_ROWS 64 /* verify rows per pass (draft tree nodes + 1), prefill chunk */

/* Errors -- SeedlessError {noMetal, notReady, unsupportedShape(N,K,gs)}
 * (SeedlessMetal.swift:3718-3728) plus argument, abort, capacity and runtime failures.
 * mj_last_error() gives the message (shape errors carry N, K and gs). */
typedef enum mj_status {
    MJ_OK = 0,
    MJ_NO_DEVICE = 1,          /* no gfx950 device (noMetal) */
    MJ_NOT_READY = 2,          /* library / model not initialised (notReady) */
    MJ_UNSUPPORTED_SHAPE = 3,  /* unsupportedShape(N:K:gs:) */
    MJ_INVALID_ARG = 4,        /* null pointer, bad index, bad tree */
    MJ_ABORTED = 5,            /* abort word set (stopBuf, SeedlessMetal.swift:60, 69-70) */
    MJ_HIP_ERROR = 6,          /* HIP runtime failure */
    MJ_CAPACITY = 7,           /* KV capacity / prompt too long (SeedlessAttn.swift:279-286) */
    MJ_OUT_OF_MEMORY = 8       /* host allocation failed (draft indexes) */
} mj_status;

typedef struct mj_ctx mj_ctx;
typedef struct mj_model mj_model;

/* ---------------------------------------------------------------- context ---- */
/* SeedlessMetal.ensureCompiled (SeedlessMetal.swift:63-104): device, queue, stop buffer. */
mj_status mj_init(int device, mj_ctx** out);
mj_status mj_destroy(mj_ctx* ctx);
const char* mj_last_error(const mj_ctx* ctx);
const char* mj_status_str(mj_status s);
int mj_abi_version(void);
/* Use an external hipStream_t (e.g. the caller's current stream); NULL restores the own one. */
mj_status mj_set_stream(mj_ctx* ctx, void* hip_stream);
void* mj_get_stream(const mj_ctx* ctx);
/* Abort word (stopBuf, SeedlessMetal.swift:60, 69-70): non-zero makes every kernel of this
 * context that starts after the call return early.  Safe from any thread at any time, also
 * while the owning thread's pass is queued, running or being captured into a graph: the word is
 * written by a copy on a stream of the context's own that no pass uses, and mj_set_abort waits
 * for that copy only.  A synchronising call (mj_sync, mj_prefill's chunks, the verify and step
 * calls) reports MJ_ABORTED when the word is set at its entry (then nothing is queued) or at its
 * end, or was set at any time in between -- whenever some of its kernels may have skipped their
 * work -- and its results are then void (a model's offset does not advance).  Cleared with
 * flag = 0; the next call runs normally. */
mj_status mj_set_abort(mj_ctx* ctx, int flag);
/* Bound of the fused MoE launch's waits (no counterpart in the reference: it has no fused
 * launch).  Passes of at most 32 rows run the up||gate and down products as one launch whose
 * blocks all stay resident; a down item computes once the act rows it stages hold no value the
 * up product has yet to write, staging them again at most `polls` times (default 131072, each
 * after a short sleep: well under a second).  A wait that runs out its bound -- the launch's
 * blocks were not all resident, e.g. kernels of another stream held CUs -- sets the context's
 * fault word, and the next synchronising call reports MJ_HIP_ERROR (the results since the
 * previous one are invalid) and clears it.  polls = 0 forces that report whenever a down item's
 * rows are not complete at its first check.  A pass replayed from a graph keeps the bound it
 * was captured with. */
mj_status mj_set_wait_limit(mj_ctx* ctx, int polls);
/* One wait for everything queued (cb.commit + waitUntilCompleted,
 * SeedlessDecodeEngine.swift:324-325).  Reports MJ_ABORTED if the abort word is set or was set
 * since the previous synchronising call. */
mj_status mj_sync(mj_ctx* ctx);

/* ---------------------------------------------------------------- memory ----- */
mj_status mj_alloc(mj_ctx* ctx, size_t bytes, void** out);
mj_status mj_free(mj_ctx* ctx, void* p);
mj_status mj_h2d(mj_ctx* ctx, void* dst, const void* src, size_t bytes);  /* synchronous */
mj_status mj_d2h(mj_ctx* ctx, void* dst, const void* src, size_t bytes);  /* synchronous */

/* ------------------------------------------------------------------ ops ------ */
/* 2-bit affine gather-qmv / verify GEMM -- SeedlessMetal.gqmm2 (SeedlessMetal.swift:312-438),
 * kernel gqmm2_rows (2168-2221):
 *   y[mk, n] = half( sum_k (s[e,n,k/gs]*q[e,n,k] + b[e,n,k/gs]) * x[row(mk), k] ),
 *   e = inds[mk], row(mk) = lhs_per_expert ? mk : mk / ktop, mk < M*ktop.
 * x fp16 [M or M*ktop][K], w uint32 [E][N][K/16], scales/biases fp16 [E][N][K/gs],
 * inds int32 [M*ktop] (device), y fp16 [M*ktop][N].
 * Shapes: K % 512 == 0 (as the reference, SeedlessMetal.swift:336-338), N % 16 == 0,
 * gs in {64, 128}, M*ktop <= MJ_MAX_ROWS*8.
 * epilogue MJ_EPI_STORE writes y; MJ_EPI_ADD writes y = half(y + half(acc)) (o-proj residual,
 * gqmm2_rows_fold_add 3488-3543; requires ktop == 1). */
#define MJ_EPI_STORE 0
#define MJ_EPI_ADD 1
mj_status mj_gather_qmm2(mj_ctx* ctx, const void* x, const uint32_t* w, const void* scales,
                         const void* biases, const int32_t* inds, void* y, int M, int ktop,
                         int K, int N, int gs, int lhs_per_expert, int epilogue);

/* MoE expert weights of one layer (MapleMoE.swift:6-33 / SeedlessAttn.swift:93-99). */
typedef struct mj_moe_weights {
    const void* norm_w;        /* fp16 [H] post_attention_layernorm (MJ_MOE_PRENORM) */
    const void* router_w;      /* fp16 [E][H] mlp.gate */
    const uint32_t* up_gate_w; /* [E][2I][H/16], rows 0..I-1 up, I..2I-1 gate */
    const void* up_gate_s;     /* fp16 [E][2I][H/gs] */
    const void* up_gate_b;
    const uint32_t* down_w;    /* [E][H][I/16] */
    const void* down_s;        /* fp16 [E][H][I/gs] */
    const void* down_b;
    int E, top_k, H, I, gs;  /* H 2048 or 4096; I a multiple of 512, <= 4096; gs 64 or 128 */
    float eps;
    /* optional row-alpha form (WeightStore.swift:47-63: scales = alpha in every group of a
     * row, biases = -alpha): fp16 [E][2I] and [E][H], 16-byte aligned, or NULL.  When set,
     * up_gate_s/_b and down_s/_b must still hold that expansion: the batched expert kernels
     * read one alpha per row, the one-row and general kernels read the arrays, and the two are
     * not compared (an alpha that is not the arrays' expansion makes decode and verify
     * disagree). */
    const void* up_gate_alpha;
    const void* down_alpha;
} mj_moe_weights;

/* MoE block -- encodeMoEBlock (SeedlessMetal.swift:576-609), MapleMoE.callAsFunction
 * (MapleMoE.swift:58-80): [rms(x)] -> router logits -> softmax top-k (lowest index on ties,
 * renormalised) -> up||gate gather -> clamped SwiGLU -> down gather -> score-weighted combine.
 * flags: MJ_MOE_PRENORM applies norm_w first; MJ_MOE_RESIDUAL writes y = x + moe.
 * x, y fp16 [M][H] (may alias); out_inds int32 [M][top_k], out_scores fp32 [M][top_k]
 * (device, nullable).  Rows are bucketed by expert so each routed expert's weights stream
 * once per call. */
#define MJ_MOE_PRENORM 1
#define MJ_MOE_RESIDUAL 2
mj_status mj_moe_block(mj_ctx* ctx, const mj_moe_weights* w, const void* x, void* y, int M,
                       int flags, int32_t* out_inds, float* out_scores);

/* mj_moe_block without any device allocation.  No counterpart in the reference: it is for
 * callers that cannot allocate (code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc).  Same kernels, arguments and results as mj_moe_block, with the
 * scratch in one statically allocated device array of MJ_MOE_NOALLOC_BYTES per GPU (held until
 * the process ends) instead of the context's growable scratch.  A call whose scratch would
 * exceed it (M rows x top_k x (I + H) halves dominate: H <= 2048 fits any I <= 4096 at
 * M = 64) is refused with MJ_CAPACITY before any work is queued.  Every call on one GPU shares
 * that GPU's array, which keeps the last call's contents: calls that overlap on one GPU (from
 * several contexts, or one context whose stream mj_set_stream changed between calls) race, so
 * the caller must order them -- issue them on one stream, or make each stream wait for the
 * previous call's completion event.  No synchronisation is added here: a wait on an event
 * recorded outside a graph capture would break the capture this entry point exists for. */
#define MJ_MOE_NOALLOC_BYTES (8u << 20)
mj_status mj_moe_block_noalloc(mj_ctx* ctx, const mj_moe_weights* w, const void* x, void* y,
                               int M, int flags, int32_t* out_inds, float* out_scores);

/* Attention weights of one layer (SeedlessAttn.swift:74-92). */
typedef struct mj_attn_weights {
    const void* norm_w;      /* fp16 [H] input_layernorm */
    const uint32_t* qkv_w;   /* [(nQ+2nKV)*D][H/16], q rows then k then v (WeightStore 66-79) */
    const void* qkv_s;
    const void* qkv_b;
    const void* q_norm_w;    /* fp16 [D] */
    const void* k_norm_w;    /* fp16 [D] */
    const uint32_t* o_w;     /* [H][nQ*D/16] */
    const void* o_s;
    const void* o_b;
} mj_attn_weights;

typedef struct mj_attn_config {
    int H, n_heads, n_kv_heads, head_dim; /* head_dim must be 128 */
    int rope_dim;                         /* rotated leading dims (0 = NoPE) */
    float rope_base, eps;
    int window;                           /* sliding window (0 = full attention) */
    int64_t kv_capacity;                  /* slots C of the cache; >= window + M */
    int gs;
} mj_attn_config;

/* Attention block with residual -- encodeAttnBlock (SeedlessMetal.swift:926-1005) with the
 * input RMSNorm of encodeLayerBlock (1008-1048): h += o_proj(attn(rms(h))).
 * Verify row r sits at position L + depth(r); parents_host[r] < r gives the draft tree
 * (NULL = linear chain, parents[0] = -1).  Row r attends the committed positions inside its
 * window plus its ancestors and itself.  New K/V rows are written at slot (L + r) % C of the
 * caches kcache/vcache fp16 [n_kv][C][128]; committed position p lives at slot p % C. */
mj_status mj_attn_block(mj_ctx* ctx, const mj_attn_config* cfg, const mj_attn_weights* w,
                        void* h, void* kcache, void* vcache, int64_t L,
                        const int32_t* parents_host, int M);

/* ------------------------------------------------- a KV cache in 8 bits ------ */
/* The context of a full-attention layer in two tiers (no counterpart in the reference, whose caches
 * are fp16): an fp16 ring holds the newest positions, and blocks of MJ_KV8_BLOCK positions are
 * sealed from it into pages of 8-bit codes.  Attention reads both.  Keys are rotated before they are
 * cached, so which position a block held does not matter once it is sealed: blocks may be left out
 * of a call (mj_kv8_select) or for good (mj_kv8_evict).  Heads of 128 only.
 *
 * Every call below is asynchronous on the context's stream and takes no host array but
 * parents_host: with a tree it is refused while the stream is being captured (a replay would run on
 * the captured call's); with NULL, a chain, it may be captured.  Lengths and positions are
 * captured as they are.  Calls that need device scratch take it from ws (16-byte aligned,
 * mj_kv8_workspace bytes), or, ws NULL, from the context's growable scratch, and are then refused
 * while the stream is being captured (a later call may replace that scratch).  Calls that share a ws
 * must be ordered by the caller.  Calls that may overlap may share a pool as long as none of them
 * writes pages, table entries or ring slots that another one touches.  Device pointers must be
 * 16-byte aligned. */
#define MJ_KV8_BLOCK 64

/* Pool of pages and the lists of them.  A page holds one block of one KV head: 64 x 128 codes of K
 * and of V, a scale for each, and the greatest and the least K code of every dim.  A value is
 * code * scale, scales 0 or more (a V scale below 2^-31, which sealing never writes, counts as 2^-31).
 * Page bytes are in the order the matrix instructions take them:
 *   K: byte 2048 (t / 16) + 1024 (d / 64) + 256 (d / 16 % 4) + 16 (t % 16) + d % 16
 *   V: byte 1024 (d / 16) + 256 (t / 4 % 4) + 16 (d % 16) + 4 (t / 16) + t % 4
 * of token t, dim d, each byte its code + 128.  table[g * table_stride + i] is the page of the i-th
 * block of head g: a head's row lists its n_blocks blocks in use, then (after mj_kv8_evict, or as
 * the caller filled it) its free pages.  An entry outside [0, n_pages) names no block: it is neither
 * read nor written, and its keys are left out.  Two entries naming one page must not both be
 * sealed. */
typedef struct mj_kv8 {
    int n_kv_heads;
    int n_pages;           /* pages of the pool, of all heads together */
    void* k_codes;         /* [n_pages][8192] */
    void* v_codes;         /* [n_pages][8192] */
    float* k_scale;        /* [n_pages] */
    float* v_scale;        /* [n_pages] */
    int8_t* k_bounds;      /* [n_pages][2][128]: greatest, least code */
    int32_t* table;        /* [n_kv_heads][table_stride] */
    int table_stride;      /* blocks a head can list */
} mj_kv8;

/* fp16 rows [n_kv_heads][capacity][128] of K and V, position p at slot p % capacity (the layout of
 * mj_attn_block's caches and of mj_model_kv); n_kv_heads is that of the cache or configuration it is used
 * with (it has no count of its own to check). */
typedef struct mj_kv_ring {
    void* k;
    void* v;
    int64_t capacity;
} mj_kv_ring;

/* Queries and keys of a pass finished and appended: per-head RMSNorm(eps) * weight, then RoPE of the
 * first rope_dim dims (0, 32, 64 or 128; halves (i, i + rope_dim / 2) of a head rotate together) at
 * the row's position L + depth(r), angles formed in 64 bits; parents_host as in mj_attn_block.  qkv
 * fp16 [M] rows of ld_qkv halves (0: packed; else a multiple of 8): the q, k and v heads of a raw
 * projection.  q_out fp16 [M][n_heads * 128], not over qkv; keys and values of row r go to slot (L + r) %
 * capacity.  Reads n_heads, n_kv_heads, head_dim, rope_dim, rope_base and eps of cfg. */
mj_status mj_qkv_append(mj_ctx* ctx, const mj_attn_config* cfg, const void* qkv, int64_t ld_qkv,
                        const void* q_norm_w, const void* k_norm_w, const mj_kv_ring* ring,
                        int64_t L, const int32_t* parents_host, int M, void* q_out);

/* Positions [pos, pos + 64 count) of the ring sealed into the pages of table entries at .. at +
 * count - 1 of every head: scale = m / 127 and code = round(x * (127 / m)) to the nearest whole
 * number, ties to even, each operation in fp32, m the block's greatest finite magnitude (0: all
 * codes 0).  An infinity takes the code +-127, a NaN 0.  64 count <= capacity. */
mj_status mj_kv8_seal(mj_ctx* ctx, const mj_kv8* cache, const mj_kv_ring* ring, int64_t pos,
                      int count, int at);
/* The way back, for a rewind into sealed blocks: entries at .. at + count - 1 to positions
 * [pos, pos + 64 count) of the ring, half(code * scale).  Masses are the caller's: those of entries
 * that will be sealed again want clearing. */
mj_status mj_kv8_unseal(mj_ctx* ctx, const mj_kv8* cache, int at, int count,
                        const mj_kv_ring* ring, int64_t pos);

/* Blocks for each row to read: sel int32 [M][n_kv_heads][n_sel], indices into the head's list in
 * increasing order: the first n_first and the last n_last of the n_blocks blocks and, of the others,
 * those of the greatest score (the lower index on ties); all blocks, then -1, where n_sel >
 * n_blocks.  n_first + n_last <= n_sel (each is cut to n_blocks).  The score bounds q k over the
 * block: with c the query's 8-bit codes of scale s_q (formed as sealed ones are),
 *   max over the group's heads of  (sum_d max(c_d greatest_d, c_d least_d)) * k_scale * s_q,
 * the sum in whole numbers, the products in fp32 from left to right.  A NaN score counts as the
 * least.  q fp16 [M] rows of ld_q halves (0: packed; else a multiple of 8).  Takes scratch at every
 * length, also where a short list's scores stay in the kernel. */
mj_status mj_kv8_select(mj_ctx* ctx, const mj_kv8* cache, int n_heads, const void* q, int64_t ld_q,
                        int M, int n_blocks, int n_sel, int n_first, int n_last, int32_t* sel,
                        void* ws, size_t ws_bytes);

/* Attention of M rows: softmax(q k^T / sqrt(128)) v over the sealed blocks [0, n_blocks) of each
 * head, or (sel, as mj_kv8_select writes it) those listed for the row and head, and over the ring's
 * positions [start, L) and the row's ancestors and itself among the pass's own rows at L + r
 * (parents_host as in mj_attn_block).  A listed index outside [0, n_blocks) names no block; one that
 * is listed twice counts twice.  q as in mj_kv8_select, out fp16 [M] rows of ld_out halves.  0 <=
 * start <= L, L - start + M <= ring capacity.
 * mass_out (nullable; not with sel) float [n_kv_heads][table_stride]: for every block its entry of
 * mass_in (same layout, NULL: zeros; may be mass_out, not a part of it) plus the softmax weight that
 * all rows and the group's heads gave the block's keys (every row's, whether or not it is kept after the
 * pass).
 * Scores, softmax statistics and outputs are summed in fp32.  For the product with V a weight is rounded
 * to fp16 together with its block's V scale: off by half a step, 2^-11 of itself, or, where it is less
 * than 2^-23 of a greater one, by up to 2^-34 of that one (times the code).  A call repeats bit for
 * bit; a row's result in a call of other rows may differ by rounding (the keys are split differently). */
mj_status mj_kv8_attn(mj_ctx* ctx, const mj_kv8* cache, const mj_kv_ring* ring, int n_heads,
                      const void* q, int64_t ld_q, int M, int n_blocks, const int32_t* sel,
                      int n_sel, int64_t start, int64_t L, const int32_t* parents_host, void* out,
                      int64_t ld_out, const float* mass_in, float* mass_out, void* ws,
                      size_t ws_bytes);

/* Eviction down to `keep` of n_blocks blocks a head: the first n_first, the last n_last and, of the
 * others, those of the greatest mass stay (the lower index on ties; a NaN counts as the least; each
 * head by its own masses).  table_out [n_kv_heads][table_stride] lists the kept blocks in their
 * order, then the evicted ones' pages (free now) in theirs, then the rest of the row unchanged;
 * mass_out likewise, 0 from `keep` on.  n_first + n_last <= keep <= n_blocks.  table_out and
 * mass_out must lie over neither cache->table, mass_in nor each other. */
mj_status mj_kv8_evict(mj_ctx* ctx, const mj_kv8* cache, int n_blocks, int keep, int n_first,
                       int n_last, const float* mass_in, int32_t* table_out, float* mass_out);

/* Bytes of workspace that mj_kv8_select and mj_kv8_attn with these sizes or smaller ones of the same heads
 * (ring_rows = L - start + M; n_sel 0: every block; mass: mass_out given) take at most; 0 where an
 * argument is out of range. */
size_t mj_kv8_workspace(int n_heads, int n_kv_heads, int M, int n_blocks, int n_sel,
                        int64_t ring_rows, int mass);

/* mj_attn_block over this cache (full attention: cfg->window must be 0): h += o_proj(attn(rms(h))),
 * the pass's keys appended to the ring at L + r; start, n_blocks, mass_in and mass_out as in
 * mj_kv8_attn; n_sel > 0: every row reads the blocks that mj_kv8_select with n_sel, n_first and
 * n_last chooses (no mass then).  cfg->kv_capacity is not read (the ring's counts).  Scratch is the
 * context's: refused while the stream is being captured. */
mj_status mj_attn_block_kv8(mj_ctx* ctx, const mj_attn_config* cfg, const mj_attn_weights* w,
                            const mj_kv8* cache, const mj_kv_ring* ring, void* h, int n_blocks,
                            int n_sel, int n_first, int n_last, int64_t start, int64_t L,
                            const int32_t* parents_host, int M, const float* mass_in,
                            float* mass_out);

/* ------------------------------------- the verify step of many requests ------ */
/* A server's requests in one pool of fp16 pages (no counterpart in the reference, whose engine holds one
 * request): every layer's page p holds the same tokens of that layer, so one table serves all layers.
 * A step of a batch of sequences:
 *   mj_pages_reserve   room for the batch's rows (shared pages that they go to are copied first)
 *   mj_paged_append    in every layer: queries and keys finished, keys and values written
 *   mj_paged_attn      in every layer: the rows' attention over their sequences' pages
 *   mj_accept_rows     the drafts checked against the target's probabilities
 *   mj_pages_commit    the accepted rows' keys and values together, lengths advanced
 * mj_pages_fork lets sequences share another's pages, mj_pages_truncate gives pages back.
 *
 * Lengths, tables, counts and the rows of a batch are device arrays: every call is asynchronous and may be
 * captured, and a replay goes by what the arrays hold then (calls with workspace, as the 8-bit
 * cache's: from ws, 16-byte aligned, or, ws NULL, from the context's growable scratch, and then refused while
 * the stream is being captured; calls that share a ws must be ordered by the caller).  Whatever the
 * device arrays hold, no call reads or writes outside of the arrays given: lengths count as at most what a table
 * row can hold, a table entry outside [0, n_pages) names no page (its tokens are neither read nor
 * written), rows beyond the batch's or beyond max_rows are left out.  Calls on one pool must be ordered
 * by the caller, except that mj_paged_attn may overlap itself.  Heads of 128 only. */
typedef struct mj_pages {
    int n_layers;
    int n_kv_heads;
    int n_pages;      /* at most 2^28 */
    int page_tokens;  /* 32, 64, 128 or 256 */
    /* fp16 [n_layers][n_pages][n_kv_heads][page_tokens / 32][4096]: units of 32 tokens by 128 dims in the
     * order the matrix instructions take them.  Of token t of a unit and dim d,
     *   K: half 2048 (t / 4 % 2) + 512 (d / 32) + 128 (d / 8 % 4) + 32 (t / 8) + 8 (t % 4) + d % 8
     *   V: half 512 (d / 16) + 128 (t / 8) + 8 (d % 16) + t % 8 */
    void* k;
    void* v;
    int32_t* table;   /* [n_seqs][table_stride]: page of a sequence's block, -1 none */
    int n_seqs;       /* at most 1024 */
    int table_stride; /* blocks a sequence can have; times page_tokens at most 2^30 */
    int32_t* lens;    /* [n_seqs] committed tokens */
    int32_t* refs;    /* [n_pages] how many entries name the page; 0: it is free */
    /* [n_seqs] what the last mj_pages_reserve with rows of a sequence said of it: 1 it had room, 0 it had
     * none; others (to begin with, and after the sequence was forked into or cut): not known.  By this append
     * and commit leave out whoever has no room.  NULL: not known of any.  Where it is not known the counts
     * decide: rows that go to a page with refs above 1 are not written, and a step of which one row has no page, or
     * such a page, is not kept.  (Then a branch made between a step's append and its commit has the step dropped;
     * with 1 it does not.)  Who changes the table by other means than these calls sets it to -1. */
    int32_t* served;
} mj_pages;

/* The rows of a pass: sequence s has rows row_start[s] .. row_start[s + 1] - 1 (none: it takes no
 * part), at most max_rows <= MJ_MAX_ROWS.  anc [rows]: bit a of a row's mask is set if it sees row a of
 * its sequence (a tree's: its ancestors and itself); NULL: chains (every row sees those before it and
 * itself).  Row r of a sequence of L committed tokens is written at token L + r and stands at position L +
 * depth, depth the count of rows before it that it sees; its parent is the last of those. */
typedef struct mj_batch {
    const int32_t* row_start; /* device [n_seqs + 1], not decreasing, from 0 */
    const uint64_t* anc;      /* device [rows], or NULL */
    int n_seqs;
    int rows;                 /* rows of the arrays (those from row_start[n_seqs] on are left as they are) */
    int max_rows;
} mj_batch;

/* Room for the batch's rows: every block of a sequence that rows L .. L + rows - 1 go to gets a page of its
 * own, where it has none or one that others name too (refs other than 1).  The lowest free pages are
 * taken, in order of the sequences and their blocks.  A sequence is served if its table row has the
 * entries and the pages that it and all before it lack are there; others stay as they are (a sequence that
 * lacks nothing is always served).  A shared page loses a reference for each sequence that leaves it, all
 * counted as before the call; of the block that holds committed tokens these are copied in all layers
 * (in groups of eight).  out int32 [n_seqs][4]: 1 if served, pages taken, then the page copied from
 * and to (-1: none).  A sequence with rows that is not served has no part in the step: nothing of it is appended
 * or kept (its attention and its drafts' acceptance are formed, of what there is, and mean nothing). */
mj_status mj_pages_reserve(mj_ctx* ctx, const mj_pages* pages, const mj_batch* batch, int32_t* out);
/* Sequence s becomes a branch of from[s]: what it had is given back, the pages of the source's committed
 * tokens gain a reference, the length is the source's.  from [n_seqs]: outside [0, n_seqs), or s itself:
 * s stays as it is; so it does if the source has an entry of its own in `from`. */
mj_status mj_pages_fork(mj_ctx* ctx, const mj_pages* pages, const int32_t* from);
/* Sequence s cut to len[s] tokens if that is not negative: blocks behind its length lose their pages,
 * also those that were reserved for rows not kept.  len [n_seqs] (pages->lens itself: only these).
 * A page whose count comes to 0 is free. */
mj_status mj_pages_truncate(mj_ctx* ctx, const mj_pages* pages, const int32_t* len);
/* The accepted rows of a pass kept: rows path[0] .. path[accepted] of a sequence (accepted [n_seqs], path
 * [rows] at the sequence's first row, as mj_accept_rows gives them) are moved to its tokens L, L + 1, ...
 * in all layers, and lens_out[s] = L + accepted + 1 (accepted below 0, or no rows: L).  path NULL: the rows
 * of a chain, in place already.  An entry that names no row of the sequence moves nothing.  A sequence whose
 * rows were not all appended, because it had no room, keeps none: lens_out[s] = L.  lens_out [n_seqs] may be
 * pages->lens. */
mj_status mj_pages_commit(mj_ctx* ctx, const mj_pages* pages, const mj_batch* batch,
                          const int32_t* accepted, const int32_t* path, int32_t* lens_out);

/* mj_qkv_append for a batch: queries and keys normed (a NULL weight: not), rotated at their positions,
 * keys and values written to layer `layer` of the sequences' pages (of a sequence without room: not, and never
 * over another sequence's tokens).  qkv fp16 [rows] rows of ld_qkv halves
 * (0: packed; else a multiple of 8), q_out fp16 [rows][n_heads * 128], not over qkv.  Reads n_heads,
 * n_kv_heads, head_dim, rope_dim, rope_base and eps of cfg. */
mj_status mj_paged_append(mj_ctx* ctx, const mj_attn_config* cfg, const mj_pages* pages, int layer,
                          const mj_batch* batch, const void* qkv, int64_t ld_qkv,
                          const void* q_norm_w, const void* k_norm_w, void* q_out);

/* Attention of the batch's rows: softmax(q k^T / sqrt(128)) v over the sequence's committed tokens (window >
 * 0: those less than window before the row's position) and over the rows that the row sees, where they were
 * written.  A row that sees nothing gives zeros.  q fp16 [rows] rows of ld_q halves (0: packed; else a
 * multiple of 8), out likewise, not over q; at most 64 query heads a KV head.
 * Scores, softmax statistics and outputs are summed in fp32; a weight is rounded to fp16 for the product with V
 * (half a step, or at most 2^-34 of the row's greatest weight).  A call repeats bit for bit; a row's result
 * in a batch of other sequences may differ by rounding (the keys are split differently). */
mj_status mj_paged_attn(mj_ctx* ctx, const mj_pages* pages, int layer, const mj_batch* batch,
                        int n_heads, int window, const void* q, int64_t ld_q, void* out,
                        int64_t ld_out, void* ws, size_t ws_bytes);
/* Bytes of workspace that mj_paged_attn takes with these heads and at most max_rows rows a sequence; 0
 * where an argument is out of range. */
size_t mj_paged_workspace(int n_heads, int n_kv_heads, int max_rows);

/* The drafts of a batch checked from given random numbers.  logits fp32 [rows] rows of ld_logits (0: V):
 * row r's are of the token after it; tokens int32 [rows]: the token fed there (a sequence's first row: not a
 * draft).  p = softmax(logits / T) of the sequence's temperature T [n_seqs]; up to 1e-5 (or NaN): all on the
 * greatest logit, the lowest id of equal ones.  A NaN logit counts as -inf; several +inf share the row.
 * From the first row on, the current row's drafts (its children, in order) are tested: draft x with the
 * uniform u = u_accept[its row] is accepted if q(x) > 0, p(x) > 0 and u q(x) rest <= p(x); q the
 * distribution it was drawn from (q fp32 [rows] rows of ld_q, the parent's row; chains only; negative
 * and NaN count as 0) or 1 (q NULL: drafts that are certain), rest 1 less p of the drafts of the row refused
 * before it (one whose token was refused before has nothing left).  The last row reached samples its token: from p
 * if it has no drafts, else from max(p - q, 0), or (q NULL) from p without the refused tokens; from p
 * where that leaves nothing.  It is the lowest id where the running sum passes u_sample[s] times the whole.
 * accepted int32 [n_seqs]: drafts accepted; path int32 [rows]: the rows kept, the first one included, then
 * -1; token int32 [n_seqs]: the token sampled (-1: a row without any probability; a sequence without
 * rows: accepted 0, token -1).  u in [0, 1).  Sums are held in 64 bits in a fixed order: a call repeats bit
 * for bit.  V at most 2^23. */
mj_status mj_accept_rows(mj_ctx* ctx, const mj_batch* batch, const float* logits, int64_t ld_logits,
                         int V, const int32_t* tokens, const float* q, int64_t ld_q,
                         const float* temperature, const float* u_accept, const float* u_sample,
                         int32_t* accepted, int32_t* path, int32_t* token, void* ws,
                         size_t ws_bytes);
/* Bytes of workspace that mj_accept_rows takes with these sizes; 0 where one is out of range. */
size_t mj_accept_workspace(int n_seqs, int rows, int V);

/* lm_head verify -- encodeMetalHead -> maple_lm_head_argmax/reduce
 * (SeedlessDecodeEngine.swift:481-498, SeedlessMetal.swift:3005-3111) for an fp16 head:
 * logits[m][v] = sum_k w[v][k] * x[m][k] (fp32), argmax per row with the lowest id winning
 * ties and banned ids skipped.  x fp16 [M][K], w fp16 [V][K]; out_argmax int32 [M];
 * out_row_max fp32 [M] (nullable): the row's largest logit; out_row_logsumexp fp32 [M]
 * (nullable): ln sum_v exp(logits[m][v] / temperature) over the ids not banned, so that
 * ln p = logits / T - logsumexp is LogitsProcessor.probabilities' softmax
 * (LogitsProcessor.swift:168-189; needs temperature > 1e-5, otherwise ignored);
 * out_logits fp32 [M][V] (nullable; written when sampling).  banned int32 [n_banned] device
 * (nullable), n_banned <= 64 (the reference stages at most 16, SeedlessDecodeEngine.swift:470). */
mj_status mj_lm_head_verify(mj_ctx* ctx, const void* x, const void* w, int M, int K, int V,
                            const int32_t* banned, int n_banned, float temperature,
                            int32_t* out_argmax, float* out_row_max, float* out_row_logsumexp,
                            float* out_logits);

/* lm_head verify over the Maple checkpoint's 4-bit head -- maple_lm_head_argmax/reduce
 * (SeedlessMetal.swift:3005-3111, bound by SeedlessDecodeEngine.swift:481-498 when head_bits
 * is 4, SeedlessDecodeEngine.swift:144): logits[m][v] = sum_k (q[v][k] s[v][k/64] +
 * b[v][k/64]) x[m][k] (fp32), argmax per row with the lowest id winning ties and banned ids
 * skipped.  w uint32 [V][K/8] (8 codes a word, LSB first), scales/biases fp16 [V][K/64],
 * x fp16 [M][K]; group_size must be 64 and K a multiple of 512 (K <= 4096, <= 2048 for
 * M > 16); all four operands 16-byte aligned; n_banned <= 64 (the reference stages at most
 * 16, SeedlessDecodeEngine.swift:470).  Outputs as mj_lm_head_verify. */
mj_status mj_lm_head_verify_q4(mj_ctx* ctx, const void* x, const void* w, const void* scales,
                               const void* biases, int M, int K, int V, int group_size,
                               const int32_t* banned, int n_banned, float temperature,
                               int32_t* out_argmax, float* out_row_max,
                               float* out_row_logsumexp, float* out_logits);

/* Greedy acceptance -- verifyDraftChain (SeedlessDecodeEngine.swift:1574-1603) generalised to
 * a tree: from row 0 step to the lowest-index child whose token equals the current row's
 * argmax; stop when none does.  tokens/argmax int32 [n_rows] device, parents_host as above.
 * out int32 device [2 + 2*n_rows]: out[0] = accepted, out[1] = bonus token,
 * out[2 .. 2+acc] = accepted row path (row 0 first), out[2+n_rows .. 2+n_rows+acc] = emitted
 * tokens (accepted drafts then the bonus). */
mj_status mj_accept_greedy(mj_ctx* ctx, const int32_t* tokens, const int32_t* parents_host,
                           const int32_t* argmax, int n_rows, int32_t* out);

/* Sampled acceptance over the full vocabulary -- SpeculativeSampling.tryAccept / walkDraft
 * (SpeculativeSampling.swift:27-99) with LogitsProcessor.probabilities / samplePrepared
 * (LogitsProcessor.swift:116-189), no penalties.  logits fp32 [rows][V] device (row i = target
 * after feed i), draft int32 [rows-1] device.  q_mode MJ_Q_POINT: q = q_point[i] at the draft
 * token (q_point: a DEVICE float array [rows-1], read by the kernels; NULL = 1 on every draft, the
 * reference default); MJ_Q_UNIFORM: q = 1/V.  q < 0 counts as 0 (max(0, draftQ)): such a
 * draft is rejected without a uniform and the residual is the target itself.
 * Uniforms: Philox4x32-10, key = seed, counter = (row, counter lo, counter hi, 0x6d6a6a76),
 * u0 = accept test, u1 = residual walk (row rows-1: u0 = bonus).  Sums and walks use a fixed
 * blocked order (16-element chunks, 64-chunk blocks) so results are reproducible bit for bit.
 * out int32 device [2]: accepted count, emitted token.  temperature must be > 1e-5. */
#define MJ_Q_POINT 0
#define MJ_Q_UNIFORM 1
mj_status mj_accept_sampled(mj_ctx* ctx, const float* logits, int rows, int V,
                            const int32_t* draft, float temperature, int q_mode,
                            const float* q_point, uint64_t seed, uint64_t counter, int32_t* out);

/* LogitsProcessor options (LogitsProcessor.swift:17-49): temperature > 1e-5; top_p (nucleus,
 * 1 = off, clamped to [0, 1]); repetition (1 = off, > 0), presence and frequency (0 = off)
 * penalties.  hist_tokens / hist_counts (host, n_hist <= MJ_MAX_HIST, tokens distinct): the
 * seen set and the counts the penalties read (prepare, 91-104); drafts accepted in the walk
 * join both before the next row (walkDraft, SpeculativeSampling.swift:86-87). */
#define MJ_MAX_HIST 65536
typedef struct mj_sampling {
    float temperature;
    float top_p;
    float repetition_penalty;
    float presence_penalty;
    float frequency_penalty;
    const int32_t* hist_tokens;
    const int32_t* hist_counts;
    int n_hist;
} mj_sampling;

/* mj_accept_sampled with the options: every row's logits penalised (row i with the history
 * plus drafts 0 .. i-1; the caller's logits are not modified), the bonus and a residual of zero
 * mass sampled through samplePrepared's nucleus (LogitsProcessor.swift:137-164): tokens ranked
 * by e descending, the lower id first among equal e, kept up to the first ranked prefix whose
 * blocked prefix sum reaches top_p * Z, sampled in id order at u * (kept mass). */
mj_status mj_accept_sampled_ex(mj_ctx* ctx, const float* logits, int rows, int V,
                               const int32_t* draft, const mj_sampling* s, int q_mode,
                               const float* q_point, uint64_t seed, uint64_t counter,
                               int32_t* out);

/* ---------------------------------------------------------------- model ------ */
typedef struct mj_model_config {
    int n_layers;
    int H, n_heads, n_kv_heads, head_dim, rope_dim;
    float rope_base, eps;
    int window;            /* sliding window of every layer (0 = full) */
    int64_t kv_capacity;   /* ring slots per layer (>= window + MJ_MAX_ROWS when windowed) */
    int E, top_k, I, gs;
    int vocab;
    /* Maple's layer mix (MapleConfig.isSliding, MapleConfig.swift:145-148; SeedlessAttn.swift
     * 81-83): host arrays [n_layers] overriding window and rope_dim per layer -- sliding layers
     * window w with partial RoPE, full-attention layers 0 / 0 (NoPE).  NULL: every layer takes
     * window / rope_dim.  The non-zero rope dims must all equal rope_dim. */
    const int32_t* layer_window;
    const int32_t* layer_rope_dim;
    /* 4: lm_head is the 4-bit gs64 head of the checkpoint (headBits, MapleConfig.swift:141),
     * uint32 [V][H/8] with lm_head_scales / lm_head_biases fp16 [V][H/64], decoded by
     * mj_lm_head_verify_q4's kernel (H <= 2048).  0 or 16: fp16 [V][H]. */
    int head_bits;
    const void* lm_head_scales;
    const void* lm_head_biases;
} mj_model_config;

typedef struct mj_layer_weights {
    mj_attn_weights attn;
    mj_moe_weights moe;    /* moe.norm_w = post_attention_layernorm */
} mj_layer_weights;

/* A resident stack (SeedlessLayerStack, SeedlessAttn.swift:369-456): caller-owned weights,
 * library-owned KV caches and scratch sized for MJ_MAX_ROWS rows.  layers [n_layers] is copied;
 * the device buffers it points to must outlive the model.  embed fp16 [V][H], final_norm_w
 * fp16 [H], lm_head fp16 [V][H]. */
mj_status mj_model_create(mj_ctx* ctx, const mj_model_config* cfg, const mj_layer_weights* layers,
                          const void* embed, const void* final_norm_w, const void* lm_head,
                          mj_model** out);
mj_status mj_model_destroy(mj_model* model);
/* Committed tokens (SeedlessLayerBlock.offset) and rewind (rewindOffset, SeedlessAttn.swift
 * 319-322; the reject rollback of snapshotForChain 540-586 when writes are append-only). */
int64_t mj_model_offset(const mj_model* model);
mj_status mj_model_rewind(mj_model* model, int64_t offset);
/* Device pointers of layer `layer`'s caches, fp16 [n_kv][kv_capacity][head_dim]. */
mj_status mj_model_kv(mj_model* model, int layer, void** kcache, void** vcache);

/* prefillPrompt (SeedlessDecodeEngine.swift:516-545): feed tokens in chunks of <= chunk rows
 * (<= MJ_MAX_ROWS), commit them, return the argmax after the last token.  Synchronises.  With
 * chunk = MJ_MAX_ROWS up to four chunks share a pass (the same results; an abort voids the pass,
 * and the model goes on from its start). */
mj_status mj_prefill(mj_model* model, const int32_t* tokens, int n, int chunk,
                     int32_t* out_next);

/* stepChainFeeds (SeedlessDecodeEngine.swift:194-228): one pass over the chain `feeds`
 * (M rows), commit all M, return the greedy argmax after each row.  Synchronises. */
mj_status mj_step_chain_feeds(mj_model* model, const int32_t* feeds, int M, int32_t* out_evals);

/* verifyDraftChain (SeedlessDecodeEngine.swift:1574-1603), tree-capable: one pass over rows
 * [y] + draft (parents NULL = chain; else parents[0] = -1 and parents[r] < r over the rows),
 * greedy acceptance on the device, accepted rows compacted into the cache, offset advanced by
 * accepted + 1.  out_tokens [n_draft + 1]: accepted drafts then the bonus token.
 * One device wait per call. */
mj_status mj_verify_greedy(mj_model* model, int32_t y, const int32_t* draft, int n_draft,
                           const int32_t* parents, int32_t* out_accepted, int32_t* out_tokens);

/* verifyDraftSampled (SeedlessDecodeEngine.swift:1541-1571) over the exact fp16 head and the
 * full vocabulary (chain drafts): one pass, device-side sampled acceptance (mj_accept_sampled
 * rules), commit accepted + 1 rows.  out_token = resampled token or bonus.  Unlike
 * mj_accept_sampled, draft and q_point are HOST arrays here: q_point float [n_draft] holds
 * draftQ (qAlong's q on draft i, mergedDraftQ at SeedlessDecodeEngine.swift:1530-1538) and is
 * copied into the pass's descriptor; NULL = 1 on every draft. */
mj_status mj_verify_sampled(mj_model* model, int32_t y, const int32_t* draft, int n_draft,
                            float temperature, int q_mode, const float* q_point, uint64_t seed,
                            uint64_t counter, int32_t* out_accepted, int32_t* out_token);
/* mj_verify_sampled with LogitsProcessor options (mj_accept_sampled_ex's rules) --
 * verifyDraftSampled (SeedlessDecodeEngine.swift:1541-1571) with the processor's penalties
 * and nucleus. */
mj_status mj_verify_sampled_ex(mj_model* model, int32_t y, const int32_t* draft, int n_draft,
                               const mj_sampling* s, int q_mode, const float* q_point,
                               uint64_t seed, uint64_t counter, int32_t* out_accepted,
                               int32_t* out_token);

/* Debug capture for layer-by-layer checks: when set, each pass copies h after the embedding
 * and after every layer into h_capture fp16 [n_layers+1][MJ_MAX_ROWS][H], the routing into
 * inds_capture int32 [n_layers][MJ_MAX_ROWS][top_k] and the head logits into logits_capture
 * fp32 [MJ_MAX_ROWS][V] (device pointers, any may be NULL; all NULL disables). */
mj_status mj_model_set_capture(mj_model* model, void* h_capture, int32_t* inds_capture,
                               float* logits_capture);

/* The same capture with every block boundary, so each block can be re-run from the exact
 * inputs the device used (no counterpart in the reference; its layer-by-layer checks read
 * MTLBuffers directly).  Device pointers, any may be NULL (all NULL disables); while any is
 * set, passes run without graphs.  R = MJ_MAX_ROWS, rows beyond the pass's M are untouched. */
typedef struct mj_capture {
    void* h;               /* fp16 [n_layers+1][R][H]: after the embedding and after each layer */
    int32_t* inds;         /* int32 [n_layers][R][top_k]: each layer's routing */
    float* logits;         /* fp32 [R][V]: lm_head logits */
    void* attn_out;        /* fp16 [n_layers][R][H]: h after each layer's attention block */
    void* moe_in;          /* fp16 [n_layers][R][H]: the normed MoE input (router and up gather) */
    float* router_logits;  /* fp32 [n_layers][R][E]: router logits */
    void* head_in;         /* fp16 [R][H]: the final-normed rows fed to the lm_head */
    void* kv_rows;         /* fp16 [n_layers][2][n_kv_heads][R][head_dim]: the K and V rows the
                              pass appended (row r at slot (L + r) % C), before any commit */
} mj_capture;
mj_status mj_model_set_capture_ex(mj_model* model, const mj_capture* cap);

/* Use HIP graphs for verify passes (one graph per row count and mode, replayed with a device
 * step descriptor).  On by default. */
mj_status mj_model_set_graphs(mj_model* model, int enable);

/* Per-pass device timing of the last verify call (ms), from HIP events on the model stream. */
float mj_model_last_pass_ms(const mj_model* model);

/* Per-kernel timing for measurement: when enabled, verify passes run without graphs and record
 * HIP events around each launch of the classes below on the model stream (counters reset on
 * every call).  A profiled pass waits behind a 15 ms hold kernel, so its launches are queued
 * before the GPU reaches them, and starts with 8 brackets around a kernel that waits 20 us of
 * wall-clock time: each bracketed time is the kernel's duration plus the timer's own cost, and
 * MJ_KERNEL_TIMER minus 20 us per launch is that cost.  A profiled prefill runs its 64-row chunks
 * as passes of their own: the classes are those passes' kernels, not a shared pass's.
 * mj_model_kernel_ms returns the summed milliseconds and the launch count. */
#define MJ_KERNEL_EXPERT_UP 0   /* bucketed up||gate gather + SwiGLU */
#define MJ_KERNEL_EXPERT_DOWN 1 /* bucketed down gather */
#define MJ_KERNEL_LM_HEAD 2     /* fp16 lm_head + argmax partials */
#define MJ_KERNEL_ATTENTION 3   /* split-K attention + combine */
#define MJ_KERNEL_DENSE 4       /* qkv and o projections */
#define MJ_KERNEL_TIMER 5       /* the same bracket around a 20 us wall-clock hold */
#define MJ_KERNEL_EXPERT_MOE 6  /* up||gate + SwiGLU then down, one launch (passes of at most
                                   32 rows over at most 64 experts, H 2048, intermediate 1024) */
mj_status mj_model_profile(mj_model* model, int enable);
float mj_model_kernel_ms(const mj_model* model, int kernel_class, int64_t* launches);

/* Hardware self-check of the MFMA operand layout the kernels rely on (16x16x32 f16):
 * D = A[16x32] * B[32x16] with A, B fp16 row-major device, D fp32 [16][16] device. */
mj_status mj_selftest_mfma(mj_ctx* ctx, const void* A, const void* B, float* D);

/* ---------------------------------------------------------- draft sources ---- */
/* Host-only drafters that propose the rows a verify pass checks (no device work).
 *
 * Online suffix-tree index -- SuffixDraftIndex (SuffixDraftIndex.swift:12-156): every suffix of
 * the inserted sequences, truncated to max_depth (>= 4), with occurrence counts.  A draft takes
 * the longest suffix of `history` (at most max_depth) that ends at a node with children, then
 * follows the most frequent child mj_suffix_max_spec(match, max_k, alpha) times; equal counts
 * take the lowest token id (the reference's order there is its dictionary's).  out_tokens
 * holds max_k ids; *out_n drafted, *out_match_len the suffix length (0: no match). */
typedef struct mj_suffix_index mj_suffix_index;
mj_status mj_suffix_index_create(int max_depth, mj_suffix_index** out);
mj_status mj_suffix_index_destroy(mj_suffix_index* idx);
mj_status mj_suffix_index_clear(mj_suffix_index* idx);
int64_t mj_suffix_index_tokens(const mj_suffix_index* idx);
mj_status mj_suffix_index_insert(mj_suffix_index* idx, const int32_t* tokens, int n);
mj_status mj_suffix_index_draft(const mj_suffix_index* idx, const int32_t* history, int n,
                                int max_k, double alpha, int32_t* out_tokens, int* out_n,
                                int* out_match_len);
/* MAX_SPEC = alpha * match, at least 1 with a match, at most max_k -- maxSpec (48-53). */
int mj_suffix_max_spec(int match_len, int max_k, double alpha);
/* bestDraft (103-121): the local then the global index (either NULL), longer match first, then
 * the longer draft. */
mj_status mj_suffix_best_draft(const mj_suffix_index* local, const mj_suffix_index* global,
                               const int32_t* history, int n, int max_k, double alpha,
                               int32_t* out_tokens, int* out_n, int* out_match_len);
/* qAlong (123-156): the draft model's q along `draft`, child count over sibling mass from the
 * longest matching suffix; positions past the tree stay 1.  out_q float [n_draft]. */
mj_status mj_suffix_index_q_along(const mj_suffix_index* idx, const int32_t* history, int n,
                                  const int32_t* draft, int n_draft, float* out_q);
/* Prompt-lookup draft -- SuffixSpec.suffixDraft (SuffixSpec.swift:17-55): the longest pattern
 * (<= max_ngram, reference default 16) ending the history, its latest earlier occurrence (one
 * inside the first prompt_len tokens first, when prompt_len > 0), and up to k tokens after it. */
mj_status mj_suffix_draft_pld(const int32_t* history, int n, int k, int max_ngram,
                              int prompt_len, int32_t* out_tokens, int* out_n);
/* treeDraft (SuffixDraftIndex.swift:160-178): best tree draft, else the prompt lookup. */
mj_status mj_tree_draft(const int32_t* history, int n, int k, const mj_suffix_index* local,
                        const mj_suffix_index* global, double alpha, int prompt_len,
                        int32_t* out_tokens, int* out_n);
/* adaptiveDraftK (SuffixSpec.swift:8-15): draft length from the mean accepted length. */
int mj_adaptive_draft_k(double mean_accept, int draft_k);

/* Token recycling -- TokenRecycleIndex (TokenRecycleIndex.swift:9-57): per token the top_k
 * (>= 2) latest candidate successors, newest first; a draft follows first successors until one
 * repeats or is missing. */
typedef struct mj_recycle_index mj_recycle_index;
mj_status mj_recycle_index_create(int top_k, mj_recycle_index** out);
mj_status mj_recycle_index_destroy(mj_recycle_index* r);
mj_status mj_recycle_index_clear(mj_recycle_index* r);
mj_status mj_recycle_index_observe(mj_recycle_index* r, int32_t from_token,
                                   const int32_t* candidates, int n);
mj_status mj_recycle_index_draft(const mj_recycle_index* r, int32_t last, int max_k,
                                 int32_t* out_tokens, int* out_n);
int mj_recycle_index_entries(const mj_recycle_index* r);

#ifdef __cplusplus
}
#endif
#endif
