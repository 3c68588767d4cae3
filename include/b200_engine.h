/*
 * Engine-level C ABI: the B200 counterpart of the runtime's engine wrapper
 * engine_t (board/tp/tp_llama.cpp:289-375), i.e. the call the decode loop
 * makes per matrix: quantise float32 x to Q8_0, run the Q4_0 GEMV, and name
 * the matrix that comes next so its bytes can start moving early.
 *
 * Weights are one contiguous 16-byte-aligned allocation per matrix, either
 * in the GGUF Q4_0 row layout (18-byte blocks, row-major) or re-laid once at
 * load into the engine's tiles (b200_repack_q4_0), which the fast kernel
 * reads. Results are bit-exact to src/llm_kv260/q4_0.py:185-188
 * (gemv_q4_0_f32).
 *
 * All addresses are CUDA device addresses; all functions return 0 or a
 * negative errno value (see gemv_dev.h), and b200_last_error() says why.
 * An engine belongs to one device and one caller thread.
 */
#ifndef B200_ENGINE_H
#define B200_ENGINE_H

#include <stdint.h>

#ifndef B200_API
#define B200_API __attribute__((visibility("default")))
#endif

#ifdef __cplusplus
extern "C" {
#endif

typedef struct b200_engine b200_engine_t;

/* A Q4_0 matrix in device memory: replaces qmat (tp_llama.cpp:105-119), one
 * region instead of four staggered port quarters (HBM has no DDR-bank
 * collisions to dodge). Two layouts:
 *   B200_LAYOUT_ROWS   the GGUF bytes as they are: rows of k/32 18-byte blocks;
 *   B200_LAYOUT_TILES  the engine's re-laid form (b200_repack_q4_0), which the
 *                      fast kernel reads; the same 18 bytes per 32 weights, rows
 *                      padded to a multiple of 16 (b200_tiled_bytes).
 * The reference re-lays its weights at load in the same way for its own
 * engine (tp_llama.cpp:102-118, the gemv2 chunk interleave). */
#define B200_LAYOUT_ROWS 0
#define B200_LAYOUT_TILES 1

typedef struct {
    uint64_t w;  /* first byte of the matrix, 16-byte aligned */
    int rows;
    int k;
    int layout;  /* B200_LAYOUT_ROWS or B200_LAYOUT_TILES */
} b200_qmat_t;

typedef struct {
    int stage_bytes;     /* target bytes per shared-memory pipeline stage (default 16384) */
    int stages;          /* stages in flight per CTA, 1..8 (default 4) */
    int ctas_per_sm;     /* grid = SMs x this (default 2) */
    int l2_policy;       /* weight bytes: 0 evict-first (default), 1 normal, 2 evict-last */
    int pdl;             /* 1: launch with programmatic dependent launch (default 1) */
    int round_mode;      /* Q8_0 rounding: 0 floor(|s|+0.5f) as q4_0.py:96 (default), 1 roundf as tp_llama.cpp:343 */
    int fuse_quantize;   /* b200_gemv_f32: 1 quantise inside each GEMV CTA, 0 a separate quantise kernel (default 0) */
    int prefetch_next;   /* 1: a `next` hint issues an L2 prefetch of that matrix on a side stream (default 0) */
    int xreg_chunks;     /* GGUF-row kernel: unused; kept for the layout of this struct (default 8) */
    int kslices;         /* tile kernel: split each row's block dots over at least this many thread slices: 1, 2 or 4 (default 1) */
} b200_engine_config_t;

/* Replaces engine_t::probe + engine_t::open (tp_llama.cpp:303-317). */
B200_API int b200_engine_open(b200_engine_t **e, int device);
B200_API int b200_engine_close(b200_engine_t *e);
B200_API int b200_engine_get_config(b200_engine_t *e, b200_engine_config_t *cfg);
B200_API int b200_engine_set_config(b200_engine_t *e, const b200_engine_config_t *cfg);
/* Queue work on the caller's cudaStream_t (NULL: the legacy default stream).
 * Until this is called the engine uses a non-blocking stream of its own.
 * Serving calls (b200_kv_*, b200_sample, b200_rope, b200_rms_norm) and graph
 * launches on the new stream wait for those queued on the old one, which must
 * still exist (they share scratch, and one reads what another wrote); calls
 * that are being recorded do not. */
B200_API int b200_engine_set_stream(b200_engine_t *e, void *stream);
B200_API void *b200_engine_stream(b200_engine_t *e);

/* Replaces engine_t::gemv (tp_llama.cpp:355-374): y[rows] = W x for float32
 * x[k]; `next` (may be NULL) is the matrix the caller passes next. */
B200_API int b200_gemv_f32(b200_engine_t *e, const b200_qmat_t *W, uint64_t x, uint64_t y, const b200_qmat_t *next);
/* The same over an already-quantised x in the engine layout, int8[k] then
 * float32[k/32] (q4_0.py:193-200); this is gemv_dev_start's computation. */
B200_API int b200_gemv_q8(b200_engine_t *e, const b200_qmat_t *W, uint64_t xpacked, uint64_t y, const b200_qmat_t *next);
/* Replaces engine_t::quantize_x (tp_llama.cpp:330-352) with the contract's
 * rounding by default: x float32[k] -> xpacked int8[k] + float32[k/32]. */
B200_API int b200_quantize_q8_0(b200_engine_t *e, uint64_t x, uint64_t xpacked, int k);
/* Replaces engine_t::prefetch (tp_llama.cpp:318-323): L2 prefetch of W. */
B200_API int b200_prefetch(b200_engine_t *e, const b200_qmat_t *W);

/* Bytes of the tile layout of a rows x k matrix (0 for an unusable shape). */
B200_API uint64_t b200_tiled_bytes(int rows, int k);
/* Re-lay GGUF Q4_0 rows at `src` (2-byte aligned) into tiles at `dst`
 * (16-byte aligned, b200_tiled_bytes(rows, k) bytes) on the engine's stream. */
B200_API int b200_repack_q4_0(b200_engine_t *e, uint64_t src, int rows, int k, uint64_t dst);

/* b200_gemv_f32 plus the greedy pick over its output, fused into the GEMV
 * (the lm_head call of a decode token): y as b200_gemv_f32, and the 8 bytes at
 * `out` as b200_argmax_f32 over y[0..rows). W must be in the tile layout. */
B200_API int b200_gemv_argmax_f32(b200_engine_t *e, const b200_qmat_t *W, uint64_t x, uint64_t y, int index_base,
                                  uint64_t out);

/* Greedy pick over y[0..n) on the device, as the runtime's scan does
 * (tp_llama.cpp:879-882: first index of the largest value): writes the
 * int32 index + index_base, then the float32 value, to the 8 bytes at `out`. */
B200_API int b200_argmax_f32(b200_engine_t *e, uint64_t y, int n, int index_base, uint64_t out);

/* Graphs: record a sequence of engine calls once and replay it with one
 * launch (a decode token is ~70 dependent kernels; replaying them as a CUDA
 * graph with programmatic dependent launch removes the per-kernel CPU cost).
 * Between capture_begin and capture_end the engine's calls are recorded, not
 * run; run every call once before capturing it (first calls set up caches).
 * The engine must be on a stream of its own (not the legacy default). */
typedef struct b200_graph b200_graph_t;
B200_API int b200_capture_begin(b200_engine_t *e);
B200_API int b200_capture_end(b200_engine_t *e, b200_graph_t **g);
B200_API int b200_graph_launch(b200_engine_t *e, b200_graph_t *g);
B200_API int b200_graph_destroy(b200_graph_t *g);
/* Asynchronous copy of `bytes` bytes on the engine's stream, any direction
 * (unified addressing); host memory should be pinned. */
B200_API int b200_copy_async(b200_engine_t *e, uint64_t dst, uint64_t src, uint64_t bytes);

/* The greedy pick of b200_argmax_f32 for callers that cannot allocate device
 * memory. No counterpart in the reference: its engine had no allocator of
 * its own. Opening an engine calls cudaMalloc; this entry point needs no
 * engine and allocates nothing, so it serves code that runs during stream
 * capture, callers whose device memory all comes from their own allocator,
 * and processes where allocating after start-up is not allowed. Its scratch
 * is a fixed 8 KB array inside the library (1024 per-CTA candidates) that
 * every GPU loading the library holds until exit. Runs on the current
 * device, on `stream` (NULL: the legacy default stream); y holds n floats,
 * n <= 33554432 (larger n is refused with -EINVAL); out gets the int32 index
 * + index_base, then the float32 value. The first call on a device looks up
 * the array's device address, so make it before any stream capture. All
 * calls share the array: calls that overlap on the GPU race. */
B200_API int b200_argmax_f32_noalloc(uint64_t y, int n, int index_base, uint64_t out, void *stream);

/* ------------------------------------------------------------ serving ops
 * What a server of several sequences needs around the GEMVs: a key-value
 * cache in pages, attention of one new token per sequence over it, eviction
 * from it by accumulated attention weight, and a sampler. No counterpart in
 * the reference, which has one sequence, a cache [layer][head][position] and
 * a host sampler (tp_llama.cpp:643-705, 809-815, 894-936).
 *
 * All calls queue on the engine's stream, allocate nothing and can be
 * recorded into a graph. Lengths, page tables and sampler settings are read
 * on the device, so the host need not know them; what a call finds there
 * that it cannot use is handled as each call says, never read out of range. */
#define B200_F32 0
#define B200_F16 1
#define B200_BF16 2

/* A paged cache. Slot i of sequence b lies in page table[b][i / page_size] at
 * row i % page_size of each head; a row is head_dim contiguous elements. The
 * strides (in elements) order pages, heads and rows freely, so a pool
 * [page][head][row][head_dim] and one [page][row][head][head_dim] both do. k
 * and v share strides; both addresses and all strides are multiples of 16
 * bytes. lengths[b] (< 0: 0; beyond table_cols * page_size: that) slots are in
 * use. A page number outside [0, n_pages) stands for rows that are not there:
 * they take no part in attention and nothing is written to them. */
typedef struct {
    uint64_t k, v;
    int dtype;           /* B200_F32, B200_F16 or B200_BF16 */
    int n_pages, page_size, n_head_kv;
    int head_dim;        /* a multiple of 8, at most 256 */
    int64_t page_stride, head_stride, row_stride;
    uint64_t table;      /* int32 [batch][table_stride] */
    int64_t table_stride;
    int table_cols;      /* table_cols * page_size <= 1048576 slots a sequence */
    uint64_t lengths;    /* int32 [batch] */
    int batch;
} b200_kv_t;

/* Append: row i of a sequence's new rows goes to slot lengths[b] + i, rounded
 * to the cache's type (to nearest even); its position seen[b] + i and a weight
 * of 0 go beside it. Rows past the last slot, or in a page that is not there,
 * are dropped. */
typedef struct {
    uint64_t k_new, v_new;             /* [n_tokens][n_head_kv][head_dim], strides in elements */
    int dtype;                         /* B200_F32 or the cache's type */
    int n_tokens;
    int64_t token_stride, head_stride; /* both and the addresses multiples of 16 bytes */
    uint64_t offsets;                  /* int32 [batch + 1]: sequence b has rows offsets[b] up to offsets[b + 1],
                                          from 0 to n_tokens in all, not falling (an offset outside [0, n_tokens]
                                          counts as the nearer of these, a row that no sequence has is dropped);
                                          0: row b is sequence b's */
    uint64_t seen;                     /* int32 [batch]: tokens each sequence has had; 0: as lengths */
    uint64_t positions;                /* int32 [batch][n_head_kv][aux_stride], or 0 */
    uint64_t weights;                  /* float [batch][n_head_kv][aux_stride], or 0 */
    int64_t aux_stride;                /* >= table_cols * page_size */
    uint64_t lengths_out, seen_out;    /* int32 [batch], or 0; may be lengths and seen themselves */
} b200_kv_append_t;
B200_API int b200_kv_append(b200_engine_t *e, const b200_kv_t *kv, const b200_kv_append_t *a);

/* Attention of one new token per sequence over its slots in use:
 * s = scale * q . k, out = sum exp(s) v / sum exp(s), lse = log sum exp(s);
 * with no slot left (a score of -infinity leaves none), out = 0 and lse =
 * -infinity; with a score that is NaN or +infinity, out, lse and the head's
 * weights are NaN; an element of out that values which are not finite enter is
 * infinite or NaN. n_head / n_head_kv query heads read each cache head. Dot
 * products, the running maximum and sum and the output are held in float32;
 * the rounding to the output's type is the last step. The weights meet the
 * values with 22 bits (16 over a bfloat16 cache), over a float16 cache those
 * below 2^-26 of the row's largest to within 2^-48 of that. With weights_out the
 * weights of the softmax, summed over the query heads of a cache head, are
 * added up: weights_out = decay * weights +
 * sum, for slots in use (others are not written). */
typedef struct {
    uint64_t q, out;                   /* [batch][n_head][head_dim], strides in elements, rows contiguous */
    int dtype;                         /* of both: the cache's type, or B200_F32 with a B200_F16 cache */
    int n_head;                        /* a multiple of n_head_kv */
    int64_t q_batch_stride, q_head_stride, out_batch_stride, out_head_stride;
    float scale;
    uint64_t lse;                      /* float [batch][n_head], or 0 */
    uint64_t weights;                  /* float [batch][n_head_kv][aux_stride]; 0: as zeros */
    uint64_t weights_out;              /* the same shape, may be `weights` itself; 0: not wanted */
    int64_t aux_stride;
    float decay;
    uint64_t workspace;                /* b200_kv_attend_workspace() bytes, 16-byte aligned; holds nothing between calls */
    uint64_t workspace_bytes;
} b200_kv_attend_t;
/* Bytes a call with these sizes needs, the more of them with weights_out (0 for unusable sizes). */
B200_API uint64_t b200_kv_attend_workspace(const b200_kv_t *kv, int n_head, int with_weights);
B200_API int b200_kv_attend(b200_engine_t *e, const b200_kv_t *kv, const b200_kv_attend_t *a);
/* 1 if a b200_kv_attend or b200_kv_attend_chunk call of this engine was recorded into a graph since
 * this was asked last, else 0: the graph holds the call's workspace, which
 * then has to outlive it. */
B200_API int b200_engine_recorded(b200_engine_t *e);

/* Eviction: each head of a sequence with more than `budget` slots in use keeps
 * the tokens at positions >= seen[b] - recent or < sinks, then those of the
 * largest weights (the lower slot where equal; NaN is the smallest), budget in
 * all (of tokens kept by position, too, the lower slots if they are more).
 * The i-th kept slot >= budget moves into the i-th slot < budget that was
 * given up -- key and value rows, weight and position -- and nothing else
 * moves, so slots are not in the order of their positions afterwards
 * (attention does not mind). Slots < the new length of weights_out and
 * positions_out are written, no others. Sequences within budget are left as
 * they are. Pages must not be shared between sequences that are cut, and those
 * of their slots in use must all be there: of a kept slot without a page only
 * weight and position move, and beside them then lies the row of the token
 * that was given up. */
typedef struct {
    uint64_t weights, weights_out;     /* float [batch][n_head_kv][aux_stride]; may be the same */
    uint64_t positions, positions_out; /* int32, the same shape; may be the same */
    int64_t aux_stride;
    uint64_t seen;                     /* int32 [batch] */
    uint64_t lengths_out;              /* int32 [batch], or 0; may be the cache's lengths */
    int budget, recent, sinks;         /* budget >= 1, recent + sinks <= budget */
} b200_kv_evict_t;
B200_API int b200_kv_evict(b200_engine_t *e, const b200_kv_t *kv, const b200_kv_evict_t *a);

/* Sampling. With x a row's logits (NaN counts as -infinity), M the largest and
 * T the temperature, token i weighs w_i = floor(2^40 * 2^((x_i - M) * c)),
 * c = log2(e) / T, whole numbers whose sums do not depend on an order. Filters
 * keep a prefix of the tokens in falling order of x (the lower index where
 * equal): top_k its first k; top_p the fewest of those whose weight reaches
 * p of theirs together, at least one; min_p those with
 * 2^((x_i - M) * c) >= min_p. The token is the first whose weight, added to
 * that of all kept tokens of lower index, passes u of the whole; u and p count
 * in units of 2^-24. So the same logits and u give the same token on every
 * run. A temperature of 0 (or less, or NaN) takes the lowest index of the
 * largest logit. Where M is +infinity, the tokens at it weigh the same and all
 * others nothing; a row with no logit above -infinity gives token -1. */
typedef struct {
    uint64_t logits;                   /* [batch][row_stride] */
    int dtype;                         /* B200_F32, B200_F16 or B200_BF16 */
    int batch;
    int n_vocab;                       /* at most 4194304 */
    int64_t row_stride;
    uint64_t temperature;              /* float [batch]; 0: all 1 */
    uint64_t top_k;                    /* int32 [batch], <= 0 in a row: off; 0: off */
    uint64_t top_p;                    /* float [batch], >= 1 or NaN in a row: off; 0: off */
    uint64_t min_p;                    /* float [batch], <= 0 or NaN in a row: off; 0: off */
    uint64_t u;                        /* float [batch] in [0, 1) (clamped to it; NaN: 0) */
    uint64_t token;                    /* int32 [batch] */
    uint64_t logprob;                  /* float [batch]: log of the token's share of the kept weight, or 0 */
} b200_sample_t;
B200_API int b200_sample(b200_engine_t *e, const b200_sample_t *s);

/* --------------------------------------------------- prompts in chunks
 * What new tokens pass through on their way into the caches of several
 * sequences, prompts in chunks and single tokens mixed: pages and slots, the
 * norm in front of a matrix, rotary positions with the store into the cache,
 * and attention of all new tokens. As the calls above, they queue on the
 * engine's stream, allocate nothing, can be recorded, and read on the device
 * what the host need not know. */

/* Pages and slots for new tokens. A pool's free pages are a stack, free[0] up
 * to free[count - 1]; sequence b holds the pages in the first held[b] columns
 * of its table row and asks for new_tokens[b] slots behind its lengths[b], or,
 * with a negative number, is done (its length becomes 0). It wants
 * ceil((length + new) / page_size) pages. First, all pages beyond what a
 * sequence wants go onto the stack, in the order of sequences and columns
 * (those that it has no room for are lost). Then, in the same order, sequences
 * take what they lack from its top. A sequence gets all or nothing: nothing
 * where the table has no slots for its tokens, or where it lacks pages and all
 * lacks up to its own exceed the stack (so later ones that lack pages get none
 * either). Its pages, length and seen then stay as they were.
 *
 * Tokens are numbered by sequence: b's are offsets[b] up to offsets[b + 1],
 * whether it got its slots or not. For token t of sequence b, its i-th:
 * sequences[t] = b, positions[t] = seen[b] + i, and slots[t] = page *
 * page_size + row, or -1 where it got none or the page is not in the pool. For
 * t behind the last sequence's tokens all three are -1. Table entries that
 * were given up keep their value, and free entries behind the count stay: with
 * held_out, free_count_out, lengths_out and seen_out elsewhere a call can be
 * repeated. Only page_size, table, lengths and n_pages of the cache are used. */
typedef struct {
    uint64_t new_tokens;               /* int32 [batch] */
    uint64_t held, held_out;           /* int32 [batch], may be the same */
    uint64_t free_pages;               /* int32 [free_capacity] */
    int free_capacity;
    uint64_t free_count, free_count_out; /* int32 [1], may be the same */
    uint64_t offsets;                  /* int32 [batch + 1], written; n_tokens where they would be more */
    int n_tokens;                      /* of slots, positions and sequences */
    uint64_t slots;                    /* int64 [n_tokens], or 0 */
    uint64_t positions, sequences;     /* int32 [n_tokens], or 0 */
    uint64_t granted;                  /* int32 [batch]: tokens that got slots, or 0 */
    uint64_t seen, seen_out;           /* int32 [batch], or 0; seen 0: as lengths */
    uint64_t lengths_out;              /* int32 [batch], may be the cache's lengths */
} b200_kv_plan_t;
B200_API int b200_kv_plan(b200_engine_t *e, const b200_kv_t *kv, const b200_kv_plan_t *a);

/* Rotary positions. The first rot_dim elements of a head are pairs (x, y): i
 * and i + rot_dim / 2, or, interleaved, 2 i and 2 i + 1. Pair i of a token at
 * position p becomes mscale * (x cos a - y sin a, y cos a + x sin a) with the
 * angle a = p * freqs[i], held in units of 2^-64 turns, so that the angle of
 * any position is good to 2^-28 turns; the other elements are copied. With a
 * cache, k's rotated rows go to its rows slots[t], and v's rows beside them,
 * both in the cache's type (a slot outside the pool, as -1, is dropped; k_out
 * is not used; no two tokens have one slot). q, k and v in float32 may go to any type, others to their own.
 * A row may go where it comes from, in its own type and with the same strides;
 * otherwise inputs and outputs do not overlap, nor do an output's rows. */
typedef struct {
    uint64_t q, q_out;                 /* [n_tokens][n_head][head_dim], strides in elements; 0: no q */
    int n_head;
    int64_t q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride;
    uint64_t k, k_out;                 /* [n_tokens][n_head_kv][head_dim]; 0: no k */
    int n_head_kv;
    int64_t k_token_stride, k_head_stride, k_out_token_stride, k_out_head_stride;
    uint64_t v;                        /* as k; only with a cache, where it may be 0 */
    int64_t v_token_stride, v_head_stride;
    int dtype;                         /* of q, k, v */
    int out_dtype;                     /* of q_out, k_out: dtype, or any with B200_F32 */
    int n_tokens;
    int head_dim;                      /* a multiple of 8, at most 256 */
    int rot_dim;                       /* even, 2 up to head_dim */
    int interleaved;
    uint64_t positions;                /* int32 [n_tokens] */
    uint64_t freqs;                    /* uint64 [rot_dim / 2], see b200_rope_freqs */
    float mscale;
    uint64_t slots;                    /* int64 [n_tokens], with a cache */
} b200_rope_t;
B200_API int b200_rope(b200_engine_t *e, const b200_kv_t *kv, const b200_rope_t *a);

/* The frequencies of b200_rope on the host, base^(-2 i / rot_dim) radians for
 * pair i, divided by factors[i] (NULL: 1, as a model file's rope_freqs), and for
 * contexts longer than a model was trained for:
 *   LINEAR divided by factor;
 *   BANDS  by the turns n that a pair makes in `context` positions: divided by
 *          factor where n <= low, as it is where n >= high, the mean of the two
 *          weighted by (n - low) / (high - low) between;
 *   YARN   the same over the index i of a pair instead: as it is up to the pair
 *          with `high` turns (its index rounded down), divided from the one with
 *          `low` on (rounded up), the mean weighted by i between. */
#define B200_ROPE_PLAIN 0
#define B200_ROPE_LINEAR 1
#define B200_ROPE_BANDS 2
#define B200_ROPE_YARN 3
B200_API int b200_rope_freqs(uint64_t *freqs, int rot_dim, double base, const float *factors, int scaling, double factor,
                             double context, double low, double high);

/* Residual addition and root-mean-square norm: r = residual + x (x alone where
 * residual is 0), residual_out = r, y = r / sqrt(mean(r^2) + eps) * weight, in
 * float32 with one rounding per output. y goes to out, and with q8 row by row
 * to the engine's Q8_0 form, int8[k] then float32[k / 32], as
 * b200_quantize_q8_0 makes it and b200_gemv_q8 reads it. An output's rows do not
 * overlap, and nothing else but what is said below. */
typedef struct {
    uint64_t x;                        /* [n_rows][k], strides in elements, rows contiguous */
    int dtype;
    uint64_t residual, residual_out;   /* or 0; may be the same, with the same stride */
    int residual_dtype;                /* dtype, or B200_F32 */
    uint64_t weight;                   /* float32 [k] */
    uint64_t out;                      /* or 0; may be x, its rows as many bytes apart */
    int out_dtype;                     /* dtype, or any with B200_F32 */
    uint64_t q8;                       /* or 0 */
    int n_rows, k;                     /* k: a multiple of 8 (of 32 with q8), at most 32768 */
    int64_t x_stride, residual_stride, residual_out_stride, out_stride;
    int64_t q8_stride;                 /* bytes, >= k + k / 8 */
    float eps;
} b200_rms_norm_t;                     /* addresses and strides are multiples of 16 bytes, q8's of 4 */
B200_API int b200_rms_norm(b200_engine_t *e, const b200_rms_norm_t *a);

/* Attention of each sequence's new tokens, which are its last slots in use
 * (b200_kv_append or b200_rope has put them there): with n = offsets[b + 1] -
 * offsets[b], its row i stands at slot p = lengths[b] - n + i and sees the slots
 * up to p, with a window > 0 the last `window` of them. out = sum exp(s) v / sum
 * exp(s), s = scale * q . k, lse = log sum exp(s), with the conventions of
 * b200_kv_attend for rows that see nothing (p < 0, pages that are not there,
 * scores of -infinity), for NaN and for infinities; what a row does not see has
 * no influence on it, to the bit, whatever it holds, and a value that is not
 * finite makes its element infinite or NaN in every row that sees it, however
 * small its weight. Rows that no sequence has are left as they are. Dot
 * products, maximum, sum and output are held in float32. With 16-bit queries the
 * weights of the softmax are rounded to the cache's type before they meet the
 * values (as much as the output is; in float16 one below 2^-24 of the row's
 * largest to within 2^-35 of that). With float32 queries over a float16 cache
 * the weights keep 22 bits however small they are (down to 2^-111), and an
 * element of q, 2^-j of its row's largest, min(22, 50 - j); over a float32 cache
 * nothing is rounded. */
typedef struct {
    uint64_t q, out;                   /* [n_tokens][n_head][head_dim], strides in elements, rows contiguous, without
                                          overlap; addresses and strides are multiples of 16 bytes */
    int dtype;                         /* of both: the cache's type, or B200_F32 with a B200_F16 cache */
    int n_tokens, n_head;              /* n_head: a multiple of n_head_kv, at most 4096 times it */
    int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
    uint64_t offsets;                  /* int32 [batch + 1], as in b200_kv_append_t */
    float scale;                       /* positive, 1e-37 to 1e37 */
    int window;                        /* 0: none */
    uint64_t lse;                      /* float [n_tokens][n_head], or 0 */
    uint64_t workspace;                /* b200_kv_chunk_workspace() bytes, 16-byte aligned; holds nothing between calls */
    uint64_t workspace_bytes;
} b200_kv_chunk_t;
/* Bytes that calls with these sizes need on any device of this machine, whatever
 * the number of tokens (0 for unusable sizes). */
B200_API uint64_t b200_kv_chunk_workspace(const b200_kv_t *kv, int dtype, int n_head);
B200_API int b200_kv_attend_chunk(b200_engine_t *e, const b200_kv_t *kv, const b200_kv_chunk_t *a);

/* Block until the engine's queued work is done (bounded; -ETIMEDOUT). */
B200_API int b200_engine_sync(b200_engine_t *e, int timeout_ms);
/* Device status word (see gemv_dev_status); reading clears it. */
B200_API int b200_engine_status(b200_engine_t *e, unsigned *status);
/* Launch shape the GEMV would use for W (for roofline accounting). */
B200_API int b200_gemv_plan(b200_engine_t *e, int rows, int k, int layout, int fused_f32, int *grid, int *smem_bytes);

B200_API int b200_device_count(void);
/* Message for the last error on this thread (never NULL). */
B200_API const char *b200_last_error(void);

#ifdef __cplusplus
}
#endif
#endif
