/*
 * fa_hip.h -- C ABI of the MI355X FlashAttention library (libfa_hip.so).
 *
 * The drop-in boundary for the reference crate amaye15/flash-attention-cpu:
 * every entry point below replaces one public Rust function of that crate
 * (cited per declaration) with the same argument meaning: row-major f32
 * Q/K/V/O, [batch, heads, seq, d_head] for the multi-head forms, the causal
 * flag of FlashAttentionConfig, and the implicit softmax scale
 * 1/sqrt(d_head) computed in f32.  Rust slices become (pointer, length)
 * pairs so the crate's shape asserts keep their meaning; a failed assert
 * becomes a non-zero status instead of a panic, naming the same operand.
 *
 * All compute runs on the GPU (hand-written gfx950 kernels loaded from a
 * code object with hipModuleLoad); there is no CPU fallback.  Host-slice
 * entry points copy to device memory, launch, copy back and synchronise;
 * the _device forms take caller-owned device pointers and the caller's HIP
 * stream and return as soon as the kernels are queued.
 *
 * Thread safety: every entry point may be called from several threads at
 * once (the crate's functions are Sync).  Up to four host-slice calls per
 * device run concurrently, each on its own stream, device staging buffer and
 * pinned copy ring; further callers wait until one of those four finishes.
 * Calls that several threads make on one stream are queued one after the
 * other, all kernels of one before those of the next.
 */
#ifndef FA_HIP_H
#define FA_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ------------------------------------------------------ */
#define FA_OK 0
#define FA_ERR_Q_SHAPE 1      /* "q shape mismatch"   src/common.rs:51, :87 */
#define FA_ERR_K_SHAPE 2      /* "k shape mismatch"   src/common.rs:52, :88 */
#define FA_ERR_V_SHAPE 3      /* "v shape mismatch"   src/common.rs:53, :89 */
#define FA_ERR_OUT_SHAPE 4    /* "out shape mismatch" src/common.rs:54, :90 */
#define FA_ERR_INVALID_ARG 5  /* NULL pointer with a non-zero length, bad variant/option */
#define FA_ERR_UNSUPPORTED 6  /* d_head > 256 with 16-bit inputs or a forced split-KV path,
                                 d_head > 2048 with a forced stream split or a split count, or a
                                 size beyond 32-bit row indexing (f32 heads of any width run the
                                 flash kernels) */
#define FA_ERR_NO_DEVICE 7    /* no HIP device visible */
#define FA_ERR_MODULE 8       /* code object missing / unloadable (FA_HIP_MODULE), or an operator's
                                 that another build of the library made */
#define FA_ERR_ALLOC 9        /* device allocation failed, or the request exceeds the free
                                 device memory (checked before anything is queued) */
#define FA_ERR_LAUNCH 10      /* kernel launch failed */
#define FA_ERR_COPY 11        /* host<->device copy or synchronisation failed */
#define FA_ERR_SCRATCH 12     /* fa_device_ex_noalloc: the call needs more split workspace than
                                 the 64 MiB scratch array, or the array is unavailable */

/* Human-readable text for a status code (static storage). */
const char* fa_status_string(int status);

/* ---- configuration ------------------------------------------------------
 * Mirrors FlashAttentionConfig (src/common.rs:16-36).  block_size_q and
 * block_size_kv are accepted for signature parity; the GPU tiles are fixed
 * per d_head and results do not depend on block sizes beyond rounding, as
 * in the reference (tests/correctness.rs:137-171).  causal: key j is
 * visible to query i iff j <= i, in absolute indices (src/naive.rs:37). */
typedef struct fa_config {
    size_t block_size_q;   /* default 64  */
    size_t block_size_kv;  /* default 128 */
    uint8_t causal;        /* default 0   */
} fa_config;

/* FlashAttentionConfig::default() -- src/common.rs:28-36 */
fa_config fa_config_default(void);

/* ---- single head, host slices ------------------------------------------
 * q: [seq_len_q, d_head], k/v: [seq_len_k, d_head], out: [seq_len_q, d_head].
 * Checks q/k/v/out lengths in that order (check_shapes, src/common.rs:41-57);
 * if seq_len_q, seq_len_k or d_head is 0 returns FA_OK without touching out.
 * config == NULL means fa_config_default(). */

/* flash_attention_v1 -- src/v1.rs:51-123 (FA-1: per-step normalisation,
 * no causal tile skip) */
int fa_v1(const float* q, size_t q_len, const float* k, size_t k_len, const float* v, size_t v_len,
          size_t seq_len_q, size_t seq_len_k, size_t d_head, const fa_config* config, float* out,
          size_t out_len);
/* flash_attention_v2 -- src/v2.rs:49-121 (FA-2: deferred normalisation,
 * causal skip of fully-future tiles) */
int fa_v2(const float* q, size_t q_len, const float* k, size_t k_len, const float* v, size_t v_len,
          size_t seq_len_q, size_t seq_len_k, size_t d_head, const fa_config* config, float* out,
          size_t out_len);
/* flash_attention_v3 -- src/v3.rs:61-133 (v2 with the next tile's QK^T
 * overlapped with the current softmax + PV) */
int fa_v3(const float* q, size_t q_len, const float* k, size_t k_len, const float* v, size_t v_len,
          size_t seq_len_q, size_t seq_len_k, size_t d_head, const fa_config* config, float* out,
          size_t out_len);
/* flash_attention (alias of v2) -- src/lib.rs:87 */
int fa_attention(const float* q, size_t q_len, const float* k, size_t k_len, const float* v,
                 size_t v_len, size_t seq_len_q, size_t seq_len_k, size_t d_head,
                 const fa_config* config, float* out, size_t out_len);

/* ---- batched multi-head, host slices ----------------------------------
 * q/out: [batch, heads, seq_len_q, d_head], k/v: [batch, heads, seq_len_k,
 * d_head], contiguous (multihead_dispatch, src/common.rs:72-101).  All
 * batch*heads slices run in one launch. */

/* flash_attention_multihead_v1 -- src/v1.rs:134-159 */
int fa_multihead_v1(const float* q, size_t q_len, const float* k, size_t k_len, const float* v,
                    size_t v_len, size_t batch, size_t heads, size_t seq_len_q, size_t seq_len_k,
                    size_t d_head, const fa_config* config, float* out, size_t out_len);
/* flash_attention_multihead_v2 -- src/v2.rs:132-157 */
int fa_multihead_v2(const float* q, size_t q_len, const float* k, size_t k_len, const float* v,
                    size_t v_len, size_t batch, size_t heads, size_t seq_len_q, size_t seq_len_k,
                    size_t d_head, const fa_config* config, float* out, size_t out_len);
/* flash_attention_multihead_v3 -- src/v3.rs:144-169 */
int fa_multihead_v3(const float* q, size_t q_len, const float* k, size_t k_len, const float* v,
                    size_t v_len, size_t batch, size_t heads, size_t seq_len_q, size_t seq_len_k,
                    size_t d_head, const fa_config* config, float* out, size_t out_len);
/* flash_attention_multihead (alias of multihead v2) -- src/lib.rs:86 */
int fa_attention_multihead(const float* q, size_t q_len, const float* k, size_t k_len,
                           const float* v, size_t v_len, size_t batch, size_t heads,
                           size_t seq_len_q, size_t seq_len_k, size_t d_head,
                           const fa_config* config, float* out, size_t out_len);

/* ---- device-resident, stream-ordered -----------------------------------
 * Same computation as fa_multihead_vN on device pointers (hipMalloc'd or any
 * device-accessible memory), queued on `stream` (a hipStream_t; NULL = the
 * default stream).  No length checks are possible on raw pointers; zero
 * dims return FA_OK with nothing queued.  Every variant picks the split-KV
 * (flash-decoding) kernels for short query blocks against long key ranges,
 * and smaller workgroups (v2, v3) or a key or stream split on grids smaller
 * than the GPU (v1 on kernels of its own that keep its per-step normalisation and visit every key, causal
 * or not).  Their partials go to a
 * workspace kept per stream (up to 256 MiB; larger ones are allocated and
 * released stream-ordered around the call): the first call on a stream that
 * needs more allocates it with hipMalloc, and buffers are kept (outgrown ones
 * included) until fa_release_stream_workspace or the end of the process, so
 * graphs captured with these calls stay valid.  A call made under graph
 * capture takes the stream's buffer over for the graph (make one eager call
 * on the stream before each capture; the next eager call allocates anew), so
 * replays never share partials with other calls.  Calls on one stream share
 * its buffer in stream order; a stream handle value reused after
 * hipStreamDestroy inherits the buffer, so release a stream's workspace (or
 * synchronise it) before destroying it if its handle may be reused.
 * These have no single counterpart in the reference (its API takes host
 * slices); they are the device form of the multihead entry points. */
int fa_device_v1(void* stream, const float* q, const float* k, const float* v, size_t batch,
                 size_t heads, size_t seq_len_q, size_t seq_len_k, size_t d_head,
                 const fa_config* config, float* out);
int fa_device_v2(void* stream, const float* q, const float* k, const float* v, size_t batch,
                 size_t heads, size_t seq_len_q, size_t seq_len_k, size_t d_head,
                 const fa_config* config, float* out);
int fa_device_v3(void* stream, const float* q, const float* k, const float* v, size_t batch,
                 size_t heads, size_t seq_len_q, size_t seq_len_k, size_t d_head,
                 const fa_config* config, float* out);
/* Frees the split workspace kept for `stream` on the current device (and the
 * buffers it outgrew), after synchronising the stream.  For servers that
 * create and destroy streams: call it before hipStreamDestroy.  Graphs
 * captured with split calls on `stream` must not be replayed afterwards.  A
 * later split call on the stream allocates a new workspace.  No counterpart
 * in the reference (the crate's scratch is per call). */
int fa_release_stream_workspace(void* stream);

/* ---- extension: explicit scale and path control ------------------------
 * Not in the reference.  softmax_scale <= 0 or NaN keeps the reference's
 * 1/sqrt(d_head).  path: FA_PATH_AUTO (what fa_device_vN does),
 * FA_PATH_PREFILL (query-block kernel; with num_splits > 1, each block's
 * keys are divided over num_splits workgroups whose partials are merged),
 * FA_PATH_SPLITKV (16-row decode tiles; with one split -- num_splits = 1, or
 * chosen -- each tile is written directly, no merge), FA_PATH_SPLITKV_ROWS
 * (row-streaming split-KV for seq_len_q <= 4: K and V read as whole rows,
 * dot products on the vector ALUs; f32, d_head % 4 == 0 and 16-byte aligned
 * operands, else FA_ERR_UNSUPPORTED), FA_PATH_STREAM (query-block kernel
 * with the stream split: the key stages of every (slice, query block) cut
 * into equal runs, one per workgroup -- num_splits workgroups, 0 = one per
 * resident workgroup slot -- with partials merged where a block is shared).
 * Every path takes every variant; v1's split kernels keep its per-step
 * normalisation and visit every key (no causal skip).  AUTO runs
 * decode steps -- seq_len_q <= 32, any batch and key count -- on split-KV
 * (the row-streaming kernel where it applies, else 16-row tiles; 16-bit
 * inputs on the row kernel for one query; for 2 .. 32 queries -- 16 where
 * d_head > 128 -- on a streaming prefill kernel if non-causal, with 256 keys
 * or more, d_head > 32, d_head % 8 == 0 and 16-byte aligned operands, unless
 * that would run as a few short splits, which go to the small prefill grids
 * below), and prefills smaller than the GPU on smaller workgroups whose
 * waves share the keys of a query tile, on the stream split or on the key
 * split, whichever it estimates to be fastest; a 16-bit grid that nearly
 * fills the GPU runs without a workspace.
 * num_splits = 0 lets the library choose (at most 1024). */
#define FA_PATH_AUTO 0
#define FA_PATH_PREFILL 1
#define FA_PATH_SPLITKV 2
#define FA_PATH_SPLITKV_ROWS 3
#define FA_PATH_STREAM 4
/* Element type of Q, K, V (O is always f32). */
#define FA_DTYPE_F32 0
#define FA_DTYPE_BF16 1
#define FA_DTYPE_F16 2
typedef struct fa_launch_opts {
    float softmax_scale;
    int path;
    int num_splits;
    int dtype;   /* FA_DTYPE_*: read by fa_describe_launch; fa_device_ex accepts only F32 */
} fa_launch_opts;

int fa_device_ex(int variant, void* stream, const float* q, const float* k, const float* v,
                 size_t batch, size_t heads, size_t seq_len_q, size_t seq_len_k, size_t d_head,
                 const fa_config* config, const fa_launch_opts* opts, float* out);

/* ---- allocation-free form ------------------------------------------------
 * No counterpart in the reference.  For callers that cannot allocate device
 * memory: code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc.  Same arguments, kernels and results as fa_device_ex,
 * but the split partials (split-KV decode, prefill key split) go to a
 * device-global scratch array of 64 MiB per GPU, held until the process
 * ends, and the call allocates and frees nothing.  Calls whose plan needs a
 * larger workspace return FA_ERR_SCRATCH (out untouched).  Call fa_init()
 * on each device first (it loads the kernels and maps the array; a first
 * call does it itself, which allocates).  All calls on one GPU share its
 * array: calls that may overlap on one GPU (different streams, or graphs
 * replayed concurrently) race on it and must be ordered by the caller. */
int fa_device_ex_noalloc(int variant, void* stream, const float* q, const float* k, const float* v,
                         size_t batch, size_t heads, size_t seq_len_q, size_t seq_len_k, size_t d_head,
                         const fa_config* config, const fa_launch_opts* opts, float* out);

/* ---- 16-bit inputs (bf16 / f16) -------------------------------------------
 * Not in the reference, whose roadmap plans bf16 dot products with f32
 * accumulation (ROADMAP.md, item 2 "bf16 dot-product acceleration").  Q, K, V
 * hold bfloat16 (FA_DTYPE_BF16, raw 16-bit patterns) or IEEE binary16
 * (FA_DTYPE_F16) in the layout of the f32 entry points; O is f32.  QK^T and PV
 * run on 16-bit MFMA with f32 accumulation (every product exact), the softmax
 * in f32, and the probabilities are rounded to the input type for PV (the
 * row sums add up the rounded values), so each output element is within
 * u/(1-u) * max|V| of f32 attention on the same 16-bit inputs (u = 2^-8
 * bf16, 2^-11 f16; f16 probabilities are rounded as 2^7 p, so only those
 * below 2^-21 of the row's reference fall below f16's normal range, adding
 * at most n * 2^-32 * max|V| over a row of n keys).  Causal masking, shape checks and
 * zero-dimension behaviour are those of fa_multihead_v2; d_head <= 256.  The
 * algorithm is v2/v3's (deferred normalisation, causal skip); no variant
 * argument.  opts: softmax_scale, path and num_splits as for fa_device_ex;
 * opts->dtype is ignored.  The split-KV kernels (FA_PATH_SPLITKV, and
 * FA_PATH_SPLITKV_ROWS for seq_len_q = 1, d_head % 8 == 0, d_head > 32, which
 * AUTO picks for decode steps) widen the 16-bit values exactly and compute in
 * f32 without rounding the probabilities. */
int fa_device_lp(int dtype, void* stream, const void* q, const void* k, const void* v, size_t batch,
                 size_t heads, size_t seq_len_q, size_t seq_len_k, size_t d_head,
                 const fa_config* config, const fa_launch_opts* opts, float* out);
/* Host-slice form; lengths count elements. */
int fa_multihead_lp(int dtype, const void* q, size_t q_len, const void* k, size_t k_len,
                    const void* v, size_t v_len, size_t batch, size_t heads, size_t seq_len_q,
                    size_t seq_len_k, size_t d_head, const fa_config* config, float* out,
                    size_t out_len);

/* ---- attention with modified scores ---------------------------------------
 * No counterpart in the reference.  Softmax attention, forward and backward,
 * on device pointers, stream-ordered.  Query i of head h stands at position
 * i' = q_start + i, key j at position j:
 *     x = softmax_scale * (q_i . k_j)
 *     y = softcap > 0 ? softcap * tanh(x / softcap) : x
 *     z = slopes ? y - slopes[h] * |i' - j| : y
 *     key j is visible to query i iff
 *         (!causal || j <= i' || (prefix && j < prefix[b]))  and
 *         (!q_doc  || (q_doc[b][i] == k_doc[b][j] && q_doc[b][i] >= 0))
 *     lse_i = log sum over visible j of e^z,   o_i = sum e^(z - lse_i) v_j
 * A query that sees no key gets o = 0 and lse = -inf.  Document ids may come
 * in any order; tokens with a negative id (padding) see nothing and are seen
 * by none.  Keys and values that a query does not see do not reach it, also
 * where they are infinite or NaN.
 *
 * heads is a multiple of kv_heads: query head h reads key / value head
 * h / (heads / kv_heads).  Q, K, V, O and all gradients have the type `dtype`
 * (products accumulate in f32; 16-bit inputs: probabilities and score
 * gradients are rounded to the type for the products they enter, f16 ones
 * scaled by powers of two so that neither small nor large ones leave the
 * type's range there).  slopes, prefix
 * and lse are f32 / int32 / f32 whatever the type.  d_head <= 256.
 *
 * Layouts: element strides between batches, tokens and heads, columns next to
 * each other; all three 0 means contiguous [batch, heads, seq, d_head].  The
 * token stride is at least d_head and below 2^22 (FA_ERR_UNSUPPORTED beyond);
 * strides of dimensions of one entry are not looked at.  Inputs may share memory between batches or heads
 * (stride 0); outputs may not overlap.  Any alignment works; 16-byte aligned
 * rows (pointers, strides and d_head) are faster. */
typedef struct fa_strides {
    int64_t batch, seq, head;
} fa_strides;

typedef struct fa_score_config {
    int dtype;                 /* FA_DTYPE_* */
    int causal;
    size_t batch, heads, kv_heads, seq_len_q, seq_len_k, d_head;
    int64_t q_start;           /* position of query 0 (a decode step: the cache length) */
    float softmax_scale;       /* <= 0 or NaN: 1/sqrt(d_head) */
    float softcap;             /* 0: none; 16-bit inputs: above 512 slower.  One whose ratio to the
                                  scale, or itself times log2(e), is no normal f32 is refused */
    const float* slopes;       /* [heads], device memory; NULL: no bias */
    const int32_t* q_doc;      /* [batch, seq_len_q], device memory; both or neither */
    const int32_t* k_doc;      /* [batch, seq_len_k] */
    const int32_t* prefix;     /* [batch], device memory; NULL: none; read if causal */
    fa_strides q, k, v, out, dout, dq, dk, dv;
} fa_score_config;

/* O and, if lse != NULL, lse [batch, heads, seq_len_q].  With no keys
 * (seq_len_k = 0) O is zero and lse -inf; any other zero dimension queues
 * nothing. */
int fa_score_forward(void* stream, const fa_score_config* cfg, const void* q, const void* k, const void* v,
                     void* out, float* lse);
/* dQ, dK, dV of fa_score_forward from its inputs, its O and lse and the
 * gradient of O (lse itself gets none; slopes are constants).  Each of dq, dk and dv may be NULL
 * where it is not wanted.  Results do not depend on the order in which
 * workgroups run. */
int fa_score_backward(void* stream, const fa_score_config* cfg, const void* q, const void* k, const void* v,
                      const void* out, const float* lse, const void* dout, void* dq, void* dk, void* dv);

/* ---- rotary positions -------------------------------------------------------
 * No counterpart in the reference.  Column pairs of the first rot_dim columns
 * of each head row are rotated by position * 2 pi * turns[c]:
 *     (a, b) -> gain * (a cos - b sin, a sin + b cos)
 * pairs (c, c + rot_dim / 2), or (2c, 2c + 1) where interleaved; the other
 * columns are copied.  inverse rotates back with the same gain, which is the
 * gradient.  Angles are reduced in 64 bits, so far positions keep their
 * accuracy.  fa_rotary_init (host only) fills a config:
 *     turns[c] = base^(-2c / rot_dim) / (2 pi), and
 *     FA_ROTARY_LINEAR  turns / factor
 *     FA_ROTARY_NTK     base * factor^(rot_dim / (rot_dim - 2)) as base
 *     FA_ROTARY_YARN    turns of pairs that make more than 32 turns over
 *                       original_len, turns / factor below one turn, a linear
 *                       ramp between them; gain = 0.1 ln(factor) + 1
 * or the caller writes turns and gain (of other schemes) into it. */
#define FA_ROTARY_NONE 0
#define FA_ROTARY_LINEAR 1
#define FA_ROTARY_NTK 2
#define FA_ROTARY_YARN 3
#define FA_ROTARY_MAX_DIM 256
typedef struct fa_rotary_config {
    int dtype;                 /* FA_DTYPE_* */
    int interleaved;
    size_t d_head, rot_dim;    /* rot_dim even, 2 .. d_head; d_head <= 256 */
    float gain;
    double turns[FA_ROTARY_MAX_DIM / 2];
} fa_rotary_config;
int fa_rotary_init(fa_rotary_config* cfg, int dtype, size_t d_head, size_t rot_dim, int interleaved, double base,
                   int scaling, double factor, double original_len);

/* A tensor of `heads` head rows a token and the layouts of its input and
 * output (as in fa_score_config; in place where pointers and strides are the same). */
typedef struct fa_rotary_tensor {
    size_t heads;
    fa_strides in, out;
} fa_rotary_tensor;
/* positions: int32 [batch, seq_len], device memory.  k_layout may be NULL
 * (one tensor). */
int fa_rotary(void* stream, const fa_rotary_config* cfg, size_t batch, size_t seq_len, const int32_t* positions,
              int inverse, const fa_rotary_tensor* q_layout, const void* q, void* q_out,
              const fa_rotary_tensor* k_layout, const void* k, void* k_out);

/* ---- key / value cache and attention of drafted trees -----------------------
 * No counterpart in the reference.  A cache holds capacity rows a sequence,
 * either one after another (block_table NULL: row r of sequence b at
 * b * batch + r * seq + head * head elements) or in pages of a pool: row r
 * lies in page block_table[b][r / page_size] at row r % page_size of it, and
 * the batch stride is the stride between pages (page_size: a power of two;
 * capacity is pages_per_seq * page_size).  Page numbers outside [0, n_pages)
 * hold no rows: their keys are not seen, and writes to them are dropped.
 * lens[b] rows of sequence b are filled (device memory); the drafted tokens'
 * rows come right after them.  lens[b] < 0 marks an idle sequence: its
 * queries get zeros, and nothing is written to it.  Rows at or past the capacity are not seen. */
typedef struct fa_kv_cache {
    int dtype;
    size_t batch, kv_heads, d_head;
    void *k, *v;
    fa_strides k_strides, v_strides;   /* all 0: [batch or pages, kv_heads, rows, d_head] */
    const int32_t* lens;               /* [batch] */
    size_t capacity;                   /* rows a sequence, without pages */
    const int32_t* block_table;        /* [batch, pages_per_seq] or NULL */
    size_t page_size, n_pages, pages_per_seq;
} fa_kv_cache;

/* Writes the n tokens' keys and values (layouts as in fa_score_config,
 * [batch, kv_heads, n, d_head]) to rows lens[b] .. lens[b] + n - 1; lens stays
 * as it is.  With rotary and positions (int32 [batch, n]) the keys are
 * rotated on the way, and so are, in the same launch, the queries q -> q_out
 * where q_layout is given (rotary then has to be too). */
typedef struct fa_append_config {
    size_t n_tokens;
    fa_strides k, v;
    const fa_rotary_config* rotary;    /* NULL: keys are copied, positions not read */
    const fa_rotary_tensor* q_layout;  /* NULL: no queries */
} fa_append_config;
int fa_cache_append(void* stream, const fa_kv_cache* cache, const fa_append_config* cfg, const void* k, const void* v,
                    const int32_t* positions, const void* q, void* q_out);

/* Attention of n drafted tokens a sequence: token i sees the rows before
 * lens[b] and the drafted row lens[b] + t iff bit t % 64 of
 * mask[b][i][t / 64] is set (mask: [batch, n, ceil(n / 64)] 64-bit words, device memory;
 * mask_shared: one for all sequences; NULL: t <= i, so one token is a decode
 * step).  softmax_scale, softcap and slopes as in fa_score_config, where
 * filled rows stand at their row number and drafted ones at positions[b][t]
 * (int32 [batch, n]; NULL: lens[b] + t).  q, out: [batch, heads, n, d_head]
 * by default; lse: f32 [batch, heads, n] or NULL.  n <= 256, d_head <= 256. */
typedef struct fa_tree_config {
    size_t heads, n_tokens;
    float softmax_scale, softcap;
    const float* slopes;
    const int32_t* positions;
    const uint64_t* mask;
    int mask_shared;
    fa_strides q, out;
} fa_tree_config;
int fa_tree_attention(void* stream, const fa_tree_config* cfg, const fa_kv_cache* cache, const void* q, void* out,
                      float* lse);

/* ---- naive attention (materialised scores) -------------------------------
 * naive_attention -- src/naive.rs:14-75: the textbook O(seq_q * seq_k)
 * memory form (scores, row softmax, PV) that the crate keeps as its
 * correctness oracle, here on the GPU.  Same shape checks and order
 * (src/naive.rs:24-27); seq_len_q or d_head == 0 writes nothing, seq_len_k
 * == 0 writes zeros (the crate's out_row.fill).  f32 arithmetic. */
int fa_naive_attention(const float* q, size_t q_len, const float* k, size_t k_len, const float* v,
                       size_t v_len, size_t seq_len_q, size_t seq_len_k, size_t d_head, int causal,
                       float* out, size_t out_len);
/* Device-resident, multi-head form of the above ([batch, heads, seq, d],
 * caller's stream).  precision FA_NAIVE_F64 computes scores, softmax and PV
 * in f64 (output rounded to f32): an on-device reference for checking the
 * flash kernels at sizes a CPU oracle cannot reach.  The score buffer is
 * allocated stream-ordered for as many whole heads at a time as fit in both
 * 8 GiB and half the device memory free at the call (at least one head); a
 * single head's score matrix larger than half the free memory returns
 * FA_ERR_ALLOC with nothing queued.  No counterpart beyond naive_attention
 * itself in the reference. */
#define FA_NAIVE_F32 0
#define FA_NAIVE_F64 1
int fa_naive_device(void* stream, const float* q, const float* k, const float* v, size_t batch,
                    size_t heads, size_t seq_len_q, size_t seq_len_k, size_t d_head, int causal,
                    int precision, float* out);

/* ---- introspection -------------------------------------------------------
 * fa_init loads the code object on the current device (done lazily by every
 * entry point).  fa_describe_launch writes the kernel name(s) and grid the
 * given call would launch, e.g. "fa_prefill_v2_d128_1 grid=512x1x1 block=512",
 * launching nothing and needing no device (it plans for the current
 * device's CU count, or 256 CUs when no device is visible); it returns the
 * argument / support status the launch would return. */
int fa_init(void);
int fa_describe_launch(int variant, size_t batch, size_t heads, size_t seq_len_q, size_t seq_len_k,
                       size_t d_head, int causal, const fa_launch_opts* opts, char* buf,
                       size_t buf_len);

/* ---- peak probes ---------------------------------------------------------
 * No counterpart in the reference: a measurement aid, so the roofline
 * denominators (the MI355X data-sheet peaks) can be checked against the
 * machine.  Queues one probe kernel on `stream` (device memory `buf`, 16-byte
 * aligned, `bytes` long) and stores its work in *work; the caller times it.
 *   FA_PROBE_MFMA_*: every wave of 8 x #CUs four-wave workgroups (two
 *     resident per CU) runs independent chains of `iters` (1 .. 2^20)
 *     back-to-back MFMAs of that kind and writes one checksum float to buf
 *     (bytes >= 128 x #CUs); *work = FLOP.
 *   FA_PROBE_COPY: copies the first bytes/2 of buf (whole 16-byte elements)
 *     onto the second half; *work = bytes read + bytes written;
 *   FA_PROBE_READ: reads the first bytes/2 of buf (whole 16-byte elements),
 *     each workgroup one contiguous chunk, and writes nothing; *work = bytes
 *     read. */
#define FA_PROBE_MFMA_F32_32X32X2 0
#define FA_PROBE_MFMA_F32_16X16X4 1
#define FA_PROBE_MFMA_BF16_16X16X32 2
#define FA_PROBE_COPY 3
#define FA_PROBE_MFMA_BF16_32X32X16 4
#define FA_PROBE_READ 5
int fa_probe_launch(int kind, void* stream, void* buf, size_t bytes, unsigned iters, double* work);

#ifdef __cplusplus
}
#endif
#endif /* FA_HIP_H */
