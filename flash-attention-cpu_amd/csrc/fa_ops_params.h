// fa_ops_params.h -- parameter blocks and geometry shared by the host code
// (fa_ops_host.h) and the kernels of fa_score.hip, fa_cache.hip, fa_cache4.hip,
// fa_rotary.hip and fa_norm.hip.
#ifndef FA_OPS_PARAMS_H
#define FA_OPS_PARAMS_H

#include <stdint.h>

// Every code object of the operators holds an (empty) kernel of this name: fa_ops_params_ and the build's stamp of this
// file.  The host loads none that lacks it, since kernels of other parameter blocks would read pointers from wrong places.
#ifndef OPS_STAMP
#define OPS_STAMP none
#endif
#define OPS_PASTE2_(a, b) a##b
#define OPS_PASTE2(a, b) OPS_PASTE2_(a, b)
#define OPS_STAMP_KERNEL OPS_PASTE2(fa_ops_params_, OPS_STAMP)

// Element strides between batches, tokens and heads.
struct OpsStrides {
    int64_t b, s, h;
};

// Tokens per entry of the document range tables.
constexpr int kDocTile = 64;
// The largest cap whose scores 16-bit kernels take with the short formula (within 1e-4, a quarter of f16's rounding of
// the weights).
constexpr float kFastCap = 512.0f;
// What fa_score_doc_order takes: blocks to order, and tiles of the other side, of all batches.
constexpr int kOrderBlocks = 1024, kOrderTiles = 4096;

struct ScoreParams {
    const void *q, *k, *v, *out_in, *dout;
    void *out, *dq, *dk, *dv;
    float* lse;               // forward: written where not NULL
    const float* lse_in;      // backward
    float *lse2, *delta;      // [batch, heads, sq]: lse * log2(e) (+inf: empty row) and dO . O
    const float* slopes;
    const int32_t *q_doc, *k_doc, *prefix;
    int32_t *q_rng, *k_rng;   // (min, max) id of each kDocTile tokens
    int32_t *q_order, *k_order;   // batch * blocks + block, in the order of their workgroups; NULL: none
    int q_rows, k_rows;       // rows of a block (for fa_score_doc_order)
    OpsStrides qs, ks, vs, os, dos, dqs, dks, dvs;
    int batch, heads, kv_heads, group, sq, sk, d;
    int causal, q_start;
    int window, sinks;        // window 0: none
    int nqb;                  // query (dK/dV: key) blocks a slice
    int splits;               // dK/dV: workgroups that share a key block, each some heads of the group
    float* part;              // their sums: [dK, dV][split][batch, kv head][key][padded d]
    // dK/dV in a window: workgroups from far_first on take far_stages stages each of the queries that see the first
    // far_blocks key blocks (far_rows rows) as sinks alone
    // (shared out over far_chunks chunks of stages and far_splits parts of the group's heads)
    int far_first, far_stages, far_chunks, far_splits, far_blocks, far_rows;
    float* far_part;          // [dK, dV][1 + chunk, split][batch, kv head][far_rows][padded d]
    float scale;              // of the scores
    float scale_log2e;
    float cap_in;             // 2 log2(e) scale / softcap: exponent of the cap's tanh
    float cap_log2e;          // softcap * log2(e); 0: no cap
};

// Largest position of a token over a cache where a window looks at it, and largest window that hides anything.
constexpr int kWindowMaxPos = 1 << 30;

// Waves of a workgroup of the streaming rows kernel, by the bytes of a padded row (up to 512): each has
// two slots of 32 rows of K and V in LDS.
template <int ROW>
constexpr int kStreamWaves = ROW <= 256 ? 4 : 2;

// Attention of few rows over a long key range, keys split over workgroups.
struct RowsParams {
    const void *q, *k, *v;
    void* out;
    float* lse;               // [batch, heads, n] or NULL
    float *part_o, *part_ml;  // [run][kv head][row block][block_rows][D], [..][2][block_rows]
    const float* slopes;
    const int32_t *q_doc, *k_doc, *prefix;   // score attention
    const int32_t *lens, *table, *pos;       // tree attention (lens != NULL)
    const uint64_t* mask;
    OpsStrides qs, ks, vs, os;
    int batch, heads, kv_heads, group, n, sk, d;   // n: tokens; sk: keys (tree: capacity)
    int causal, q_start;
    int window, sinks;        // window 0: none
    int page_shift, n_pages, pages_per_seq;
    int mask_words, mask_shared;
    int nrb, block_rows;      // row blocks of a (batch, kv head), and rows of one
    int num_runs, share;      // runs of keys a kv head, all sequences together; what the keys are shared out over
    int step;                 // keys that a run's length is a multiple of
    float scale_log2e, cap_in, cap_log2e;   // as in ScoreParams
    const void *k_scale, *v_scale;          // a cache in 4 bits: its steps and offsets,
    int block4;               // the rows of a page (without pages: of a sequence),
    int vec4;                 // and whether rows of q and out are aligned
};

// Waves of a workgroup of the kernel over a cache in 4 bits.
constexpr int kRows4Waves = 4;
// Largest size of a value in such a cache: larger ones count as that, and what codes stand for stays in f16's range.
constexpr float kCache4Max = 60000.0f;
// Rows that a thread reads back.
constexpr int kCache4ReadRows = 4;
// Append to and rows out of such a cache.
struct Cache4Params {
    const void *k, *v;        // append
    void *ko, *vo;            // read; NULL: not wanted
    OpsStrides ks, vs;
    uint32_t *k4, *v4;        // [blocks, kv_heads, rows, d / 8], [blocks, kv_heads, rows / 8, d]
    uint16_t *kscale, *vscale;   // [blocks, kv_heads, rows, d / 32, (S, O)], [blocks, kv_heads, rows / 8, d / 32, (S, O), 8]
    const int32_t *lens, *table, *rows;
    int batch, kv_heads, n, d;
    int capacity, block_rows, page_shift, n_pages, pages_per_seq;
    int nparts;               // workgroups of a head's rows
    int loops;                // append: how often a workgroup takes 256 / d runs of 8 rows
    int vec;                  // rows of k, v (ko, vo) are aligned
};

// One tensor of a rotary or append launch.
struct RotTensor {
    const void* src;
    void* dst;
    OpsStrides in, out;
    int heads;
    int rotate;               // 0: copied
    int cache;                // dst is a cache: rows lens[b] + token
};

struct RotParams {
    RotTensor t[3];
    int nt;
    int batch, seq, d, rot, interleaved;
    int cols;                 // units of a token and head (columns or column pairs, or chunks of them)
    int hthreads;             // threads that share a token's heads
    const int32_t *pos, *lens, *table;
    int capacity, page_shift, n_pages, pages_per_seq;
    float gain, sign;
    double turns[128];
};

// One tensor of a launch of norms with rotary positions.
constexpr int kNormThreads = 256;
constexpr int kNormTokens = 16;   // most tokens of a workgroup
constexpr int kNormColumns = 8;   // of a workgroup of fa_norm_weights
struct NormTensor {
    const void *x, *dy, *w;   // w: NULL: ones
    void* out;                // y, or dx (NULL: not wanted)
    float *dw, *part;         // backward: the weights' gradient, and its partial sums [blocks][d]
    OpsStrides xs, dys, outs;
    int heads;
    int norm;                 // 0: copied
    int cache;                // out is a cache: rows lens[b] + token
    int tokens, blocks;       // of a workgroup; workgroups
};

struct NormParams {
    NormTensor t[3];
    int nt;
    int batch, seq, d, rot, interleaved;
    int units, lanes;         // units of columns of a row, and the lanes that keep them
    const int32_t *pos, *lens, *table;
    int capacity, page_shift, n_pages, pages_per_seq;
    float gain, eps;
    double turns[128];
};

#endif  // FA_OPS_PARAMS_H
