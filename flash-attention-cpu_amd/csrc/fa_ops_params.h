// fa_ops_params.h -- parameter blocks and geometry shared by the host code
// (fa_ops_host.h) and the kernels of fa_score.hip, fa_cache.hip and
// fa_rotary.hip.
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
    int nqb;                  // query (dK/dV: key) blocks a slice
    int splits;               // dK/dV: workgroups that share a key block, each some heads of the group
    float* part;              // their sums: [dK, dV][split][batch, kv head][key][padded d]
    float scale;              // of the scores
    float scale_log2e;
    float cap_in;             // 2 log2(e) scale / softcap: exponent of the cap's tanh
    float cap_log2e;          // softcap * log2(e); 0: no cap
};

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
    int page_shift, n_pages, pages_per_seq;
    int mask_words, mask_shared;
    int nrb, block_rows;      // row blocks of a (batch, kv head), and rows of one
    int num_runs, share;      // runs of keys a kv head, all sequences together; what the keys are shared out over
    int step;                 // keys that a run's length is a multiple of
    float scale_log2e, cap_in, cap_log2e;   // as in ScoreParams
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

#endif  // FA_OPS_PARAMS_H
