// fa_cache.hip -- gfx950 kernels for few query rows over many keys: drafted trees
// over a key / value cache (fa_tree_attention) and short query blocks of score
// attention (fa_score_forward).
//
// The rows of a (sequence, kv head) are its tokens times the query heads of the
// group, so K and V are read once for all of them.  A workgroup takes a run of keys and up
// to 16 MT rows; each of its waves walks 32-key blocks of its own through LDS that only it
// uses, with no barrier until the waves' sums are joined at the end.  Runs
// of one sequence leave partial sums that fa_rows_merge joins.

#include "fa_ops_common.h"

template <typename T, int D>
struct RowsGeo {
    static constexpr int NW = sizeof(T) == 4 && D > 128 ? 2 : 4;   // LDS: 2 x 32 rows a wave
    static constexpr int SK = 32;
};

// Where row `key` of sequence b lies (element offset), or -1: no such row.
struct CacheRows {
    const int32_t* table;
    int64_t seq, batch;
    int shift, n_pages, limit;
    __device__ __forceinline__ int64_t at(int key) const {
        if (key >= limit) return -1;
        if (!table) return key * seq;
        const int page = table[key >> shift];
        if ((unsigned)page >= (unsigned)n_pages) return -1;
        return page * batch + (key & ((1 << shift) - 1)) * seq;
    }
};

template <typename T, int D, int MT>
__device__ __forceinline__ void rows_body(const RowsParams& p) {
    using M = Mma<T>;
    using v8 = typename M::v8;
    constexpr int NW = RowsGeo<T, D>::NW, SK = RowsGeo<T, D>::SK;
    constexpr int KB = SK / 16, NDC = D / 32, NDB = D / 16, LD = D + kPad<T>, CPR = D / 8;
    constexpr int TILE = SK * LD;
    constexpr int SLOT = MT * NDB * 64;   // f32x4 of a wave's sums
    constexpr int BYTES = 2 * NW * TILE * (int)sizeof(T);
    static_assert(NW / 2 * SLOT * 16 <= BYTES, "the sums fit the tiles");
    __shared__ __attribute__((aligned(16))) char smem[BYTES];
    __shared__ float Ml[NW / 2][MT][2][16];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, li = lane & 15;
    T* const Ks = reinterpret_cast<T*>(smem) + wave * 2 * TILE;
    T* const Vs = Ks + TILE;

    // split, row block and (sequence, kv head) of the workgroup: the row blocks of one run
    // of keys side by side on one XCD where the counts allow
    const int nkv = p.batch * p.kv_heads, runs = nkv * p.num_splits;
    int run, rb;
    if ((runs & 7) == 0) {
        const int t = blockIdx.x >> 3;
        rb = t % p.nrb;
        run = t / p.nrb * 8 + (blockIdx.x & 7);
    } else {
        rb = blockIdx.x % p.nrb;
        run = blockIdx.x / p.nrb;
    }
    const int kv = run / p.num_splits, split = run % p.num_splits;
    const int b = kv / p.kv_heads, hk = kv % p.kv_heads;
    const bool tree = p.lens != nullptr, docs = p.q_doc != nullptr;

    // keys of the sequence: all of the filled rows, then the drafted ones
    const int len = tree ? p.lens[b] : 0;
    const int prefix = p.prefix ? p.prefix[b] : 0;
    int total;
    if (tree) {
        total = len < 0 ? 0 : (int)min((int64_t)len + p.n, (int64_t)p.sk);
    } else {
        total = p.causal ? max(min(max(p.q_start + p.n, prefix), p.sk), 0) : p.sk;
    }
    // keys that every row sees: those before `open`
    const int open = tree ? min(max(len, 0), p.sk) : docs ? 0 : p.causal ? max(p.q_start + 1, prefix) : p.sk;
    const int per = ((total + p.num_splits - 1) / p.num_splits + SK - 1) / SK * SK;
    const int kbeg = min(split * per, total), kend = min(kbeg + per, total);

    const T* K = reinterpret_cast<const T*>(p.k) + hk * p.ks.h + (p.table ? 0 : b * p.ks.b);
    const T* V = reinterpret_cast<const T*>(p.v) + hk * p.vs.h + (p.table ? 0 : b * p.vs.b);
    const int32_t* table = p.table ? p.table + (int64_t)b * p.pages_per_seq : nullptr;
    const CacheRows krows = {table, p.ks.s, p.ks.b, p.page_shift, p.n_pages, kend};
    const CacheRows vrows = {table, p.vs.s, p.vs.b, p.page_shift, p.n_pages, kend};

    // the wave's rows: token r / group, head r % group
    const int nrows = p.n * p.group, rfirst = rb * 16 * MT;
    v8 qreg[MT][NDC];
    f32x4 o[MT][NDB];
    float m[MT], l[MT], slope[MT];
    int token[MT], pos[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int r = rfirst + 16 * t + li;
        const bool real = r < nrows;
        token[t] = real ? r / p.group : 0;
        const int h = hk * p.group + (real ? r % p.group : 0);
        const T* q = reinterpret_cast<const T*>(p.q) + b * p.qs.b + h * p.qs.h;
#pragma unroll
        for (int dc = 0; dc < NDC; ++dc)
            qreg[t][dc] = global_row<T>(q, p.qs.s, token[t], real ? p.n : 0, 32 * dc + 8 * g, p.d, p.vec);
        pos[t] = !tree ? p.q_start + token[t] : p.pos ? p.pos[b * p.n + token[t]] : len + token[t];
        slope[t] = p.slopes ? p.slopes[h] * kLog2e : 0.0f;
#pragma unroll
        for (int j = 0; j < NDB; ++j) o[t][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        m[t] = OPS_NEG_INF;
        l[t] = 0.0f;
    }

    // whether token `tok` sees a key
    auto sees = [&](int tok, int key) -> bool {
        if (krows.at(key) < 0) return false;
        if (!tree) {
            if (p.causal && !(key <= p.q_start + tok || key < prefix)) return false;
            if (!docs) return true;
            const int id = p.q_doc[(int64_t)b * p.n + tok];
            return id >= 0 && p.k_doc[(int64_t)b * p.sk + key] == id;
        }
        if (key < len) return true;
        const int bit = key - len;
        if (!p.mask) return bit <= tok;
        const int64_t row = (p.mask_shared ? 0 : (int64_t)b * p.n) + tok;
        return (p.mask[row * p.mask_words + (bit >> 6)] >> (bit & 63)) & 1;
    };
    bool special = false;   // V held infinities or NaN in a masked block

    for (int k0 = kbeg + SK * wave; k0 < kend; k0 += SK * NW) {
        bool hidden = k0 + SK > min(open, kend);
#pragma unroll
        for (int i = 0; i < SK * CPR / 64; ++i) {
            const int r = (i * 64 + lane) / CPR, col = 8 * ((i * 64 + lane) % CPR);
            const int64_t ka = krows.at(k0 + r), va = vrows.at(k0 + r);
            hidden = hidden || ka < 0;
            *reinterpret_cast<v8*>(Ks + r * LD + col) = global_row<T>(K + ka, 0, 0, ka >= 0, col, p.d, p.vec);
            *reinterpret_cast<v8*>(Vs + r * LD + col) = global_row<T>(V + va, 0, 0, va >= 0, col, p.d, p.vec);
        }
        const bool masked = __builtin_amdgcn_ballot_w64(hidden) != 0;
        reread();
        v8 pb[MT][1];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            f32x4 s[KB];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                s[kb] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int dc = 0; dc < NDC; ++dc)
                    s[kb] = M::mma(row_op<T, LD>(Ks, 16 * kb, dc, g, li), qreg[t][dc], s[kb]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = k0 + 16 * kb + 4 * g + r;
                    float z = s[kb][r] * p.scale_log2e, th;
                    if (p.cap_log2e != 0.0f) z = capped<T>(s[kb][r], p.cap_in, p.cap_log2e, &th);
                    int kpos = key;
                    bool see = true;
                    if (masked) {
                        see = sees(token[t], key);
                        if (tree && p.pos && key >= len && see) kpos = p.pos[b * p.n + key - len];
                    }
                    z -= slope[t] * fabsf((float)(pos[t] - kpos));
                    s[kb][r] = see ? z : OPS_NEG_INF;
                }
            }
            float mt = OPS_NEG_INF;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int r = 0; r < 4; ++r) mt = fmaxf(mt, s[kb][r]);
            mt = row4_max(mt);
            const float mn = fmaxf(m[t], mt);
            const float ref = mn == OPS_NEG_INF ? 0.0f : mn;
            const float corr = ops_exp2(m[t] - ref);
            m[t] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float x = ops_exp2(s[kb][r] - ref + kProbLog2<T>);
                    pb[t][0][4 * kb + r] = T(x);
                    sum += x;
                }
            l[t] = l[t] * corr + row4_sum(sum);
#pragma unroll
            for (int j = 0; j < NDB; ++j) o[t][j] *= corr;
        }
        if (masked) {
            reread();
            special = tile_clean<T, LD, D, SK, 64>(Vs, lane) || special;
            reread();
        }
        {
#pragma unroll
            for (int j = 0; j < NDB; ++j) {
                const v8 a = col_op<T, LD>(Vs, 0, 16 * j, g, li);
#pragma unroll
                for (int t = 0; t < MT; ++t) o[t][j] = M::mma(a, pb[t][0], o[t][j]);
            }
        }
        reread();
    }

    __shared__ int any_special[NW];
    if (lane == 0) any_special[wave] = 0;
    if (__builtin_amdgcn_ballot_w64(special) != 0 && lane == 0) any_special[wave] = 1;

    // join the waves' sums: the upper half leaves its own, the lower half adds them
    f32x4* const sums = reinterpret_cast<f32x4*>(smem);
#pragma unroll
    for (int half = NW / 2; half >= 1; half /= 2) {
        __syncthreads();
        if (wave >= half && wave < 2 * half) {
            f32x4* to = sums + (wave - half) * SLOT;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
#pragma unroll
                for (int j = 0; j < NDB; ++j) to[(t * NDB + j) * 64 + lane] = o[t][j];
                if (g == 0) {
                    Ml[wave - half][t][0][li] = m[t];
                    Ml[wave - half][t][1][li] = l[t];
                }
            }
        }
        __syncthreads();
        if (wave < half) {
            const f32x4* from = sums + wave * SLOT;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const float m2 = Ml[wave][t][0][li], l2 = Ml[wave][t][1][li];
                const float mn = fmaxf(m[t], m2), ref = mn == OPS_NEG_INF ? 0.0f : mn;
                const float c1 = ops_exp2(m[t] - ref), c2 = ops_exp2(m2 - ref);
                m[t] = mn;
                l[t] = l[t] * c1 + l2 * c2;
#pragma unroll
                for (int j = 0; j < NDB; ++j) o[t][j] = o[t][j] * c1 + from[(t * NDB + j) * 64 + lane] * c2;
            }
        }
    }
    if (wave != 0) return;
    int specials = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) specials |= any_special[i];
    auto row_at = [&](int key) -> const T* {
        const int64_t at = vrows.at(key);
        return at < 0 ? nullptr : V + at;
    };
    auto row_sees = [&](int key, int r) { return sees((rfirst + r) / p.group, key); };
    const int mine = min(16 * MT, nrows - rfirst);

    if (p.num_splits > 1) {
        const int64_t part = ((int64_t)kv * p.nrb + rb) * p.num_splits + split;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            float* po = p.part_o + (part * 16 * MT + 16 * t + li) * D;
#pragma unroll
            for (int j = 0; j < NDB; ++j) *reinterpret_cast<f32x4*>(po + 16 * j + 4 * g) = o[t][j];
            if (g == 0) {
                p.part_ml[part * 32 * MT + 16 * t + li] = m[t];
                p.part_ml[part * 32 * MT + 16 * MT + 16 * t + li] = l[t];
            }
        }
        if (specials) {
            __threadfence();
            add_specials<T, float, true>(kbeg, kend, mine, p.d, lane, row_at, row_sees,
                                         [&](int r) { return p.part_o + (part * 16 * MT + r) * D; });
        }
        return;
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int r = rfirst + 16 * t + li;
        if (r >= nrows) continue;
        const int h = hk * p.group + r % p.group;
        T* out = reinterpret_cast<T*>(p.out) + b * p.os.b + h * p.os.h + token[t] * p.os.s;
        const float inv = l[t] == 0.0f ? 0.0f : 1.0f / l[t];
#pragma unroll
        for (int j = 0; j < NDB; ++j) store4<T>(out, 16 * j + 4 * g, p.d, p.ovec, o[t][j] * inv);
        if (p.lse && g == 0)
            p.lse[((int64_t)b * p.heads + h) * p.n + token[t]] =
                l[t] == 0.0f ? OPS_NEG_INF : (m[t] + __builtin_log2f(l[t]) - kProbLog2<T>) * kLn2;
    }
    if (specials) {
        __threadfence();
        add_specials<T, T, true>(kbeg, kend, mine, p.d, lane, row_at, row_sees, [&](int r) {
            const int h = hk * p.group + (rfirst + r) % p.group;
            return reinterpret_cast<T*>(p.out) + b * p.os.b + h * p.os.h + (rfirst + r) / p.group * p.os.s;
        });
    }
}

// Joins the partial sums of a row, a wave a row, four columns a lane.
template <typename T, int D, int ROWS>
__device__ __forceinline__ void rows_merge(const RowsParams& p) {
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int nrows = p.n * p.group;
    if (row >= (int64_t)p.batch * p.kv_heads * nrows) return;
    const int kv = row / nrows, r = row % nrows;
    const int b = kv / p.kv_heads, h = kv % p.kv_heads * p.group + r % p.group, token = r / p.group;
    const int64_t part = ((int64_t)kv * p.nrb + r / ROWS) * p.num_splits;
    const float* ml = p.part_ml + part * 2 * ROWS + r % ROWS;
    const float* po = p.part_o + (part * ROWS + r % ROWS) * D + 4 * lane;
    float mx = OPS_NEG_INF;
    for (int s = lane; s < p.num_splits; s += 64) mx = fmaxf(mx, ml[(int64_t)s * 2 * ROWS]);
#pragma unroll
    for (int s = 1; s < 64; s *= 2) mx = fmaxf(mx, __shfl_xor(mx, s));
    const float ref = mx == OPS_NEG_INF ? 0.0f : mx;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
    for (int s = 0; s < p.num_splits; ++s) {
        const float c = ops_exp2(ml[(int64_t)s * 2 * ROWS] - ref);
        l += c * ml[(int64_t)s * 2 * ROWS + ROWS];
        if (4 * lane < D) o += c * *reinterpret_cast<const f32x4*>(po + (int64_t)s * ROWS * D);
    }
    if (4 * lane < D)
        store4<T>(reinterpret_cast<T*>(p.out) + b * p.os.b + h * p.os.h + token * p.os.s, 4 * lane, p.d, p.ovec,
                  o * (l == 0.0f ? 0.0f : 1.0f / l));
    if (p.lse && lane == 0)
        p.lse[((int64_t)b * p.heads + h) * p.n + token] =
            l == 0.0f ? OPS_NEG_INF : (mx + __builtin_log2f(l) - kProbLog2<T>) * kLn2;
}

#define ROWS_KERNELS(N, T, D, MT)                                                                               \
    extern "C" __global__ __launch_bounds__((64 * RowsGeo<T, D>::NW)) void fa_rows_##N##_d##D##_t##MT(RowsParams p) { \
        rows_body<T, D, MT>(p);                                                                                 \
    }                                                                                                           \
    extern "C" __global__ __launch_bounds__(256) void fa_rows_merge_##N##_d##D##_t##MT(RowsParams p) {          \
        rows_merge<T, D, 16 * MT>(p);                                                                           \
    }
ROWS_KERNELS(bf16, __bf16, 64, 1)
ROWS_KERNELS(bf16, __bf16, 64, 2)
ROWS_KERNELS(bf16, __bf16, 64, 4)
ROWS_KERNELS(bf16, __bf16, 128, 1)
ROWS_KERNELS(bf16, __bf16, 128, 2)
ROWS_KERNELS(bf16, __bf16, 128, 4)
ROWS_KERNELS(bf16, __bf16, 256, 1)
ROWS_KERNELS(bf16, __bf16, 256, 2)
ROWS_KERNELS(f16, _Float16, 64, 1)
ROWS_KERNELS(f16, _Float16, 64, 2)
ROWS_KERNELS(f16, _Float16, 64, 4)
ROWS_KERNELS(f16, _Float16, 128, 1)
ROWS_KERNELS(f16, _Float16, 128, 2)
ROWS_KERNELS(f16, _Float16, 128, 4)
ROWS_KERNELS(f16, _Float16, 256, 1)
ROWS_KERNELS(f16, _Float16, 256, 2)
ROWS_KERNELS(f32, float, 64, 1)
ROWS_KERNELS(f32, float, 64, 2)
ROWS_KERNELS(f32, float, 128, 1)
ROWS_KERNELS(f32, float, 128, 2)
ROWS_KERNELS(f32, float, 256, 1)
