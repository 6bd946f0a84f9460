// fa_score.hip -- gfx950 kernels of attention with modified scores
// (fa_score_forward, fa_score_backward).
//
// Scores are computed transposed, so that a lane owns one row of the tile it keeps:
// forward and dQ kernels keep query rows (S^T = K Q^T, lane: query li, keys 4g + r
// of each 16-key block) and walk the keys, the dK/dV kernel keeps key rows (S = Q K^T,
// lane: key li) and walks the queries.  The weights a lane computes are then already
// the B operand of the second product, whose A operand is the walked tile read
// transposed.
//
// Which walked tiles hold a visible pair is decided for 64 tiles at a time: each
// lane tests one (causal and prefix bounds, document ranges), and two ballots give the
// tiles to visit and those of them that need the mask element by element.

#include "fa_ops_common.h"

// Tile shapes: MT 16-row tiles a wave, NW waves a workgroup, SK walked rows a stage.
template <typename T, int D>
struct Geo {
    static constexpr bool wide = sizeof(T) == 4 || D > 128;
    static constexpr int MT = wide ? 1 : 2;
    static constexpr int NW = wide ? 8 : 4;
    static constexpr int SK = sizeof(T) == 4 || D > 128 ? 32 : 64;
};

template <typename T>
__device__ __forceinline__ const T* slice(const void* base, OpsStrides st, int b, int h) {
    return reinterpret_cast<const T*>(base) + b * st.b + h * st.h;
}
template <typename T>
__device__ __forceinline__ T* slice(void* base, OpsStrides st, int b, int h) {
    return reinterpret_cast<T*>(base) + b * st.b + h * st.h;
}

// (slice, block) of a workgroup: the slices of a kv head share its K and V, so all
// its workgroups go to one XCD where the counts allow (workgroups go round-robin over the eight); blocks in
// falling order, the longest first where causal.
struct Work {
    int b, hk, hq, blk;   // hq: head within the group
};
__device__ __forceinline__ Work find_work(unsigned id, int nblk, int nkv, int group, int kv_heads) {
    Work w;
    int kv;
    if ((nkv & 7) == 0) {
        const int per = (nkv >> 3) * group;   // slices an XCD
        const int x = id & 7, t = id >> 3;
        w.blk = nblk - 1 - t / per;
        const int s = t % per;
        kv = (s / group) * 8 + x;
        w.hq = s % group;
    } else {
        const int per = nkv * group;
        w.blk = nblk - 1 - id / per;
        const int s = id % per;
        kv = s / group;
        w.hq = s % group;
    }
    w.b = kv / kv_heads;
    w.hk = kv % kv_heads;
    return w;
}

// The stages a workgroup visits, in order.  test(stage, &part) says whether a stage
// holds a visible pair and whether it holds a hidden one.
template <typename Test>
struct Stages {
    uint64_t vis = 0, part = 0;
    int base, count, lane;
    Test test;
    __device__ __forceinline__ Stages(int n, int lane_, Test t) : base(-64), count(n), lane(lane_), test(t) {}
    // next stage (-1: none); *masked: it needs the mask
    __device__ __forceinline__ int next(bool* masked) {
        while (vis == 0) {
            base += 64;
            if (base >= count) return -1;
            bool p = false, v = false;
            if (base + lane < count) v = test(base + lane, &p);
            vis = __builtin_amdgcn_ballot_w64(v);
            part = __builtin_amdgcn_ballot_w64(v && p);
        }
        const int bit = __builtin_ctzll(vis);
        vis &= vis - 1;
        *masked = (part >> bit) & 1;
        return base + bit;
    }
};

// (min, max) document of rows [r0, r1) from the range table (the tiles they touch).
__device__ __forceinline__ void doc_range(const int32_t* rng, int r0, int r1, int* lo, int* hi) {
    *lo = 0x7fffffff;
    *hi = -0x7fffffff - 1;
    for (int t = r0 / kDocTile; t <= (r1 - 1) / kDocTile; ++t) {
        *lo = min(*lo, rng[2 * t]);
        *hi = max(*hi, rng[2 * t + 1]);
    }
}

// Pairs of two row ranges whose documents lie in [alo, ahi] and [blo, bhi].
__device__ __forceinline__ bool docs_meet(int alo, int ahi, int blo, int bhi, bool* part) {
    if (!(alo == ahi && blo == bhi && alo == blo && alo >= 0)) *part = true;
    return alo <= bhi && blo <= ahi && ahi >= 0 && bhi >= 0;
}

// ROWS rows of a matrix into LDS, zero outside [0, rows) x [0, d).
template <typename T, int D, int ROWS, int NT>
__device__ __forceinline__ void fill_tile(T* dst, const T* src, int64_t stride, int row0, int rows, int d, bool vec,
                                          int tid) {
    constexpr int CPR = D / 8, LD = D + kPad<T>;
    const T* p = src + row0 * stride;
#pragma unroll
    for (int i = 0; i < (ROWS * CPR + NT - 1) / NT; ++i) {
        const int pos = tid + i * NT;
        if (ROWS * CPR % NT == 0 || pos < ROWS * CPR) {
            const int r = pos / CPR, col = 8 * (pos % CPR);
            *reinterpret_cast<typename Mma<T>::v8*>(dst + r * LD + col) =
                global_row<T>(p, stride, r, rows - row0, col, d, vec);
        }
    }
}

// Scores in log2 units of the C registers of one 16-row block: cap and bias.
// dist: position of the lane's row minus that of register 0 of the block.
// t: the cap's tanh (backward).
template <typename T>
__device__ __forceinline__ f32x4 modify(const ScoreParams& p, f32x4 s, float slope, float dist, f32x4* t) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        float z;
        if (p.cap_log2e != 0.0f) {
            float th;
            z = capped<T>(s[r], p.cap_in, p.cap_log2e, &th);
            (*t)[r] = th;
        } else {
            z = s[r] * p.scale_log2e;
        }
        s[r] = z - slope * fabsf(dist - (float)r);
    }
    return s;
}

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------
template <typename T, int D>
__device__ __forceinline__ void score_forward(const ScoreParams& p) {
    using M = Mma<T>;
    using v8 = typename M::v8;
    using G = Geo<T, D>;
    constexpr int MT = G::MT, NW = G::NW, SK = G::SK, NT = 64 * NW, BQ = 16 * MT * NW;
    constexpr int KB = SK / 16, NCH = SK / 32, NDC = D / 32, NDB = D / 16, LD = D + kPad<T>;
    __shared__ __attribute__((aligned(16))) T Ks[SK * LD];
    __shared__ __attribute__((aligned(16))) T Vs[SK * LD];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, li = lane & 15;
    const Work w = find_work(blockIdx.x, p.nqb, p.batch * p.kv_heads, p.group, p.kv_heads);
    const int h = w.hk * p.group + w.hq;
    const int q0 = w.blk * BQ, row0 = q0 + 16 * MT * wave;
    const T* Q = slice<T>(p.q, p.qs, w.b, h);
    const T* K = slice<T>(p.k, p.ks, w.b, w.hk);
    const T* V = slice<T>(p.v, p.vs, w.b, w.hk);
    const bool docs = p.q_doc != nullptr;
    const int32_t* kdoc = docs ? p.k_doc + (int64_t)w.b * p.sk : nullptr;
    const ScoreMask mask = {p.causal, p.prefix ? p.prefix[w.b] : 0, p.sk};
    const float slope = p.slopes ? p.slopes[h] * kLog2e : 0.0f;

    v8 qreg[MT][NDC];
    int qd[MT];
    f32x4 o[MT][NDB];
    float m[MT], l[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = row0 + 16 * t + li;
#pragma unroll
        for (int dc = 0; dc < NDC; ++dc) qreg[t][dc] = global_row<T>(Q, p.qs.s, row, p.sq, 32 * dc + 8 * g, p.d, p.vec);
        qd[t] = docs && row < p.sq ? p.q_doc[(int64_t)w.b * p.sq + row] : -1;
#pragma unroll
        for (int j = 0; j < NDB; ++j) o[t][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        m[t] = OPS_NEG_INF;
        l[t] = 0.0f;
    }

    const int q1 = min(q0 + BQ, p.sq);
    int qlo = 0, qhi = 0;
    const int32_t* krng = nullptr;
    if (docs) {
        doc_range(p.q_rng + (int64_t)w.b * 2 * ((p.sq + kDocTile - 1) / kDocTile), q0, q1, &qlo, &qhi);
        krng = p.k_rng + (int64_t)w.b * 2 * ((p.sk + kDocTile - 1) / kDocTile);
    }
    auto test = [&](int st, bool* part) -> bool {
        const int k0 = st * SK, k1 = k0 + SK;
        bool v = true;
        if (k1 > p.sk) *part = true;
        if (p.causal) {
            v = k0 <= p.q_start + q1 - 1 || k0 < mask.prefix;
            if (!(k1 - 1 <= p.q_start + q0 || k1 <= mask.prefix)) *part = true;
        }
        if (docs && v) v = docs_meet(qlo, qhi, krng[k0 / kDocTile * 2], krng[k0 / kDocTile * 2 + 1], part);
        return v;
    };
    Stages<decltype(test)> stages((p.sk + SK - 1) / SK, lane, test);

    bool masked;
    for (int st = stages.next(&masked); st >= 0; st = stages.next(&masked)) {
        const int k0 = st * SK;
        __syncthreads();
        fill_tile<T, D, SK, NT>(Ks, K, p.ks.s, k0, p.sk, p.d, p.vec, tid);
        fill_tile<T, D, SK, NT>(Vs, V, p.vs.s, k0, p.sk, p.d, p.vec, tid);
        __syncthreads();
        v8 pb[MT][NCH];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            f32x4 s[KB];
            const int pos = p.q_start + row0 + 16 * t + li;
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                s[b] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int dc = 0; dc < NDC; ++dc) s[b] = M::mma(row_op<T, LD>(Ks, 16 * b, dc, g, li), qreg[t][dc], s[b]);
                f32x4 th;
                s[b] = modify<T>(p, s[b], slope, (float)(pos - (k0 + 16 * b + 4 * g)), &th);
            }
            if (masked) {
#pragma unroll
                for (int b = 0; b < KB; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int key = k0 + 16 * b + 4 * g + r;
                        bool see = mask.seen(key, pos);
                        if (docs) see = see && qd[t] >= 0 && kdoc[min(key, p.sk - 1)] == qd[t];
                        if (!see) s[b][r] = OPS_NEG_INF;
                    }
            }
            float mt = s[0][0];
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) mt = fmaxf(mt, s[b][r]);
            mt = row4_max(mt);
            const float mn = fmaxf(m[t], mt);
            const float ref = mn == OPS_NEG_INF ? 0.0f : mn;
            const float corr = ops_exp2(m[t] - ref);
            m[t] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float x = ops_exp2(s[b][r] - ref + kProbLog2<T>);
                    pb[t][b / 2][4 * (b & 1) + r] = T(x);
                    sum += x;
                }
            l[t] = l[t] * corr + row4_sum(sum);
#pragma unroll
            for (int j = 0; j < NDB; ++j) o[t][j] *= corr;
        }
        if (masked) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
                mma_seen<T>(o[t], pb[t], [&](int i, int j) { return col_op<T, LD>(Vs, 32 * i, 16 * j, g, li); });
        } else {
#pragma unroll
            for (int i = 0; i < NCH; ++i)
#pragma unroll
                for (int j = 0; j < NDB; ++j) {
                    const v8 a = col_op<T, LD>(Vs, 32 * i, 16 * j, g, li);
#pragma unroll
                    for (int t = 0; t < MT; ++t) o[t][j] = M::mma(a, pb[t][i], o[t][j]);
                }
        }
    }

    T* O = slice<T>(p.out, p.os, w.b, h);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = row0 + 16 * t + li;
        if (row >= p.sq) continue;
        const float inv = l[t] == 0.0f ? 0.0f : 1.0f / l[t];
#pragma unroll
        for (int j = 0; j < NDB; ++j) store4<T>(O + row * p.os.s, 16 * j + 4 * g, p.d, p.ovec, o[t][j] * inv);
        if (p.lse && g == 0) {
            const float lse = (m[t] + __builtin_log2f(l[t]) - kProbLog2<T>) * kLn2;
            p.lse[((int64_t)w.b * p.heads + h) * p.sq + row] = l[t] == 0.0f ? OPS_NEG_INF : lse;
        }
    }
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------

// delta = dO . O and lse2 = lse log2(e) of every row, a group of 16 lanes a row.  Empty rows get lse2 = +inf: their
// weights e^(z - lse) then come out as 0.
template <typename T>
__device__ __forceinline__ void score_delta(const ScoreParams& p) {
    const int64_t row = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 4;
    const int li = threadIdx.x & 15;
    const int64_t total = (int64_t)p.batch * p.heads * p.sq;
    if (row >= total) return;
    const int i = row % p.sq, h = row / p.sq % p.heads, b = row / p.sq / p.heads;
    const T* o = slice<T>(p.out_in, p.os, b, h);
    const T* g = slice<T>(p.dout, p.dos, b, h);
    float sum = 0.0f;
    for (int col = 8 * li; col < p.d; col += 128) {
        const auto x = global_row<T>(o, p.os.s, i, p.sq, col, p.d, p.vec);
        const auto y = global_row<T>(g, p.dos.s, i, p.sq, col, p.d, p.vec);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += float(x[e]) * float(y[e]);
    }
#pragma unroll
    for (int s = 1; s < 16; s *= 2) sum += __shfl_xor(sum, s);
    if (li == 0) {
        const float lse = p.lse_in[row];
        p.delta[row] = sum;
        p.lse2[row] = lse == OPS_NEG_INF ? -OPS_NEG_INF : lse * kLog2e;
    }
}

// dQ: query rows kept, keys walked.
template <typename T, int D>
__device__ __forceinline__ void score_dq(const ScoreParams& p) {
    using M = Mma<T>;
    using v8 = typename M::v8;
    using G = Geo<T, D>;
    constexpr int MT = G::MT, NW = G::NW, SK = G::SK, NT = 64 * NW, BQ = 16 * MT * NW;
    constexpr int KB = SK / 16, NCH = SK / 32, NDC = D / 32, NDB = D / 16, LD = D + kPad<T>;
    __shared__ __attribute__((aligned(16))) T Ks[SK * LD];
    __shared__ __attribute__((aligned(16))) T Vs[SK * LD];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, li = lane & 15;
    const Work w = find_work(blockIdx.x, p.nqb, p.batch * p.kv_heads, p.group, p.kv_heads);
    const int h = w.hk * p.group + w.hq;
    const int q0 = w.blk * BQ, row0 = q0 + 16 * MT * wave;
    const T* Q = slice<T>(p.q, p.qs, w.b, h);
    const T* dO = slice<T>(p.dout, p.dos, w.b, h);
    const T* K = slice<T>(p.k, p.ks, w.b, w.hk);
    const T* V = slice<T>(p.v, p.vs, w.b, w.hk);
    const bool docs = p.q_doc != nullptr;
    const int32_t* kdoc = docs ? p.k_doc + (int64_t)w.b * p.sk : nullptr;
    const ScoreMask mask = {p.causal, p.prefix ? p.prefix[w.b] : 0, p.sk};
    const float slope = p.slopes ? p.slopes[h] * kLog2e : 0.0f;
    const bool cap = p.cap_log2e != 0.0f;

    v8 qreg[MT][NDC], doreg[MT][NDC];
    int qd[MT];
    f32x4 dq[MT][NDB];
    float lse2[MT], delta[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = row0 + 16 * t + li;
        const int64_t at = ((int64_t)w.b * p.heads + h) * p.sq + row;
#pragma unroll
        for (int dc = 0; dc < NDC; ++dc) {
            qreg[t][dc] = global_row<T>(Q, p.qs.s, row, p.sq, 32 * dc + 8 * g, p.d, p.vec);
            doreg[t][dc] = global_row<T>(dO, p.dos.s, row, p.sq, 32 * dc + 8 * g, p.d, p.vec);
        }
        qd[t] = docs && row < p.sq ? p.q_doc[(int64_t)w.b * p.sq + row] : -1;
        lse2[t] = row < p.sq ? p.lse2[at] : -OPS_NEG_INF;
        delta[t] = row < p.sq ? p.delta[at] : 0.0f;
#pragma unroll
        for (int j = 0; j < NDB; ++j) dq[t][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int q1 = min(q0 + BQ, p.sq);
    int qlo = 0, qhi = 0;
    const int32_t* krng = nullptr;
    if (docs) {
        doc_range(p.q_rng + (int64_t)w.b * 2 * ((p.sq + kDocTile - 1) / kDocTile), q0, q1, &qlo, &qhi);
        krng = p.k_rng + (int64_t)w.b * 2 * ((p.sk + kDocTile - 1) / kDocTile);
    }
    auto test = [&](int st, bool* part) -> bool {
        const int k0 = st * SK, k1 = k0 + SK;
        bool v = true;
        if (k1 > p.sk) *part = true;
        if (p.causal) {
            v = k0 <= p.q_start + q1 - 1 || k0 < mask.prefix;
            if (!(k1 - 1 <= p.q_start + q0 || k1 <= mask.prefix)) *part = true;
        }
        if (docs && v) v = docs_meet(qlo, qhi, krng[k0 / kDocTile * 2], krng[k0 / kDocTile * 2 + 1], part);
        return v;
    };
    Stages<decltype(test)> stages((p.sk + SK - 1) / SK, lane, test);

    bool masked;
    for (int st = stages.next(&masked); st >= 0; st = stages.next(&masked)) {
        const int k0 = st * SK;
        __syncthreads();
        fill_tile<T, D, SK, NT>(Ks, K, p.ks.s, k0, p.sk, p.d, p.vec, tid);
        fill_tile<T, D, SK, NT>(Vs, V, p.vs.s, k0, p.sk, p.d, p.vec, tid);
        __syncthreads();
        v8 db[MT][NCH];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int pos = p.q_start + row0 + 16 * t + li;
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f}, dp = {0.0f, 0.0f, 0.0f, 0.0f}, th;
#pragma unroll
                for (int dc = 0; dc < NDC; ++dc) {
                    s = M::mma(row_op<T, LD>(Ks, 16 * b, dc, g, li), qreg[t][dc], s);
                    dp = M::mma(row_op<T, LD>(Vs, 16 * b, dc, g, li), doreg[t][dc], dp);
                }
                s = modify<T>(p, s, slope, (float)(pos - (k0 + 16 * b + 4 * g)), &th);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float ds = ops_exp2(s[r] - lse2[t]) * (dp[r] - delta[t]);
                    if (cap) ds *= 1.0f - th[r] * th[r];
                    if (masked) {
                        const int key = k0 + 16 * b + 4 * g + r;
                        bool see = mask.seen(key, pos) && lse2[t] != -OPS_NEG_INF;
                        if (docs) see = see && qd[t] >= 0 && kdoc[min(key, p.sk - 1)] == qd[t];
                        if (!see) ds = 0.0f;
                    }
                    db[t][b / 2][4 * (b & 1) + r] = T(ds);
                }
            }
        }
        if (masked) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
                mma_seen<T>(dq[t], db[t], [&](int i, int j) { return col_op<T, LD>(Ks, 32 * i, 16 * j, g, li); });
        } else {
#pragma unroll
            for (int i = 0; i < NCH; ++i)
#pragma unroll
                for (int j = 0; j < NDB; ++j) {
                    const v8 a = col_op<T, LD>(Ks, 32 * i, 16 * j, g, li);
#pragma unroll
                    for (int t = 0; t < MT; ++t) dq[t][j] = M::mma(a, db[t][i], dq[t][j]);
                }
        }
    }
    T* out = slice<T>(p.dq, p.dqs, w.b, h);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = row0 + 16 * t + li;
        if (row >= p.sq) continue;
#pragma unroll
        for (int j = 0; j < NDB; ++j) store4<T>(out + row * p.dqs.s, 16 * j + 4 * g, p.d, p.ovec, dq[t][j] * p.scale);
    }
}

// dK and dV: key rows kept, the queries of every head of the group walked.
template <typename T, int D>
__device__ __forceinline__ void score_dkv(const ScoreParams& p) {
    using M = Mma<T>;
    using v8 = typename M::v8;
    constexpr int MT = 1, NW = 8, SQ = 32, NT = 64 * NW, BK = 16 * MT * NW;
    constexpr int QB = SQ / 16, NCH = SQ / 32, NDC = D / 32, NDB = D / 16, LD = D + kPad<T>;
    __shared__ __attribute__((aligned(16))) T Qs[SQ * LD];
    __shared__ __attribute__((aligned(16))) T Os[SQ * LD];
    __shared__ float Ls[2][SQ];
    __shared__ int Ds[SQ];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, li = lane & 15;
    // a workgroup owns whole (batch, kv head) columns: no group in the map
    const Work w = find_work(blockIdx.x, p.nqb, p.batch * p.kv_heads, 1, p.kv_heads);
    const int kbeg = w.blk * BK, key = kbeg + 16 * wave + li;
    const T* K = slice<T>(p.k, p.ks, w.b, w.hk);
    const T* V = slice<T>(p.v, p.vs, w.b, w.hk);
    const bool docs = p.q_doc != nullptr;
    const ScoreMask mask = {p.causal, p.prefix ? p.prefix[w.b] : 0, p.sk};
    const bool cap = p.cap_log2e != 0.0f;

    v8 kreg[NDC], vreg[NDC];
    f32x4 dk[NDB], dv[NDB];
#pragma unroll
    for (int dc = 0; dc < NDC; ++dc) {
        kreg[dc] = global_row<T>(K, p.ks.s, key, p.sk, 32 * dc + 8 * g, p.d, p.vec);
        vreg[dc] = global_row<T>(V, p.vs.s, key, p.sk, 32 * dc + 8 * g, p.d, p.vec);
    }
    const int kd = docs && key < p.sk ? p.k_doc[(int64_t)w.b * p.sk + key] : -1;
#pragma unroll
    for (int j = 0; j < NDB; ++j) dk[j] = dv[j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

    const int kend = min(kbeg + BK, p.sk);
    int klo = 0, khi = 0;
    const int32_t* qrng = nullptr;
    if (docs) {
        doc_range(p.k_rng + (int64_t)w.b * 2 * ((p.sk + kDocTile - 1) / kDocTile), kbeg, kend, &klo, &khi);
        qrng = p.q_rng + (int64_t)w.b * 2 * ((p.sq + kDocTile - 1) / kDocTile);
    }
    auto test = [&](int st, bool* part) -> bool {
        const int q0 = st * SQ, q1 = min(q0 + SQ, p.sq);
        bool v = true;
        if (p.causal) {
            v = p.q_start + q1 - 1 >= kbeg || kbeg < mask.prefix;
            if (!(p.q_start + q0 >= kend - 1 || kend <= mask.prefix)) *part = true;
        }
        if (docs && v) v = docs_meet(klo, khi, qrng[q0 / kDocTile * 2], qrng[q0 / kDocTile * 2 + 1], part);
        return v;
    };

    for (int hq = 0; hq < p.group; ++hq) {
        const int h = w.hk * p.group + hq;
        const T* Q = slice<T>(p.q, p.qs, w.b, h);
        const T* dO = slice<T>(p.dout, p.dos, w.b, h);
        const int64_t rows = ((int64_t)w.b * p.heads + h) * p.sq;
        const float slope = p.slopes ? p.slopes[h] * kLog2e : 0.0f;
        Stages<decltype(test)> stages((p.sq + SQ - 1) / SQ, lane, test);
        bool masked;
        for (int st = stages.next(&masked); st >= 0; st = stages.next(&masked)) {
            const int q0 = st * SQ;
            __syncthreads();
            fill_tile<T, D, SQ, NT>(Qs, Q, p.qs.s, q0, p.sq, p.d, p.vec, tid);
            fill_tile<T, D, SQ, NT>(Os, dO, p.dos.s, q0, p.sq, p.d, p.vec, tid);
            if (tid < SQ) {
                const int i = q0 + tid;
                Ls[0][tid] = i < p.sq ? p.lse2[rows + i] : -OPS_NEG_INF;
                Ls[1][tid] = i < p.sq ? p.delta[rows + i] : 0.0f;
                Ds[tid] = docs && i < p.sq ? p.q_doc[(int64_t)w.b * p.sq + i] : -1;
            }
            __syncthreads();
            v8 pb[NCH], db[NCH];
#pragma unroll
            for (int b = 0; b < QB; ++b) {
                f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f}, dp = {0.0f, 0.0f, 0.0f, 0.0f}, th;
#pragma unroll
                for (int dc = 0; dc < NDC; ++dc) {
                    s = M::mma(row_op<T, LD>(Qs, 16 * b, dc, g, li), kreg[dc], s);
                    dp = M::mma(row_op<T, LD>(Os, 16 * b, dc, g, li), vreg[dc], dp);
                }
                // |key - query|: the lane's row is the key here
                s = modify<T>(p, s, slope, (float)(key - (p.q_start + q0 + 16 * b + 4 * g)), &th);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * b + 4 * g + r;
                    float x = ops_exp2(s[r] - Ls[0][i]);
                    float ds = x * (dp[r] - Ls[1][i]);
                    if (cap) ds *= 1.0f - th[r] * th[r];
                    if (masked) {
                        bool see = mask.seen(key, p.q_start + q0 + i) && Ls[0][i] != -OPS_NEG_INF;
                        if (docs) see = see && kd >= 0 && Ds[i] == kd;
                        if (!see) x = ds = 0.0f;
                    }
                    pb[b / 2][4 * (b & 1) + r] = T(x);
                    db[b / 2][4 * (b & 1) + r] = T(ds);
                }
            }
            if (masked) {
                mma_seen<T>(dv, pb, [&](int i, int j) { return col_op<T, LD>(Os, 32 * i, 16 * j, g, li); });
                mma_seen<T>(dk, db, [&](int i, int j) { return col_op<T, LD>(Qs, 32 * i, 16 * j, g, li); });
            } else {
#pragma unroll
                for (int i = 0; i < NCH; ++i)
#pragma unroll
                    for (int j = 0; j < NDB; ++j) {
                        dv[j] = M::mma(col_op<T, LD>(Os, 32 * i, 16 * j, g, li), pb[i], dv[j]);
                        dk[j] = M::mma(col_op<T, LD>(Qs, 32 * i, 16 * j, g, li), db[i], dk[j]);
                    }
            }
        }
    }
    if (key >= p.sk) return;
    T* outk = p.dk ? slice<T>(p.dk, p.dks, w.b, w.hk) : nullptr;
    T* outv = p.dv ? slice<T>(p.dv, p.dvs, w.b, w.hk) : nullptr;
#pragma unroll
    for (int j = 0; j < NDB; ++j) {
        if (outk) store4<T>(outk + key * p.dks.s, 16 * j + 4 * g, p.d, p.ovec, dk[j] * p.scale);
        if (outv) store4<T>(outv + key * p.dvs.s, 16 * j + 4 * g, p.d, p.ovec, dv[j]);
    }
}

// ---------------------------------------------------------------------------
// (min, max) document of every kDocTile tokens, a wave a tile.
extern "C" __global__ __launch_bounds__(256) void fa_score_doc_ranges(ScoreParams p) {
    const int qt = (p.sq + kDocTile - 1) / kDocTile, kt = (p.sk + kDocTile - 1) / kDocTile;
    const int tile = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (tile >= p.batch * (qt + kt)) return;
    const int b = tile / (qt + kt), t = tile % (qt + kt);
    const bool isq = t < qt;
    const int at = (isq ? t : t - qt) * kDocTile + lane, n = isq ? p.sq : p.sk;
    const int32_t* ids = (isq ? p.q_doc : p.k_doc) + (int64_t)b * n;
    int lo = at < n ? ids[at] : 0x7fffffff, hi = at < n ? lo : -0x7fffffff - 1;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
        lo = min(lo, __shfl_xor(lo, s));
        hi = max(hi, __shfl_xor(hi, s));
    }
    if (lane == 0) {
        int32_t* rng = isq ? p.q_rng + 2 * ((int64_t)b * qt + t) : p.k_rng + 2 * ((int64_t)b * kt + t - qt);
        rng[0] = lo;
        rng[1] = hi;
    }
}

#define SCORE_TYPE(N, T)                                                                                    \
    extern "C" __global__ __launch_bounds__(256) void fa_score_delta_##N(ScoreParams p) { score_delta<T>(p); }
#define SCORE_KERNELS(N, T, D)                                                                              \
    extern "C" __global__ __launch_bounds__((64 * Geo<T, D>::NW)) void fa_score_forward_##N##_d##D(ScoreParams p) { \
        score_forward<T, D>(p);                                                                             \
    }                                                                                                       \
    extern "C" __global__ __launch_bounds__((64 * Geo<T, D>::NW)) void fa_score_dq_##N##_d##D(ScoreParams p) {   \
        score_dq<T, D>(p);                                                                                  \
    }                                                                                                       \
    extern "C" __global__ __launch_bounds__(512) void fa_score_dkv_##N##_d##D(ScoreParams p) { score_dkv<T, D>(p); }
SCORE_TYPE(bf16, __bf16)
SCORE_TYPE(f16, _Float16)
SCORE_TYPE(f32, float)
SCORE_KERNELS(bf16, __bf16, 64)
SCORE_KERNELS(bf16, __bf16, 128)
SCORE_KERNELS(bf16, __bf16, 256)
SCORE_KERNELS(f16, _Float16, 64)
SCORE_KERNELS(f16, _Float16, 128)
SCORE_KERNELS(f16, _Float16, 256)
SCORE_KERNELS(f32, float, 64)
SCORE_KERNELS(f32, float, 128)
SCORE_KERNELS(f32, float, 256)
