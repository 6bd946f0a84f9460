// fa_score.hip -- gfx950 kernels of attention with modified scores
// (fa_score_forward, fa_score_backward; with OPS_WINDOW defined those in a
// window, fa_window_forward and fa_window_backward, as code objects of their own).
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
//
// Built once a type: OPS_T the element type, OPS_NAME its name in the kernels'.

#include "fa_ops_common.h"

template <typename T>
__device__ __forceinline__ const T* slice(const void* base, OpsStrides st, int b, int h) {
    return reinterpret_cast<const T*>(base) + b * st.b + h * st.h;
}
template <typename T>
__device__ __forceinline__ T* slice(void* base, OpsStrides st, int b, int h) {
    return reinterpret_cast<T*>(base) + b * st.b + h * st.h;
}

// (slice, block) of a workgroup.  Without documents: the slices of a kv head share its K and V, so all its
// workgroups go to one XCD where the counts allow (workgroups go round-robin over the eight), blocks in falling
// order, the longest first where causal.  With `order` (of documents): the blocks of all batches, the longest
// first, and of every block the same heads to each XCD, so that all have the same amount of work.
struct Work {
    int b, hk, hq, blk;   // hq: head within the group
};
__device__ __forceinline__ Work find_work(unsigned id, int nblk, int nkv, int group, int kv_heads, const int32_t* order) {
    Work w;
    int kv;
    if (order) {
        const int per = kv_heads * group;
        const int item = load_uniform(order + id / per);
        int s = id % per;
        if ((per & 7) == 0) s = (s & 7) * (per >> 3) + (s >> 3);
        w.b = item / nblk;
        w.blk = item % nblk;
        w.hk = s / group;
        w.hq = s % group;
        return w;
    }
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
    // Windows: stages before `from` hold no visible pair, but for the first `sinks`, which are walked in pass `when`.
    // Last where a bias by distance may put their scores so far below the others that those would lose their low bits
    // against a reference that starts there; else first, since all workgroups start on the same rows then, in cache (32 / 8
    // heads x 8192^2, window 1024, 4 sinks: 186 us, sinks last 190).
    int from = 0, sinks = 0, when = 0, pass = 0;
    Test test;
    __device__ __forceinline__ Stages(int n, int lane_, Test t) : base(-64), count(n), lane(lane_), test(t) {}
    // next stage (-1: none); *masked: it needs the mask (an int: uniform flags stay in one scalar register)
    __device__ __forceinline__ int next(int* masked) {
        while (vis == 0) {
            base += 64;
            const bool far = kWindow && sinks && pass == when;
            if (kWindow && !far && base < from) base = from;
            if (base >= (far ? sinks : count)) {
                if (!kWindow || pass || sinks == 0) return -1;
                pass = 1;
                base = -64;
                continue;
            }
            bool p = false, v = false;
            if (base + lane < count) v = test(base + lane, &p);
            if (kWindow) v = v && (base + lane < sinks) == far;
            vis = __builtin_amdgcn_ballot_w64(v);
            part = __builtin_amdgcn_ballot_w64(v && p);
        }
        const int bit = __builtin_ctzll(vis);
        vis &= vis - 1;
        *masked = (int)(part >> bit) & 1;
        return base + bit;
    }
};

// f(stage) for every stage that holds a visible and a hidden pair.
template <typename Test, typename F>
__device__ __forceinline__ void each_masked(Test test, int count, int lane, F f) {
    Stages<Test> stages(count, lane, test);
    int masked;
    for (int st = stages.next(&masked); st >= 0; st = stages.next(&masked))
        if (masked) f(st);
}

// Keys that causal and prefix bounds leave a query at position pos: those before this.
__device__ __forceinline__ int key_limit(const ScoreParams& p, int prefix, int pos) {
    return p.causal ? max(pos + 1, prefix) : 0x7fffffff;
}

// Whether the window hides key `key` from a query at position pos.
__device__ __forceinline__ bool window_hides(const ScoreParams& p, int pos, int key, int sinks) {
    return key >= sinks && (key <= pos - p.window || key >= pos + p.window);
}
__device__ __forceinline__ bool window_hides(const ScoreParams& p, int pos, int key) {
    return window_hides(p, pos, key, p.sinks);
}

// Whether query `row` sees key `key`.
__device__ __forceinline__ bool pair_seen(const ScoreParams& p, int prefix, int b, int row, int key) {
    if (key >= key_limit(p, prefix, p.q_start + row)) return false;
    if (kWindow && window_hides(p, p.q_start + row, key)) return false;
    if (!p.q_doc) return true;
    const int d = p.q_doc[(int64_t)b * p.sq + row];
    return d >= 0 && d == p.k_doc[(int64_t)b * p.sk + key];
}

// Documents of a run of rows: the range of their ids, and whether there is padding among them.
struct DocRange {
    int lo, hi;
    bool padding;
};
__device__ __forceinline__ DocRange doc_range(const int32_t* rng, int tile) {
    const int lo = rng[2 * tile];
    return {lo < 0 ? ~lo : lo, rng[2 * tile + 1], lo < 0};
}
// Of rows [r0, r1): of the tiles they touch.
__device__ __forceinline__ DocRange doc_range(const int32_t* rng, int r0, int r1) {
    DocRange x = {0x7fffffff, -1, false};
    for (int t = r0 / kDocTile; t <= (r1 - 1) / kDocTile; ++t) {
        const DocRange y = doc_range(rng, t);
        x.lo = min(x.lo, y.lo);
        x.hi = max(x.hi, y.hi);
        x.padding = x.padding || y.padding;
    }
    return x;
}

// Whether rows of two runs may share a document; *part: whether some pair may not.
__device__ __forceinline__ bool docs_meet(const DocRange& a, const DocRange& b, bool* part) {
    if (a.padding || b.padding || !(a.lo == a.hi && b.lo == b.hi && a.lo == b.lo)) *part = true;
    return a.lo <= b.hi && b.lo <= a.hi;
}

// Whether the windows of queries at positions [lo, hi] reach keys [k0, k1); *part: whether they hide some pair.
__device__ __forceinline__ bool window_meets(const ScoreParams& p, int lo, int hi, int k0, int k1, bool* part) {
    if (k1 > p.sinks && (k0 <= hi - p.window || k1 - 1 >= lo + p.window)) *part = true;
    return k0 < p.sinks || (k1 - 1 > lo - p.window && k0 < hi + p.window);
}
// The walked stages that a window leaves: rows before `sinks` (where they are walked for their own sake) and rows
// [lo, hi], of n stages of ROWS.
template <int ROWS, typename S>
__device__ __forceinline__ void window_stages(S* s, int sinks, bool last, int lo, int hi, int n) {
    const int first = (sinks + ROWS - 1) / ROWS;
    s->sinks = first;
    s->when = last ? 1 : 0;
    s->count = min(n, max(first, hi < 0 ? 0 : hi / ROWS + 1));
    s->from = lo <= 0 ? 0 : lo / ROWS;
}

// One value a lane from global memory into LDS, zero past n.
__device__ __forceinline__ void fill_words(void* dst, const void* src, int n, int lane) {
    const int bytes = 4 * min(max(n, 0), 64);   // (of 2^30 words the size would not fit)
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(src), (short)0, bytes, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)dst, 4, 4 * lane, 0, 0, 0);
}

// Walked rows of a stage: 32 at least for each of the KG groups of waves that share them out.
template <typename T, int D, int KG>
constexpr int kStageRows = KG == 1 && (sizeof(T) == 4 || D > 128) ? 32 : 64;

// Whether queries [q0, q1), of the documents qr, see a key of stage st, and whether
// some pair is hidden.
template <int SK>
__device__ __forceinline__ bool key_stage(const ScoreParams& p, int prefix, int st, int q0, int q1, bool docs,
                                          const DocRange& qr, const int32_t* krng, bool* part) {
    const int k0 = st * SK, k1 = k0 + SK;
    bool v = true;
    if (k1 > p.sk) *part = true;
    if (p.causal) {
        v = k0 <= p.q_start + q1 - 1 || k0 < prefix;
        if (!(k1 - 1 <= p.q_start + q0 || k1 <= prefix)) *part = true;
    }
    if (kWindow && v) v = window_meets(p, p.q_start + q0, p.q_start + q1 - 1, k0, k1, part);
    if (docs && v) v = docs_meet(qr, doc_range(krng, k0 / kDocTile), part);
    return v;
}
// The stages of keys that the windows of queries [q0, q1) leave.
template <int SK, typename S>
__device__ __forceinline__ void window_keys(const ScoreParams& p, S* s, bool last, int q0, int q1) {
    if (!kWindow) return;
    const int up = p.causal && !p.prefix ? 0 : p.window - 1;
    window_stages<SK>(s, p.sinks, last, p.q_start + q0 - p.window + 1, p.q_start + q1 - 1 + up, s->count);
}
// Whether rows of a wave at positions [lo, hi] see a key of [k0, k1), as far as the window tells.
__device__ __forceinline__ bool window_active(const ScoreParams& p, int lo, int hi, int k0, int k1) {
    bool part;
    return !kWindow || window_meets(p, lo, hi, k0, k1, &part);
}

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------
// Four waves of MT 16-row tiles (KG = 2: two groups of two waves keep the same rows, each with half of a stage's
// keys, and their sums meet in LDS at the end: twice the workgroups, each half as long).  K and V tiles are
// double-buffered and filled by DMA: while a stage's softmax and PV product run, K of the stage after the next and V
// of the next arrive; one barrier a stage.  The loop is unrolled by two so that each buffer is an array of its own.
//
// Bound by the issue of vector instructions (five a score, ten with a cap, transcendental ones counted twice) and of
// products, which overlap little with two waves a SIMD: bf16, 2 x 16 x 4096^2 all visible, 128 columns 281 us
// (978 TF/s), capped 339 us (810); causal 140 us (980); 64 columns, 4 x 16 x 4096^2 causal 183 us (750).
// In a window the walk of a workgroup is short (1024 of 8192 tokens, 128 query rows: 18 tiles of 64 keys), so that its
// start, the masked tiles at its two ends and the one of the sinks weigh more: bf16, 32 heads of 128 columns, 8192 tokens,
// window 1024 and 4 sinks 186 us (690 TF/s of visible pairs; matrix units busy 34 % of the time, vector units 45 %).
template <typename T, int D, int MT, int KG, int MOD, bool VEC>
__device__ __forceinline__ void score_forward(const ScoreParams& p) {
    using M = Mma<T>;
    using v8 = typename M::v8;
    constexpr int NW = 4, NR = NW / KG, SK = kStageRows<T, D, KG>, SW = SK / KG, BQ = 16 * MT * NR;
    constexpr int KB = SW / 16, NCH = SW / 32, NDC = D / 32, NDB = D / 16, LD = D + kPad<T>;
    using Fill = TileFill<T, D, SK, NW, VEC>;
    T* const Kb0 = lds_array<T, Fill::SIZE, 0>();
    T* const Vb0 = lds_array<T, Fill::SIZE, 1>();
    T* const Kb1 = lds_array<T, Fill::SIZE, 2>();
    T* const Vb1 = lds_array<T, Fill::SIZE, 3>();
    int* const Db0 = lds_array<int, 64, 4>();   // documents of the stage's keys
    int* const Db1 = lds_array<int, 64, 5>();
    int* const Special = lds_array<int, 1, 6>();   // V held infinities or NaN in a masked stage

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, li = lane & 15;
    const Work w = find_work(blockIdx.x, p.nqb, p.batch * p.kv_heads, p.group, p.kv_heads, p.q_order);
    const int h = w.hk * p.group + w.hq;
    const int kg = wave / NR, koff = kg * SW;   // the wave's keys of a stage: koff .. koff + SW - 1
    const int q0 = w.blk * BQ, row0 = q0 + 16 * MT * (wave % NR);
    const T* Q = slice<T>(p.q, p.qs, w.b, h);
    const T* K = slice<T>(p.k, p.ks, w.b, w.hk);
    const T* V = slice<T>(p.v, p.vs, w.b, w.hk);
    const bool docs = p.q_doc != nullptr;
    const int32_t* kdoc = docs ? p.k_doc + (int64_t)w.b * p.sk : nullptr;
    const int prefix = p.prefix ? load_uniform(p.prefix + w.b) : 0;
    const float slope = has_bias<MOD>(p) ? load_uniform(p.slopes + h) * kLog2e : 0.0f;
    const bool cap = has_cap<MOD>(p);
    // scores leave the QK^T chains raw, and the scale goes into the exponent; modified ones are in log2 units
    const float c = MOD != 0 ? 1.0f : p.scale_log2e;

    v8 qreg[MT][NDC];
    int qd[MT], limit[MT];   // a row's document, and the keys before which it may see
    f32x4 o[MT][NDB];
    float m[MT], l[MT], ref[MT];   // l: the lane's share of the row's sum; ref: m, or 0 while m = -inf
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = row0 + 16 * t + li;
#pragma unroll
        for (int dc = 0; dc < NDC; ++dc) qreg[t][dc] = global_row<T, VEC>(Q, p.qs.s, row, p.sq, 32 * dc + 8 * g, p.d);
        qd[t] = docs && row < p.sq ? p.q_doc[(int64_t)w.b * p.sq + row] : -1;
        limit[t] = docs && qd[t] < 0 ? 0 : min(p.sk, key_limit(p, prefix, p.q_start + row));
#pragma unroll
        for (int j = 0; j < NDB; ++j) o[t][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        m[t] = OPS_NEG_INF;
        l[t] = ref[t] = 0.0f;
    }

    const int q1 = min(q0 + BQ, p.sq);
    DocRange qr = {};
    const int32_t* krng = nullptr;
    if (docs) {
        qr = doc_range(p.q_rng + (int64_t)w.b * 2 * ((p.sq + kDocTile - 1) / kDocTile), q0, q1);
        krng = p.k_rng + (int64_t)w.b * 2 * ((p.sk + kDocTile - 1) / kDocTile);
    }
    auto test = [&](int st, bool* part) -> bool { return key_stage<SK>(p, prefix, st, q0, q1, docs, qr, krng, part); };
    Stages<decltype(test)> stages((p.sk + SK - 1) / SK, lane, test);
    window_keys<SK>(p, &stages, has_bias<MOD>(p), q0, q1);
    const Fill kfill(p.ks.s, p.d, wave, lane), vfill(p.vs.s, p.d, wave, lane);
    auto fill_k = [&](int st, T* dst, int* ids) {
        kfill(dst, K, st * SK, p.sk);
        if (docs && wave == 0 && lane < SK) fill_words(ids, kdoc + st * SK, p.sk - st * SK, lane);
    };

    // S^T of a stage, relative to the rows' references (modified: log2 units, and what 16-bit weights are taken
    // larger by)
    constexpr int PRE_K = NDC > 1 ? 2 : 1;
    constexpr float kUp = MOD != 0 ? kProbLog2<T> : 0.0f;
    f32x4 s[MT][KB];
    auto qk = [&](const T* Ks, int k0) {
        constexpr int KR = PRE_K + 1;
        v8 kk[KR][KB];
#pragma unroll
        for (int dc = 0; dc < PRE_K && dc < NDC; ++dc)
#pragma unroll
            for (int b = 0; b < KB; ++b) kk[dc][b] = row_op<T, LD>(Ks, koff + 16 * b, dc, g, li);
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const float x = MOD != 0 ? 0.0f : -ref[t];
                s[t][b] = (f32x4){x, x, x, x};
            }
#pragma unroll
        for (int dc = 0; dc < NDC; ++dc) {
            if (dc + PRE_K < NDC) {
#pragma unroll
                for (int b = 0; b < KB; ++b) kk[(dc + PRE_K) % KR][b] = row_op<T, LD>(Ks, koff + 16 * b, dc + PRE_K, g, li);
            }
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int t = 0; t < MT; ++t) s[t][b] = M::mma(kk[dc % KR][b], qreg[t][dc], s[t][b]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (MOD != 0) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const float dist = (float)(p.q_start + row0 + 16 * t + li - k0 - koff - 4 * g);
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    if (cap) {
                        s[t][b] = capped_over<T, MOD>(s[t][b], p.cap_in, p.cap_log2e, ref[t] - kUp);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][b][r] = __builtin_fmaf(s[t][b][r], p.scale_log2e, kUp - ref[t]);
                    }
                    if (has_bias<MOD>(p)) {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            s[t][b][r] = __builtin_fmaf(-slope, fabsf(dist - (float)(16 * b + r)), s[t][b][r]);
                    }
                }
            }
        }
    };
    auto hide = [&](int k0, const int* ids) {
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const int key = k0 + koff + 16 * b + 4 * g;
            if (docs) {
                const i32x4 kd = *reinterpret_cast<const i32x4*>(ids + koff + 16 * b + 4 * g);
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (kd[r] != qd[t]) s[t][b][r] = OPS_NEG_INF;
            }
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (key + r >= limit[t]) s[t][b][r] = OPS_NEG_INF;
        }
        if constexpr (kWindow) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int pos = p.q_start + row0 + 16 * t + li - k0 - koff - 4 * g;
#pragma unroll
                for (int b = 0; b < KB; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (window_hides(p, pos, 16 * b + r, p.sinks - k0 - koff - 4 * g)) s[t][b][r] = OPS_NEG_INF;
            }
        }
    };
    v8 pb[MT][NCH];
    float sum[MT];
    // At 128 columns the weights of a stage's second 32 keys are taken between the products of the first
    // (16 heads x 2 x 4096^2, bf16: 314 -> 287 us all visible, 172 -> 158 causal; nothing at 64 columns).
    constexpr bool kMix = D == 128 && NCH == 2;
    // The weights of two scores a lane of 32 keys, pair e of its 4 MT, in two steps.
    auto weigh2 = [&](int ch, int e, int step) {
        const int t = e / 4, b = 2 * ch + e % 4 / 2;
#pragma unroll
        for (int r = 2 * (e & 1); r < 2 * (e & 1) + 2; ++r) {
            const float x = s[t][b][r];
            if (step == 0) {
                s[t][b][r] = ops_exp2(MOD != 0 ? x : __builtin_fmaf(x, c, kProbLog2<T>));
            } else {
                pb[t][ch][4 * (b & 1) + r] = T(x);
                sum[t] += x;
            }
        }
    };
    auto softmax = [&] {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            float mt = s[t][0][0];
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) mt = __builtin_elementwise_maximum(mt, s[t][b][r]);
            mt -= kUp;
            // the reference moves only when a score passes it by more than kLazy, or at a row's first key
            const bool seen = m[t] != OPS_NEG_INF;
            const float limit = seen ? kLazy : OPS_NEG_INF;
            if (__builtin_amdgcn_ballot_w64(mt * c > limit) != 0) {
                mt = row4_max(mt);
                const bool grow = mt * c > limit;
                const float delta = grow ? mt : 0.0f;
#pragma unroll
                for (int b = 0; b < KB; ++b) s[t][b] -= delta;
                if (grow) m[t] = ref[t] = ref[t] + delta;
                if (__builtin_amdgcn_ballot_w64(grow && seen) != 0) {
                    const float corr = grow && seen ? ops_exp2(-delta * c) : 1.0f;
                    l[t] *= corr;
#pragma unroll
                    for (int j = 0; j < NDB; ++j) o[t][j] *= corr;
                }
            }
            sum[t] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8 * MT * (kMix ? 1 : NCH); ++e) weigh2(e / (8 * MT), e / 2 % (4 * MT), e & 1);
    };
    constexpr int PRE_V = NCH * NDB >= 4 ? 3 : 1, VR = PRE_V + 1;
    v8 va[VR];
    auto v_op = [&](const T* Vs, int i) { return col_op<T, LD>(Vs, koff + 32 * (i / NDB), 16 * (i % NDB), g, li); };
    auto pv_preload = [&](const T* Vs) {
#pragma unroll
        for (int i = 0; i < PRE_V; ++i) va[i] = v_op(Vs, i);
    };
    auto pv = [&](const T* Vs) {
#pragma unroll
        for (int i = 0; i < NCH * NDB; ++i) {
            if (i + PRE_V < NCH * NDB) va[(i + PRE_V) % VR] = v_op(Vs, i + PRE_V);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                o[t][i % NDB] = M::mma(va[i % VR], pb[t][i / NDB], o[t][i % NDB]);
                if (kMix && i < NDB) {
                    constexpr int PER = NDB / 4;   // products a pair
                    const int n = i % NDB * MT + t;
                    if (n % PER == 0) weigh2(NCH - 1, n / PER, 0);
                    if (n % PER == PER - 1) weigh2(NCH - 1, n / PER, 1);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) l[t] += sum[t];
    };
    // whether some row of the wave sees some key of the stage (as far as causal and prefix tell)
    auto active = [&](int st) -> int {
        if (st < 0 || row0 >= p.sq) return false;
        const int k0 = st * SK + koff;
        return k0 < p.sk && (!p.causal || k0 <= p.q_start + row0 + 16 * MT - 1 || k0 < prefix) &&
               window_active(p, p.q_start + row0, p.q_start + row0 + 16 * MT - 1, k0, k0 + SW);
    };

    // At 128 columns and more, waves in their products go before waves of the other workgroup in their softmax
    // (16 heads x 4096^2 all visible, bf16: 286 -> 269 us; capped 411 -> 378; slower at 64 columns)
    constexpr bool kPrio = D >= 128;
    int masked = 0, masked_next = 0;
    int st = stages.next(&masked), nx = st < 0 ? -1 : stages.next(&masked_next);
    if (st >= 0) {
        fill_k(st, Kb0, Db0);
        vfill(Vb0, V, st * SK, p.sk);
    }
    if (nx >= 0) fill_k(nx, Kb1, Db1);
    if (tid == 0) *Special = 0;
    wait_loads();
    __syncthreads();
    if (st >= 0 && masked && vfill.template special<true>(Vb0)) *Special = 1;
    int act = active(st);
    if (act) {
        qk(Kb0, st * SK);
        if (masked) hide(st * SK, Db0);
    }
    __syncthreads();
    auto step = [&](auto parity) {
        constexpr int P = decltype(parity)::value;
        T* const k_cur = P ? Kb1 : Kb0;
        T* const k_next = P ? Kb0 : Kb1;
        T* const v_cur = P ? Vb1 : Vb0;
        T* const v_next = P ? Vb0 : Vb1;
        int masked_after = 0;
        const int after = nx < 0 ? -1 : stages.next(&masked_after);
        if (after >= 0) fill_k(after, k_cur, P ? Db1 : Db0);
        if (nx >= 0) vfill(v_next, V, nx * SK, p.sk);
        if (act) {
            pv_preload(v_cur);
            softmax();
            if (kPrio) __builtin_amdgcn_s_setprio(1);
            pv(v_cur);
            if (kPrio) __builtin_amdgcn_s_setprio(0);
        }
        act = active(nx);
        if (act) {
            if (kPrio) __builtin_amdgcn_s_setprio(1);
            qk(k_next, nx * SK);
            if (kPrio) __builtin_amdgcn_s_setprio(0);
            if (masked_next) hide(nx * SK, P ? Db0 : Db1);
        }
        wait_loads();
        if (masked_next && vfill.template special<true>(v_next)) *Special = 1;
        __syncthreads();
        st = nx, masked = masked_next;
        nx = after, masked_next = masked_after;
    };
    while (st >= 0) {
        step(std::integral_constant<int, 0>{});
        if (st < 0) break;
        step(std::integral_constant<int, 1>{});
    }

    const ScoreParams lp = late_params<ScoreParams>();
    if constexpr (KG > 1) {
        // the last stage's barrier freed the tiles
        static_assert(MT == 1 && KG == 2 && NR * NDB * 64 * 16 <= Fill::SIZE * (int)sizeof(T), "sums fit a tile");
        f32x4* const sums = reinterpret_cast<f32x4*>(Kb0) + wave % NR * NDB * 64;
        float* const ml = reinterpret_cast<float*>(Vb0) + wave % NR * 128;
        if (kg == 1) {
#pragma unroll
            for (int j = 0; j < NDB; ++j) sums[j * 64 + lane] = o[0][j];
            ml[lane] = m[0];
            ml[64 + lane] = l[0];
        }
        __syncthreads();
        if (kg == 1) return;
        const float m2 = ml[lane], mn = fmaxf(m[0], m2), top = mn == OPS_NEG_INF ? 0.0f : mn;
        const float c1 = ops_exp2((m[0] - top) * c), c2 = ops_exp2((m2 - top) * c);
        m[0] = mn;
        l[0] = l[0] * c1 + ml[64 + lane] * c2;
#pragma unroll
        for (int j = 0; j < NDB; ++j) o[0][j] = o[0][j] * c1 + sums[j * 64 + lane] * c2;
    }
    T* O = slice<T>(lp.out, lp.os, w.b, h);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = row0 + 16 * t + li;
        const float lt = row4_sum(l[t]);
        if (row >= lp.sq) continue;
        const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
#pragma unroll
        for (int j = 0; j < NDB; ++j) store4<T, VEC>(O + row * lp.os.s, 16 * j + 4 * g, lp.d, o[t][j] * inv);
        if (lp.lse && g == 0) {
            const float lse = (m[t] * c + __builtin_log2f(lt) - kProbLog2<T>) * kLn2;
            lp.lse[((int64_t)w.b * lp.heads + h) * lp.sq + row] = lt == 0.0f ? OPS_NEG_INF : lse;
        }
    }
    if (*Special) {
        __threadfence();
        each_masked(test, stages.count, lane, [&](int stage) {
            add_specials<T, T, true>(
                stage * SK, min(stage * SK + SK, lp.sk), min(16 * MT, lp.sq - row0), lp.d, lane,
                [&](int key) { return V + key * lp.vs.s; },
                [&](int key, int r) { return pair_seen(lp, prefix, w.b, row0 + r, key); },
                [&](int r) { return O + (row0 + r) * lp.os.s; });
        });
    }
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------

// Of four scores: the weights p = e^(z - lse), the gradients y = p (dP - delta) of the modified scores z, and
// what these have to be multiplied by for the raw ones (1 - tanh^2; 1 without a cap).
template <typename T, int MOD>
__device__ __forceinline__ void weigh(const ScoreParams& p, bool cap, f32x4 s, f32x4 dp, f32x4 lse2, f32x4 delta,
                                      float slope, float dist, f32x4* w, f32x4* y, f32x4* f) {
    f32x4 th, capped_s;
    if (cap) capped_s = capped<T, MOD>(s, p.cap_in, p.cap_log2e, &th);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        float z = cap ? capped_s[r] - lse2[r] : __builtin_fmaf(s[r], p.scale_log2e, -lse2[r]);
        if (has_bias<MOD>(p)) z = __builtin_fmaf(-slope, fabsf(dist - (float)r), z);
        const float x = ops_exp2(z);
        (*w)[r] = x;
        (*y)[r] = x * (dp[r] - delta[r]);
        (*f)[r] = cap ? __builtin_fmaf(-th[r], th[r], 1.0f) : 1.0f;
    }
}

// Operands of the gradient kernels' products that are read from LDS ahead of their use: PRE steps, and the first ones
// of the column products before the weights are formed (bf16, 2 x 4096 tokens, 16 heads of 128 columns, documents,
// capped: forward and backward 644 -> 606 us; 16 heads x 2 x 4096^2 all visible, backward 1207 -> 1132; three steps:
// no more).
template <typename T>
constexpr int kAhead = sizeof(T) == 2 ? 2 : 1;

// f16: weights p and score gradients enter their products 2^kGradLog2 times larger, so that those down to 2^-26 round as
// normal numbers (gradients of a mean over many tokens are that small): p by an lse2 that is smaller by kGradLog2,
// and the gradients with it.  Gradients that would then pass the type's range are scaled down, each kept row's by itself,
// with its sums so far: GradScale.  Looking for them takes a vector instruction a score (backward, f16, 2 x 16 x 4096^2:
// 128 columns, all visible 1142 us without, 1175 with it; 64 columns, 4 kv heads, causal 382 and 407).
template <typename T>
constexpr float kGradLog2 = std::is_same<T, _Float16>::value ? 12.0f : 0.0f;
template <typename T>
constexpr float kGradInv = std::is_same<T, _Float16>::value ? 0x1p-12f : 1.0f;

// What a kept row's score gradients are scaled down by, a power of two u (1 where T has the range of f32).
template <typename T, int D, int MT>
struct GradScale {
    static constexpr bool kOn = std::is_same<T, _Float16>::value;
    float limit[MT];   // 2^15 / u: larger ones are brought down
    int any = 0;       // some row's u is not 1
    __device__ __forceinline__ GradScale() {
#pragma unroll
        for (int t = 0; t < MT; ++t) limit[t] = 0x1p15f;
    }
    // Brings the gradients of two blocks of rows into range; where they pass it, down to 2^13 .. 2^14 with the sums.
    template <int N>
    __device__ __forceinline__ void fit(int t, f32x4 (&y)[2], f32x4 (&sums)[N]) {
        if constexpr (kOn) {
            float mx = 0.0f;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, fabsf(y[b][r]));
            // (at 256 columns, where registers are short, dQ takes 170 us without these two hints and the second
            // branch, which spares a product a score, and 192 with them)
            constexpr bool kShort = D > 128;
            const bool pass = __builtin_amdgcn_ballot_w64(mx > limit[t]) != 0;
            if (kShort ? pass : __builtin_expect(pass, 0)) {
                any = 1;
                mx = row4_max(mx);
                if (mx > limit[t] && !not_finite(mx)) {
                    // 2^15 / u from the exponent of mx, and its inverse
                    const unsigned larger = (min(__float_as_uint(mx) >> 23, 250u) + 2) << 23;
                    const float by = limit[t] * __uint_as_float((254u << 23) - larger);
                    limit[t] = __uint_as_float(larger);
#pragma unroll
                    for (int j = 0; j < N; ++j) sums[j] *= by;
                }
            }
            if (kShort || __builtin_expect(any, 0)) {
                const float u = __uint_as_float(((254u + 15u) << 23) - __float_as_uint(limit[t]));   // 2^15 / limit
                y[0] *= u;
                y[1] *= u;
            }
        }
    }
    __device__ __forceinline__ float inverse(int t) const { return kOn ? limit[t] * 0x1p-15f : 1.0f; }
};

// dQ: query rows kept, keys walked.  Four waves of MT 16-row tiles; K and V tiles double-buffered, one barrier a stage.
// On the way in a wave leaves delta = dO . O and lse2 = lse log2(e) of its rows for the dK / dV kernel.  Empty rows get
// lse2 = +inf: their weights e^(z - lse) then come out as 0.
//
// 16-bit types: delta = dO . O comes from the rounded O, and an error of delta is common to all keys of a row, so
// it does not average out: it was the largest error of dQ and dK (bf16, 2 x 4096 tokens, documents, capped scores:
// 3.3e-3 relative, of which 1.7e-3 is the rounding of the results; 2.4e-3 now).  But sum_j p (dP - delta) is just
// that error e.  It is summed on the way, as is sum_j p K_j (its operands are in registers anyway); dQ is corrected
// by -e sum_j p K_j, and delta + e left for the dK / dV kernel, which runs after this one.  The third product takes
// the kernel from 1089 to 764 TF/s (two products counted; 4096^2, 16 heads of 128 columns), the whole backward pass
// of that shape from 1036 to 1171 us, and that of the documents above from 497 to 507.
template <typename T, int D, int MT, int KG, int MOD, bool VEC>
__device__ __forceinline__ void score_dq(const ScoreParams& p) {
    using M = Mma<T>;
    using v8 = typename M::v8;
    constexpr bool kRefine = sizeof(T) == 2;
    constexpr int NW = 4, NR = NW / KG, SK = kStageRows<T, D, KG>, BQ = 16 * MT * NR;
    constexpr int NCH = SK / 32 / KG, NDC = D / 32, NDB = D / 16, LD = D + kPad<T>;
    constexpr int PRE = D > 128 ? 1 : kAhead<T>;   // (at 256 columns registers are short)
    using Fill = TileFill<T, D, SK, NW, VEC>;
    T* const Kb0 = lds_array<T, Fill::SIZE, 0>();
    T* const Vb0 = lds_array<T, Fill::SIZE, 1>();
    T* const Kb1 = lds_array<T, Fill::SIZE, 2>();
    T* const Vb1 = lds_array<T, Fill::SIZE, 3>();
    int* const Db0 = lds_array<int, 64, 4>();
    int* const Db1 = lds_array<int, 64, 5>();
    int* const Special = lds_array<int, 3, 6>();   // met any; and the tiles of either buffer hold some

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, li = lane & 15;
    const Work w = find_work(blockIdx.x, p.nqb, p.batch * p.kv_heads, p.group, p.kv_heads, p.q_order);
    const int h = w.hk * p.group + w.hq;
    const int kg = wave / NR, koff = kg * 32 * NCH;   // the wave's keys of a stage
    const int q0 = w.blk * BQ, row0 = q0 + 16 * MT * (wave % NR);
    const T* Q = slice<T>(p.q, p.qs, w.b, h);
    const T* dO = slice<T>(p.dout, p.dos, w.b, h);
    const T* K = slice<T>(p.k, p.ks, w.b, w.hk);
    const T* V = slice<T>(p.v, p.vs, w.b, w.hk);
    const bool docs = p.q_doc != nullptr;
    const int32_t* kdoc = docs ? p.k_doc + (int64_t)w.b * p.sk : nullptr;
    const int prefix = p.prefix ? load_uniform(p.prefix + w.b) : 0;
    const float slope = has_bias<MOD>(p) ? load_uniform(p.slopes + h) * kLog2e : 0.0f;
    const bool cap = has_cap<MOD>(p);

    v8 qreg[MT][NDC], doreg[MT][NDC];
    int qd[MT], limit[MT];
    f32x4 dq[MT][NDB], pk[MT][kRefine ? NDB : 1];
    float lse2[MT], delta[MT], err[MT];
    GradScale<T, D, MT> down;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = row0 + 16 * t + li;
        const int64_t at = ((int64_t)w.b * p.heads + h) * p.sq + row;
#pragma unroll
        for (int dc = 0; dc < NDC; ++dc) {
            qreg[t][dc] = global_row<T, VEC>(Q, p.qs.s, row, p.sq, 32 * dc + 8 * g, p.d);
            doreg[t][dc] = global_row<T, VEC>(dO, p.dos.s, row, p.sq, 32 * dc + 8 * g, p.d);
        }
        qd[t] = docs && row < p.sq ? p.q_doc[(int64_t)w.b * p.sq + row] : -1;
        const T* O = slice<T>(p.out_in, p.os, w.b, h);
        float sum = 0.0f;
#pragma unroll
        for (int dc = 0; dc < NDC; ++dc) {
            const v8 o = global_row<T, VEC>(O, p.os.s, row, p.sq, 32 * dc + 8 * g, p.d);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += float(o[e]) * float(doreg[t][dc][e]);
        }
        delta[t] = row4_sum(sum);
        const float lse = row < p.sq ? p.lse_in[at] : OPS_NEG_INF;
        lse2[t] = lse == OPS_NEG_INF    ? -OPS_NEG_INF
                  : lse == -OPS_NEG_INF ? __builtin_nanf("")
                                        : lse * kLog2e - kGradLog2<T>;
        if (row < p.sq && g == 0 && kg == 0) {
            p.lse2[at] = lse2[t];
            p.delta[at] = delta[t];
        }
        limit[t] = (docs && qd[t] < 0) || lse2[t] == -OPS_NEG_INF ? 0 : min(p.sk, key_limit(p, prefix, p.q_start + row));
#pragma unroll
        for (int j = 0; j < NDB; ++j) {
            dq[t][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
            if (kRefine) pk[t][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        }
        err[t] = 0.0f;
    }
    if (!p.dq && !(kRefine && p.dk)) return;   // the dK / dV kernel wants lse2 and delta alone
    const int q1 = min(q0 + BQ, p.sq);
    DocRange qr = {};
    const int32_t* krng = nullptr;
    if (docs) {
        qr = doc_range(p.q_rng + (int64_t)w.b * 2 * ((p.sq + kDocTile - 1) / kDocTile), q0, q1);
        krng = p.k_rng + (int64_t)w.b * 2 * ((p.sk + kDocTile - 1) / kDocTile);
    }
    auto test = [&](int st, bool* part) -> bool { return key_stage<SK>(p, prefix, st, q0, q1, docs, qr, krng, part); };
    Stages<decltype(test)> stages((p.sk + SK - 1) / SK, lane, test);
    window_keys<SK>(p, &stages, false, q0, q1);
    const Fill kfill(p.ks.s, p.d, wave, lane), vfill(p.vs.s, p.d, wave, lane);
    auto fill = [&](int st, T* k, T* v, int* ids) {
        kfill(k, K, st * SK, p.sk);
        vfill(v, V, st * SK, p.sk);
        if (docs && wave == 0 && lane < SK) fill_words(ids, kdoc + st * SK, p.sk - st * SK, lane);
    };
    auto active = [&](int st) -> int {
        if (row0 >= p.sq) return false;
        const int k0 = st * SK + koff;
        return k0 < p.sk && (!p.causal || k0 <= p.q_start + row0 + 16 * MT - 1 || k0 < prefix) &&
               window_active(p, p.q_start + row0, p.q_start + row0 + 16 * MT - 1, k0, k0 + 32 * NCH);
    };

    int masked = 0, masked_next = 0;
    int st = stages.next(&masked);
    if (tid < 3) Special[tid] = 0;
    if (st >= 0) fill(st, Kb0, Vb0, Db0);
    wait_loads();
    __syncthreads();
    if (masked && kfill.template special<false>(Kb0)) Special[1] = 1;
    __syncthreads();
    auto step = [&](auto parity) {
        constexpr int P = decltype(parity)::value;
        T* const Ks = P ? Kb1 : Kb0;
        T* const Vs = P ? Vb1 : Vb0;
        const int* const ids = P ? Db1 : Db0;
        const int nx = stages.next(&masked_next);
        if (nx >= 0) fill(nx, P ? Kb0 : Kb1, P ? Vb0 : Vb1, P ? Db0 : Db1);
        const int k0 = st * SK;
        const int act = active(st), dirty = masked ? __builtin_amdgcn_readfirstlane(Special[1 + P]) : 0;
        v8 ca[PRE + 1];
        auto col = [&](int i, int j) { ca[j % (PRE + 1)] = col_op<T, LD>(Ks, koff + 32 * i, 16 * j, g, li); };
        auto preload = [&](int i) {
#pragma unroll
            for (int j = 0; j < PRE; ++j) col(i, j);
        };
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            v8 db[MT], pb[MT];
            if (act) {
                f32x4 s[MT][2], dp[MT][2];
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int b = 0; b < 2; ++b) s[t][b] = dp[t][b] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
                v8 ka[PRE + 1], va[PRE + 1];
                auto load = [&](int n) {   // operands of key block n % 2, columns 32 (n / 2)
                    ka[n % (PRE + 1)] = row_op<T, LD>(Ks, koff + 32 * i + 16 * (n % 2), n / 2, g, li);
                    va[n % (PRE + 1)] = row_op<T, LD>(Vs, koff + 32 * i + 16 * (n % 2), n / 2, g, li);
                };
#pragma unroll
                for (int n = 0; n < PRE; ++n) load(n);
#pragma unroll
                for (int n = 0; n < 2 * NDC; ++n) {
                    if (n + PRE < 2 * NDC) load(n + PRE);
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        s[t][n % 2] = M::mma(ka[n % (PRE + 1)], qreg[t][n / 2], s[t][n % 2]);
                        dp[t][n % 2] = M::mma(va[n % (PRE + 1)], doreg[t][n / 2], dp[t][n % 2]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (!dirty) preload(i);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const int pos = p.q_start + row0 + 16 * t + li;
                    f32x4 x[2], y[2];   // y: gradients of the raw scores
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        f32x4 f;
                        const int key = k0 + koff + 32 * i + 16 * b + 4 * g;
                        weigh<T, MOD>(p, cap, s[t][b], dp[t][b], (f32x4){lse2[t], lse2[t], lse2[t], lse2[t]},
                                      (f32x4){delta[t], delta[t], delta[t], delta[t]}, slope, (float)(pos - key), &x[b],
                                      &y[b], &f);
                        if (masked) {
                            if (docs) {
                                const i32x4 kd = *reinterpret_cast<const i32x4*>(ids + koff + 32 * i + 16 * b + 4 * g);
#pragma unroll
                                for (int r = 0; r < 4; ++r)
                                    if (kd[r] != qd[t]) x[b][r] = y[b][r] = 0.0f;
                            }
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (key + r >= limit[t]) x[b][r] = y[b][r] = 0.0f;
                            if constexpr (kWindow) {
#pragma unroll
                                for (int r = 0; r < 4; ++r)
                                    if (window_hides(p, pos, key + r)) x[b][r] = y[b][r] = 0.0f;
                            }
                        }
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if (kRefine) {
                                pb[t][4 * b + r] = T(x[b][r] * f[r]);
                                err[t] += y[b][r];
                            }
                            y[b][r] *= f[r];
                        }
                    }
                    down.fit(t, y, dq[t]);
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int r = 0; r < 4; ++r) db[t][4 * b + r] = T(y[b][r]);
                }
            }
            if (dirty) {   // the row products took K as it is, the column products may not
                __syncthreads();
                if (tile_clean<T, LD, D, 32 * KG, 64 * NW>(Ks + 32 * i * LD, tid)) *Special = 1;
                __syncthreads();
                if (act) preload(i);
            }
            if (act) {
#pragma unroll
                for (int j = 0; j < NDB; ++j) {
                    if (j + PRE < NDB) col(i, j + PRE);
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        dq[t][j] = M::mma(ca[j % (PRE + 1)], db[t], dq[t][j]);
                        if (kRefine) pk[t][j] = M::mma(ca[j % (PRE + 1)], pb[t], pk[t][j]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        wait_loads();
        if (nx >= 0 && masked_next && kfill.template special<false>(P ? Kb0 : Kb1)) Special[2 - P] = 1;
        if (dirty && tid == 0) Special[1 + P] = 0;
        __syncthreads();
        st = nx, masked = masked_next;
    };
    while (st >= 0) {
        step(std::integral_constant<int, 0>{});
        if (st < 0) break;
        step(std::integral_constant<int, 1>{});
    }
    const ScoreParams lp = late_params<ScoreParams>();
    if constexpr (down.kOn) {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const float by = down.inverse(t) * kGradInv<T>;
            err[t] *= kGradInv<T>;
#pragma unroll
            for (int j = 0; j < NDB; ++j) {
                dq[t][j] *= by;
                pk[t][j] *= kGradInv<T>;
            }
        }
    }
    if constexpr (KG > 1) {
        static_assert(MT == 1 && KG == 2 && NCH == 1 && NR * NDB * 64 * 16 <= Fill::SIZE * (int)sizeof(T), "sums fit a tile");
        f32x4* const sums = reinterpret_cast<f32x4*>(Kb0) + wave % NR * NDB * 64;
        f32x4* const psums = reinterpret_cast<f32x4*>(Vb0) + wave % NR * NDB * 64;
        float* const errs = reinterpret_cast<float*>(Kb1) + wave % NR * 64;
        if (kg == 1) {
#pragma unroll
            for (int j = 0; j < NDB; ++j) {
                sums[j * 64 + lane] = dq[0][j];
                if (kRefine) psums[j * 64 + lane] = pk[0][j];
            }
            if (kRefine) errs[lane] = err[0];
        }
        __syncthreads();
        if (kg == 1) return;
#pragma unroll
        for (int j = 0; j < NDB; ++j) {
            dq[0][j] += sums[j * 64 + lane];
            if (kRefine) pk[0][j] += psums[j * 64 + lane];
        }
        if (kRefine) err[0] += errs[lane];
    }
    if constexpr (kRefine) {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int row = row0 + 16 * t + li;
            const float e = row4_sum(err[t]);
            if (row < lp.sq && g == 0)
                lp.delta[((int64_t)w.b * lp.heads + h) * lp.sq + row] = delta[t] + e;
#pragma unroll
            for (int j = 0; j < NDB; ++j) dq[t][j] -= pk[t][j] * e;
        }
    }
    if (!lp.dq) return;
    T* out = slice<T>(lp.dq, lp.dqs, w.b, h);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = row0 + 16 * t + li;
        if (row >= lp.sq) continue;
#pragma unroll
        for (int j = 0; j < NDB; ++j) store4<T, VEC>(out + row * lp.dqs.s, 16 * j + 4 * g, lp.d, dq[t][j] * lp.scale);
    }
    if (*Special) {
        __threadfence();
        each_masked(test, stages.count, lane, [&](int stage) {
            add_specials<T, T, false>(
                stage * SK, min(stage * SK + SK, lp.sk), min(16 * MT, lp.sq - row0), lp.d, lane,
                [&](int key) { return K + key * lp.ks.s; },
                [&](int key, int r) { return pair_seen(lp, prefix, w.b, row0 + r, key); },
                [&](int r) { return out + (row0 + r) * lp.dqs.s; });
        });
    }
}

// What was cleaned from the Q and dO tiles of heads [first, first + count), to the n key rows from key0 that see it.
template <typename T, typename O, int SQ, typename Test>
__device__ __forceinline__ void dkv_specials(const ScoreParams& p, Test test, int nst, int prefix, int b, int first,
                                             int count, int key0, int n, int lane, O* outk, int64_t sk, O* outv,
                                             int64_t sv) {
    __threadfence();
    for (int h = first; h < first + count; ++h) {
        const T* Q = slice<T>(p.q, p.qs, b, h);
        const T* dO = slice<T>(p.dout, p.dos, b, h);
        each_masked(test, nst, lane, [&](int stage) {
            const int from = stage * SQ, to = min(from + SQ, p.sq), keys = min(n, p.sk - key0);
            auto see = [&](int row, int r) { return pair_seen(p, prefix, b, row, key0 + r); };
            if (outk)
                add_specials<T, O, false>(from, to, keys, p.d, lane, [&](int row) { return Q + row * p.qs.s; }, see,
                                          [&](int r) { return outk + (key0 + r) * sk; });
            if (outv)
                add_specials<T, O, true>(from, to, keys, p.d, lane, [&](int row) { return dO + row * p.dos.s; }, see,
                                         [&](int r) { return outv + (key0 + r) * sv; });
        });
    }
}

// Of the stages of queries: those in [first, last) but not in [out_first, out_last).
struct FarStages {
    int first, last, out_first, out_last;
    __device__ __forceinline__ bool takes(int st) const {
        return st >= first && st < last && !(st >= out_first && st < out_last);
    }
};

// dK and dV: key rows kept, the queries of every head of the group walked.  Four waves
// of MT 16-row tiles; Q and dO tiles double-buffered, one barrier a stage.  A kv head's sums over its
// query heads are formed here, in head order, or by score_dkv_sum where workgroups share them.
// Windows: key blocks that hold sinks are seen by all queries.  Those whose window does not reach them are dealt out in
// chunks to workgroups of their own (blockIdx >= p.far_first), whose sums score_dkv_sum adds, since the few long
// blocks would end long after all others.
// Bound as the forward kernel, with LDS read at half of its rate besides: bf16, 2 x 16 x 4096^2 all visible, 128
// columns some 615 us (four products, 890 TF/s), dQ 515 us.  Window 512 and 64 sinks, 2 x 16 / 4 heads x 4096^2,
// 128 columns: dK and dV 131 us, dQ 121 us.
template <typename T, int D, int MT, int KG, int MOD, bool VEC>
__device__ __forceinline__ void score_dkv(const ScoreParams& p) {
    using M = Mma<T>;
    using v8 = typename M::v8;
    constexpr int NW = 4, NR = NW / KG, SQ = kStageRows<T, D, KG>, BK = 16 * MT * NR;
    constexpr int NCH = SQ / 32 / KG, NDC = D / 32, NDB = D / 16, LD = D + kPad<T>;
    constexpr int PRE = kAhead<T>;
    using Fill = TileFill<T, D, SQ, NW, VEC>;
    T* const Qb0 = lds_array<T, Fill::SIZE, 0>();
    T* const Ob0 = lds_array<T, Fill::SIZE, 1>();
    T* const Qb1 = lds_array<T, Fill::SIZE, 2>();
    T* const Ob1 = lds_array<T, Fill::SIZE, 3>();
    int* const Wb0 = lds_array<int, 192, 4>();   // of the stage's queries: lse2, delta, document
    int* const Wb1 = lds_array<int, 192, 5>();
    int* const Special = lds_array<int, 3, 6>();   // met any; and the tiles of either buffer hold some

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, li = lane & 15;
    // a workgroup takes heads first .. first + count - 1 of a kv head's group; the first key blocks have most queries
    // where causal
    Work w;
    int chunk = -1;
    if (kWindow && (int)blockIdx.x >= p.far_first) {
        int id = blockIdx.x - p.far_first;
        chunk = id % p.far_chunks;
        id /= p.far_chunks;
        w.hq = id % p.far_splits;
        id /= p.far_splits;
        w.blk = id % p.far_blocks;
        id /= p.far_blocks;
        w.hk = id % p.kv_heads;
        w.b = id / p.kv_heads;
    } else {
        const unsigned grid = kWindow ? p.far_first : gridDim.x;
        w = find_work(p.k_order ? blockIdx.x : grid - 1 - blockIdx.x, p.nqb, p.batch * p.kv_heads, p.splits, p.kv_heads,
                      p.k_order);
    }
    const int count = p.group / (kWindow && chunk >= 0 ? p.far_splits : p.splits), first = w.hk * p.group + w.hq * count;
    const int kg = wave / NR, qoff = kg * 32 * NCH;   // the wave's queries of a stage
    const int kbeg = w.blk * BK, key0 = kbeg + 16 * MT * (wave % NR);
    const T* K = slice<T>(p.k, p.ks, w.b, w.hk);
    const T* V = slice<T>(p.v, p.vs, w.b, w.hk);
    const bool docs = p.q_doc != nullptr;
    const int prefix = p.prefix ? load_uniform(p.prefix + w.b) : 0;
    const bool cap = has_cap<MOD>(p);

    v8 kreg[MT][NDC], vreg[MT][NDC];
    f32x4 dk[MT][NDB], dv[MT][NDB];
    GradScale<T, D, MT> down;
    int kd[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int key = key0 + 16 * t + li;
#pragma unroll
        for (int dc = 0; dc < NDC; ++dc) {
            kreg[t][dc] = global_row<T, VEC>(K, p.ks.s, key, p.sk, 32 * dc + 8 * g, p.d);
            vreg[t][dc] = global_row<T, VEC>(V, p.vs.s, key, p.sk, 32 * dc + 8 * g, p.d);
        }
        kd[t] = docs && key < p.sk ? p.k_doc[(int64_t)w.b * p.sk + key] : -1;
#pragma unroll
        for (int j = 0; j < NDB; ++j) dk[t][j] = dv[t][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int kend = min(kbeg + BK, p.sk);
    DocRange kr = {};
    const int32_t* qrng = nullptr;
    if (docs) {
        kr = doc_range(p.k_rng + (int64_t)w.b * 2 * ((p.sk + kDocTile - 1) / kDocTile), kbeg, kend);
        qrng = p.q_rng + (int64_t)w.b * 2 * ((p.sq + kDocTile - 1) / kDocTile);
    }
    const int nst = (p.sq + SQ - 1) / SQ;
    // the stages of queries whose window reaches the keys, or of a chunk of the others
    FarStages far = {0, nst, 0, 0};
    if constexpr (kWindow) {
        const int lo = kbeg - p.q_start - (p.causal && !p.prefix ? 0 : p.window - 1), hi = kend - 1 - p.q_start + p.window - 1;
        const int first = lo <= 0 ? 0 : min(nst, lo / SQ), last = hi < 0 ? 0 : min(nst, hi / SQ + 1);
        if (chunk < 0 && (kbeg >= p.sinks || p.far_blocks)) far = {first, last, 0, 0};
        if (chunk >= 0) far = {chunk * p.far_stages, min(nst, (chunk + 1) * p.far_stages), first, last};
    }
    auto test = [&](int st, bool* part) -> bool {
        const int q0 = st * SQ, q1 = min(q0 + SQ, p.sq);
        bool v = true;
        if (q0 + SQ > p.sq) *part = true;
        if (p.causal) {
            v = p.q_start + q1 - 1 >= kbeg || kbeg < prefix;
            if (!(p.q_start + q0 >= kend - 1 || kend <= prefix)) *part = true;
        }
        if (kWindow && v)
            v = window_meets(p, p.q_start + q0, p.q_start + q1 - 1, kbeg, kend, part) && far.takes(st);
        if (docs && v) v = docs_meet(kr, doc_range(qrng, q0 / kDocTile), part);
        return v;
    };
    Stages<decltype(test)> stages(nst, lane, test);
    if constexpr (kWindow) {
        stages.count = far.last;
        stages.from = far.first;
    }
    const Fill qfill(p.qs.s, p.d, wave, lane), ofill(p.dos.s, p.d, wave, lane);
    // the next (head, stage): the stages of one head of the group after the other
    int head = 0;
    auto next = [&](int* m) -> int {
        int s = stages.next(m);
        while (s < 0 && head + 1 < count && stages.count > 0) {
            ++head;
            stages.base = -64;
            s = stages.next(m);
            if (s < 0) head = count;   // no stage for one head is none for any
        }
        return s;
    };
    const T* const Q = slice<T>(p.q, p.qs, w.b, first);
    const T* const dO = slice<T>(p.dout, p.dos, w.b, first);
    const float* const lse2 = p.lse2 + ((int64_t)w.b * p.heads + first) * p.sq;
    const int64_t to_delta = p.delta - p.lse2;
    const int32_t* const qdoc = docs ? p.q_doc + (int64_t)w.b * p.sq : nullptr;
    auto fill = [&](int hq, int st, T* q, T* o, int* words) {
        const int q0 = st * SQ;
        qfill(q, Q + hq * p.qs.h, q0, p.sq);
        ofill(o, dO + hq * p.dos.h, q0, p.sq);
        if (lane < SQ) {
            const float* const at = lse2 + (int64_t)hq * p.sq + q0;
            if (wave == 0) fill_words(words, at, p.sq - q0, lane);
            if (wave == 1) fill_words(words + 64, at + to_delta, p.sq - q0, lane);
            if (wave == 2 && docs) fill_words(words + 128, qdoc + q0, p.sq - q0, lane);
        }
    };
    // Rows past the last query arrive as zeros.  With an lse2 of 0 their weight would be e^bias, which overflows with
    // negative slopes, and times the zeros of Q and dO that is NaN; so they get that of empty rows.  By the wave whose
    // DMA it was, once that has arrived.
    auto end_rows = [&](int st, int* words) {
        if (wave == 0 && lane < SQ && st * SQ + lane >= p.sq) words[lane] = 0x7f800000;
    };
    auto active = [&](int st) -> int {
        if (key0 >= p.sk) return false;
        const int lo = p.q_start + st * SQ + qoff, hi = lo + 32 * NCH - 1;
        return st * SQ + qoff < p.sq && (!p.causal || hi >= key0 || key0 < prefix) &&
               window_active(p, lo, hi, key0, key0 + 16 * MT);
    };

    int masked = 0, masked_next = 0;
    int st = next(&masked), hq = head;
    if (tid < 3) Special[tid] = 0;
    if (st >= 0) fill(hq, st, Qb0, Ob0, Wb0);
    wait_loads();
    if (st >= 0) end_rows(st, Wb0);
    __syncthreads();
    auto special = [&](T* q, T* o) {
        const bool found = qfill.template special<false>(q);
        return ofill.template special<false>(o) || found;
    };
    if (masked && special(Qb0, Ob0)) Special[1] = 1;
    __syncthreads();
    auto step = [&](auto parity) {
        constexpr int P = decltype(parity)::value;
        T* const Qs = P ? Qb1 : Qb0;
        T* const Os = P ? Ob1 : Ob0;
        const int* const words = P ? Wb1 : Wb0;
        const float* const Ls = reinterpret_cast<const float*>(words);
        const int nx = next(&masked_next), hnx = head;
        if (nx >= 0) fill(hnx, nx, P ? Qb0 : Qb1, P ? Ob0 : Ob1, P ? Wb0 : Wb1);
        const int q0 = st * SQ;
        const int act = active(st), dirty = masked ? __builtin_amdgcn_readfirstlane(Special[1 + P]) : 0;
        const float slope = has_bias<MOD>(p) ? load_uniform(p.slopes + first + hq) * kLog2e : 0.0f;
        v8 co[PRE + 1], cq[PRE + 1];
        auto col = [&](int i, int j) {
            co[j % (PRE + 1)] = col_op<T, LD>(Os, qoff + 32 * i, 16 * j, g, li);
            cq[j % (PRE + 1)] = col_op<T, LD>(Qs, qoff + 32 * i, 16 * j, g, li);
        };
        auto preload = [&](int i) {
#pragma unroll
            for (int j = 0; j < PRE; ++j) col(i, j);
        };
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            v8 pb[MT][1], db[MT][1];
            if (act) {
                f32x4 s[MT][2], dp[MT][2];
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int b = 0; b < 2; ++b) s[t][b] = dp[t][b] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
                v8 qa[PRE + 1], oa[PRE + 1];
                auto load = [&](int n) {   // operands of query block n % 2, columns 32 (n / 2)
                    qa[n % (PRE + 1)] = row_op<T, LD>(Qs, qoff + 32 * i + 16 * (n % 2), n / 2, g, li);
                    oa[n % (PRE + 1)] = row_op<T, LD>(Os, qoff + 32 * i + 16 * (n % 2), n / 2, g, li);
                };
#pragma unroll
                for (int n = 0; n < PRE; ++n) load(n);
#pragma unroll
                for (int n = 0; n < 2 * NDC; ++n) {
                    if (n + PRE < 2 * NDC) load(n + PRE);
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        s[t][n % 2] = M::mma(qa[n % (PRE + 1)], kreg[t][n / 2], s[t][n % 2]);
                        dp[t][n % 2] = M::mma(oa[n % (PRE + 1)], vreg[t][n / 2], dp[t][n % 2]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (!dirty) preload(i);
                f32x4 ds[MT][2];   // gradients of the raw scores
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int at = qoff + 32 * i + 16 * b + 4 * g, pos = p.q_start + q0 + at;
                    const f32x4 lse2 = *reinterpret_cast<const f32x4*>(Ls + at);
                    const f32x4 delta = *reinterpret_cast<const f32x4*>(Ls + 64 + at);
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        const int key = key0 + 16 * t + li;
                        f32x4 x, y, f;
                        weigh<T, MOD>(p, cap, s[t][b], dp[t][b], lse2, delta, slope, (float)(key - pos), &x, &y, &f);
                        if (masked) {
                            if (docs) {
                                const i32x4 qd = *reinterpret_cast<const i32x4*>(words + 128 + at);
#pragma unroll
                                for (int r = 0; r < 4; ++r)
                                    if (qd[r] != kd[t] || kd[t] < 0) x[r] = y[r] = 0.0f;
                            }
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (key >= key_limit(p, prefix, pos + r) || lse2[r] == -OPS_NEG_INF) x[r] = y[r] = 0.0f;
                            if constexpr (kWindow) {
#pragma unroll
                                for (int r = 0; r < 4; ++r)
                                    if (window_hides(p, pos + r, key)) x[r] = y[r] = 0.0f;
                            }
                        }
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            pb[t][0][4 * b + r] = T(x[r]);
                            ds[t][b][r] = y[r] * f[r];
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    down.fit(t, ds[t], dk[t]);
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int r = 0; r < 4; ++r) db[t][0][4 * b + r] = T(ds[t][b][r]);
                }
            }
            if (dirty) {
                __syncthreads();
                const bool bad = tile_clean<T, LD, D, 32 * KG, 64 * NW>(Qs + 32 * i * LD, tid);
                if (tile_clean<T, LD, D, 32 * KG, 64 * NW>(Os + 32 * i * LD, tid) || bad) *Special = 1;
                __syncthreads();
                if (act) preload(i);
            }
            if (act) {
#pragma unroll
                for (int j = 0; j < NDB; ++j) {
                    if (j + PRE < NDB) col(i, j + PRE);
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        dv[t][j] = M::mma(co[j % (PRE + 1)], pb[t][0], dv[t][j]);
                        dk[t][j] = M::mma(cq[j % (PRE + 1)], db[t][0], dk[t][j]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        wait_loads();
        if (nx >= 0 && masked_next) {
            end_rows(nx, P ? Wb0 : Wb1);
            if (special(P ? Qb0 : Qb1, P ? Ob0 : Ob1)) Special[2 - P] = 1;
        }
        if (dirty && tid == 0) Special[1 + P] = 0;
        __syncthreads();
        st = nx, hq = hnx, masked = masked_next;
    };
    while (st >= 0) {
        step(std::integral_constant<int, 0>{});
        if (st < 0) break;
        step(std::integral_constant<int, 1>{});
    }
    const ScoreParams lp = late_params<ScoreParams>();
    if constexpr (down.kOn) {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const float by = down.inverse(t) * kGradInv<T>;
#pragma unroll
            for (int j = 0; j < NDB; ++j) {
                dk[t][j] *= by;
                dv[t][j] *= kGradInv<T>;
            }
        }
    }
    if constexpr (KG > 1) {
        static_assert(MT == 1 && KG == 2 && NCH == 1 && NR * NDB * 64 * 16 <= Fill::SIZE * (int)sizeof(T), "sums fit a tile");
        f32x4* const ksum = reinterpret_cast<f32x4*>(Qb0) + wave % NR * NDB * 64;
        f32x4* const vsum = reinterpret_cast<f32x4*>(Ob0) + wave % NR * NDB * 64;
        if (kg == 1) {
#pragma unroll
            for (int j = 0; j < NDB; ++j) {
                ksum[j * 64 + lane] = dk[0][j];
                vsum[j * 64 + lane] = dv[0][j];
            }
        }
        __syncthreads();
        if (kg == 1) return;
#pragma unroll
        for (int j = 0; j < NDB; ++j) {
            dk[0][j] += ksum[j * 64 + lane];
            dv[0][j] += vsum[j * 64 + lane];
        }
    }
    // to partial sums where several workgroups share the keys: those of the heads of the group, those of far queries,
    // and (the first of these sums) a block of sinks that otherwise one workgroup has
    const bool far_sums = kWindow && (chunk >= 0 || (lp.splits == 1 && w.blk < lp.far_blocks));
    if (lp.splits > 1 || far_sums) {
        const int64_t slices = (int64_t)lp.batch * lp.kv_heads, at = (int64_t)w.b * lp.kv_heads + w.hk;
        const int64_t rows = slices * lp.sk;   // of one split
        float *outk, *outv;
        if (far_sums) {
            const int64_t per = slices * lp.far_blocks * BK;
            const int sum = chunk < 0 ? 0 : 1 + chunk * lp.far_splits + w.hq;
            outk = lp.far_part + (sum * per + at * lp.far_blocks * BK) * D;
            outv = outk + (lp.far_chunks * lp.far_splits + 1) * per * D;
        } else {
            outk = lp.part + (w.hq * rows + at * lp.sk) * D;
            outv = outk + lp.splits * rows * D;
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int key = key0 + 16 * t + li;
            if (key >= lp.sk) continue;
#pragma unroll
            for (int j = 0; j < NDB; ++j) {
                *reinterpret_cast<f32x4*>(outk + (int64_t)key * D + 16 * j + 4 * g) = dk[t][j];
                *reinterpret_cast<f32x4*>(outv + (int64_t)key * D + 16 * j + 4 * g) = dv[t][j];
            }
        }
        if (*Special) dkv_specials<T, float, SQ>(lp, test, nst, prefix, w.b, first, count, key0, 16 * MT, lane, outk, D, outv, D);
        return;
    }
    T* const outk = lp.dk ? slice<T>(lp.dk, lp.dks, w.b, w.hk) : nullptr;
    T* const outv = lp.dv ? slice<T>(lp.dv, lp.dvs, w.b, w.hk) : nullptr;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int key = key0 + 16 * t + li;
        if (key >= lp.sk) continue;
#pragma unroll
        for (int j = 0; j < NDB; ++j) {
            if (outk) store4<T, VEC>(outk + key * lp.dks.s, 16 * j + 4 * g, lp.d, dk[t][j] * lp.scale);
            if (outv) store4<T, VEC>(outv + key * lp.dvs.s, 16 * j + 4 * g, lp.d, dv[t][j]);
        }
    }
    if (*Special)
        dkv_specials<T, T, SQ>(lp, test, nst, prefix, w.b, first, count, key0, 16 * MT, lane, outk, lp.dks.s, outv, lp.dvs.s);
}

// Adds up the splits of a key block's heads and, of sinks, the chunks of far queries: four columns a thread.  Without
// splits only rows of sinks come here.
template <typename T, int D, bool VEC>
__device__ __forceinline__ void score_dkv_sum(const ScoreParams& p) {
    constexpr int L = D / 4;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, row = id / L;
    const int col = id % L * 4, far_rows = kWindow ? p.far_rows : 0, n = p.splits > 1 ? p.sk : min(far_rows, p.sk);
    if (row >= (int64_t)p.batch * p.kv_heads * n) return;
    const int key = row % n, hk = row / n % p.kv_heads, b = row / n / p.kv_heads;
    const int64_t rows = (int64_t)p.batch * p.kv_heads * p.sk;
    f32x4 k = {0.0f, 0.0f, 0.0f, 0.0f}, v = k;
    if (p.splits > 1) {
        const float* at = p.part + row * D + col;
#pragma unroll 4
        for (int s = 0; s < p.splits; ++s) {
            k += *reinterpret_cast<const f32x4*>(at + s * rows * D);
            v += *reinterpret_cast<const f32x4*>(at + (p.splits + s) * rows * D);
        }
    }
    if (kWindow && key < far_rows) {
        const int64_t per = (int64_t)p.batch * p.kv_heads * far_rows;
        const float* at = p.far_part + ((int64_t)(b * p.kv_heads + hk) * far_rows + key) * D + col;
        const int all = p.far_chunks * p.far_splits + 1;
#pragma unroll 8
        for (int s = p.splits > 1 ? 1 : 0; s < all; ++s) {   // (the first is there without splits only)
            k += *reinterpret_cast<const f32x4*>(at + s * per * D);
            v += *reinterpret_cast<const f32x4*>(at + (all + s) * per * D);
        }
    }
    if (p.dk) store4<T, VEC>(slice<T>(p.dk, p.dks, b, hk) + key * p.dks.s, col, p.d, k * p.scale);
    if (p.dv) store4<T, VEC>(slice<T>(p.dv, p.dvs, b, hk) + key * p.dvs.s, col, p.d, v);

}

// ---------------------------------------------------------------------------
// Range of the ids of every kDocTile tokens, a wave a tile: (min, max) of those that are not padding,
// the min with all bits flipped where there is padding (none but padding: min 2^31 - 1, max -1).
extern "C" __global__ __launch_bounds__(256) void fa_score_doc_ranges(ScoreParams p) {
    const int qt = (p.sq + kDocTile - 1) / kDocTile, kt = (p.sk + kDocTile - 1) / kDocTile;
    const int tile = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (tile >= p.batch * (qt + kt)) return;
    const int b = tile / (qt + kt), t = tile % (qt + kt);
    const bool isq = t < qt;
    const int at = (isq ? t : t - qt) * kDocTile + lane, n = isq ? p.sq : p.sk;
    const int32_t* ids = (isq ? p.q_doc : p.k_doc) + (int64_t)b * n;
    const int id = at < n ? ids[at] : 0;
    const bool padding = __builtin_amdgcn_ballot_w64(id < 0) != 0;
    int lo = at < n && id >= 0 ? id : 0x7fffffff, hi = at < n ? max(id, -1) : -1;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
        lo = min(lo, __shfl_xor(lo, s));
        hi = max(hi, __shfl_xor(hi, s));
    }
    if (lane == 0) {
        int32_t* rng = isq ? p.q_rng + 2 * ((int64_t)b * qt + t) : p.k_rng + 2 * ((int64_t)b * kt + t - qt);
        rng[0] = padding ? ~lo : lo;
        rng[1] = hi;
    }
}

// Orders the blocks of all batches by the number of tiles of the other side that they meet, the most first:
// workgroup 0 the query blocks, 1 the key blocks.  Documents make blocks differ in length by far more than causal
// bounds do, and a long one that starts late ends alone (bf16, 2 x 4096 tokens, 16 heads of 128 columns, documents
// up to 2550 tokens, forward 155 -> 137 us; in
// 16384 tokens of documents up to 3400: 237 -> 222).
extern "C" __global__ __launch_bounds__(1024) void fa_score_doc_order(ScoreParams p) {
    __shared__ int2 walked[kOrderTiles];
    __shared__ int2 kept[kOrderBlocks];
    __shared__ int padded[kOrderBlocks];
    __shared__ int key[kOrderBlocks];
    const bool isq = blockIdx.x == 0;
    if (!(isq ? p.q_order : p.k_order)) return;
    const int n = isq ? p.sq : p.sk, rows = isq ? p.q_rows : p.k_rows;
    const int nt = ((isq ? p.sq : p.sk) + kDocTile - 1) / kDocTile, wt = ((isq ? p.sk : p.sq) + kDocTile - 1) / kDocTile;
    const int nblk = (n + rows - 1) / rows, items = p.batch * nblk;
    const int32_t *krng = isq ? p.q_rng : p.k_rng, *wrng = isq ? p.k_rng : p.q_rng;
    const int tid = threadIdx.x, lane = tid & 63;
    for (int i = tid; i < p.batch * wt; i += 1024) walked[i] = make_int2(wrng[2 * i], wrng[2 * i + 1]);
    if (tid < items) {
        const int r0 = tid % nblk * rows;
        const DocRange x = doc_range(krng + 2 * (tid / nblk * nt), r0, min(r0 + rows, n));
        kept[tid] = make_int2(x.lo, x.hi);
        padded[tid] = x.padding;
    }
    __syncthreads();
    for (int i = tid >> 6; i < items; i += 16) {
        const int b = i / nblk, r0 = i % nblk * rows, r1 = min(r0 + rows, n);
        const int prefix = p.prefix ? load_uniform(p.prefix + b) : 0;
        const DocRange x = {kept[i].x, kept[i].y, padded[i] != 0};
        int count = 0;
#pragma unroll 4
        for (int t0 = 0; t0 < wt; t0 += 64) {
            const int t = t0 + lane, w0 = t * kDocTile;
            const int2 y = walked[b * wt + min(t, wt - 1)];
            bool part;
            bool v = t < wt && docs_meet(x, DocRange{y.x < 0 ? ~y.x : y.x, y.y, y.x < 0}, &part);
            if (p.causal) {
                const int last = isq ? r1 : min(w0 + kDocTile, p.sq), first = isq ? w0 : r0;   // query, key
                v = v && (first <= p.q_start + last - 1 || first < prefix);
            }
            count += __builtin_popcountll(__builtin_amdgcn_ballot_w64(v));
        }
        if (lane == 0) key[i] = (count << 10) + i;   // kOrderBlocks = 2^10: no two alike
    }
    __syncthreads();
    if (tid < items) {
        int rank = 0;
        const int mine = key[tid];
#pragma unroll 8
        for (int i = 0; i < items; ++i) rank += key[i] > mine;
        (isq ? p.q_order : p.k_order)[rank] = tid;
    }
}

#define PASTE_(a, b, c, d) a##b##c##d
#define PASTE(a, b, c, d) PASTE_(a, b, c, d)
#define KERNEL(F, D, MT, KG, MOD, VEC, TAG, WAVES)                                                    \
    extern "C" __global__ __launch_bounds__(256, WAVES) void PASTE(fa_score_##F##_, OPS_NAME, _d##D##_t##MT, TAG)( \
        ScoreParams p) {                                                                              \
        score_##F<OPS_T, D, MT, KG, MOD, VEC>(p);                                                     \
    }
#define SUM(D, VEC, TAG)                                                                                         \
    extern "C" __global__ __launch_bounds__(256) void PASTE(fa_score_dkv_sum_, OPS_NAME, _d##D, TAG)(ScoreParams p) { \
        score_dkv_sum<OPS_T, D, VEC>(p);                                                                        \
    }
SUM(64, true, )
SUM(128, true, )
SUM(256, true, )
SUM(64, false, s)
SUM(128, false, s)
SUM(256, false, s)
// plain scores, capped (c), with a bias (b) or both (cb); any alignment (s); two groups of waves on a stage (k)
// windows: plain scores, or looked up (m)
#ifdef OPS_WINDOW
#define KERNELS(F, D, MT, WAVES)                      \
    KERNEL(F, D, MT, 1, 0, true, , WAVES)             \
    KERNEL(F, D, MT, 1, kAny, true, m, WAVES)
#define GROUPS(F, D, WAVES)                           \
    KERNEL(F, D, 1, 2, 0, true, k, WAVES)             \
    KERNEL(F, D, 1, 2, kAny, true, km, WAVES)
#else
#define KERNELS(F, D, MT, WAVES)                      \
    KERNEL(F, D, MT, 1, 0, true, , WAVES)             \
    KERNEL(F, D, MT, 1, kCap, true, c, WAVES)         \
    KERNEL(F, D, MT, 1, kBias, true, b, WAVES)        \
    KERNEL(F, D, MT, 1, kCap | kBias, true, cb, WAVES)
#define GROUPS(F, D, WAVES)                           \
    KERNEL(F, D, 1, 2, 0, true, k, WAVES)             \
    KERNEL(F, D, 1, 2, kCap, true, kc, WAVES)         \
    KERNEL(F, D, 1, 2, kBias, true, kb, WAVES)        \
    KERNEL(F, D, 1, 2, kCap | kBias, true, kcb, WAVES)
#endif
#define SLOW(F, W64, W128, W256)                 \
    KERNEL(F, 64, 1, 1, kAny, false, s, W64)     \
    KERNEL(F, 128, 1, 1, kAny, false, s, W128)   \
    KERNEL(F, 256, 1, 1, kAny, false, s, W256)
#define ALL(F, W64, W128, W256)  \
    KERNELS(F, 64, 1, W64)       \
    KERNELS(F, 128, 1, W128)     \
    KERNELS(F, 256, 1, W256)     \
    GROUPS(F, 64, W64)           \
    GROUPS(F, 128, W128)
SLOW(forward, 2, 1, 1)
SLOW(dq, 2, 1, 1)
SLOW(dkv, 2, 1, 1)
#ifdef OPS_16BIT
ALL(forward, 2, 2, 2)
ALL(dq, 2, 2, 2)
ALL(dkv, 2, 2, 1)
// two tiles of 64 columns: three waves a SIMD, except where a cap would spill (bf16, 16 heads x 4 x 4096^2, causal,
// plain 200 -> 172 us, bias 282 -> 248, capped 287 -> 318)
#ifdef OPS_WINDOW
KERNELS(forward, 64, 2, 2)
#else
KERNEL(forward, 64, 2, 1, 0, true, , 3)
KERNEL(forward, 64, 2, 1, kCap, true, c, 2)
KERNEL(forward, 64, 2, 1, kBias, true, b, 3)
KERNEL(forward, 64, 2, 1, kCap | kBias, true, cb, 2)
#endif
KERNELS(forward, 128, 2, 2)
KERNELS(dq, 64, 2, 2)
KERNELS(dkv, 64, 2, 2)
#else
ALL(forward, 2, 2, 1)
ALL(dq, 2, 2, 1)
ALL(dkv, 2, 2, 1)
#endif
