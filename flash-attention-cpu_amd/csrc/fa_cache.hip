// fa_cache.hip -- gfx950 kernels for query rows over a cache: drafted trees
// over a key / value cache (fa_tree_attention) and short query blocks of score
// attention (fa_score_forward).
//
// The rows of a (sequence, kv head) are its tokens times the query heads of the group, so K and V are read once for
// all of them.  The keys of all sequences are cut into runs of one length, one a workgroup, so that sequences of
// different lengths keep all of the GPU busy; a sequence of more than one run leaves partial sums that fa_rows_merge
// joins.
//   stream: up to 16 rows, up to 64 where a row of K has 128 bytes.  Bound by memory: every wave walks 32-key blocks
//           of its own through LDS that only it uses, two slots of K and V, one filled by DMA while the
//           other is used; no barrier until the waves' sums are joined at the end.  (bf16, 8 sequences of
//           32768 keys, 1 token of 32 / 8 heads of 128 columns: 208 us, 5.2 TB/s; one such sequence 31 us.)
//   shared: more rows.  Eight waves of one or two 16-row tiles share the stages of a ring, two of which are on
//           their way while one is used, so that K and V cross the L2 once for up to 256 rows.
//           Bound by vector and matrix instructions in turn and by start-up where runs are short.  (bf16, 8
//           sequences of up to 16384 keys, 64 tokens of 32 / 8 heads of 128 columns: 171 us with the merge, 592 TF/s;
//           107 without the products, 132 without the loads after the first stages.)
// Tiles in LDS have no padding, so that DMA instructions move 1 KiB of whole rows; row r keeps
// 16-byte chunk x at position x ^ turn(r), which spreads row reads and transposed
// reads over the banks.
//
// Built once a type: OPS_T the element type, OPS_NAME its name in the kernels'.

#include "fa_rows.h"

// Operands and geometry of an unpadded, swizzled tile.
template <typename T, int D>
struct Swizzled {
    using v8 = typename Mma<T>::v8;
    static constexpr int E = 16 / (int)sizeof(T);   // elements of a chunk
    static constexpr int CPR = D / E;               // chunks of a row
    static constexpr int CM = CPR < 16 ? CPR : 16;
    static constexpr int RPR = 64 / CPR > 0 ? 64 / CPR : 1;   // rows of a 1 KiB run
    static_assert(CPR <= 64, "a run holds whole rows");
    // What row `row` adds to its chunk numbers: the same for rows 16 apart.  16-bit types: a transposed read takes
    // two neighbouring chunks of eight rows in a row at a time, so these get values that differ above the lowest bit;
    // a row read takes a chunk of rows 0 - 3 and 12 - 15 and the next chunk of rows 4 - 11, so the values 2x and 2x +
    // 1 go to rows r and 15 - r: no bank conflicts are counted (with r itself the transposed reads reach 285 bytes/ns
    // a CU instead of 470, with 2r | r / 8 the row reads 290 instead of 510).
    static __device__ __forceinline__ int turn(int row) {
        if constexpr (sizeof(T) == 4) {
            return row % CM;
        } else if constexpr (CPR == 8) {   // two rows of 128 bytes stand where one of 256 does
            const int r = row >> 1 & 7;
            return r < 4 ? 2 * r : 15 - 2 * r;
        } else {
            const int r = row & 15;
            return r < 8 ? 2 * r : 31 - 2 * r;
        }
    }
    static __device__ __forceinline__ int at(int row, int col) {   // col: a multiple of E or inside its chunk
        return row * D + (((col / E) ^ turn(row)) * E) + col % E;
    }
    // An operand's chunk numbers are those of its first column block, exclusive-or the block's own (a
    // multiple of what the lanes add), so its place is base ^ block; row0 (a multiple of 16) only adds whole rows.
    static __device__ __forceinline__ v8 row_op(const T* tile, int row0, int dc, int g, int li) {
        const int base = at(li, 8 * g);
        const T* const t = tile + row0 * D;
        if constexpr (sizeof(T) == 2) {
            return *reinterpret_cast<const v8*>(t + (base ^ (32 * dc)));
        } else {
            const f32x4 a = *reinterpret_cast<const f32x4*>(t + (base ^ (32 * dc)));
            const f32x4 b = *reinterpret_cast<const f32x4*>(t + (base ^ (32 * dc + 4)));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    static __device__ __forceinline__ v8 col_op(const T* tile, int row0, int col0, int g, int li) {
        const T* const t = tile + row0 * D;
        if constexpr (sizeof(T) == 2) {
            typedef __attribute__((address_space(3))) s16x4* lds4;
            const int place = at(4 * g + (li >> 2), 4 * (li & 3)) ^ col0;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4) const_cast<T*>(t + place));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4) const_cast<T*>(t + 16 * D + place));
            return __builtin_bit_cast(v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            v8 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int place = at(4 * g + e, li) ^ col0;
                v[e] = t[place];
                v[4 + e] = t[16 * D + place];
            }
            return v;
        }
    }
    // tile_clean for this layout: chunks may be visited in any order
    template <int ROWS, int NT>
    static __device__ __forceinline__ bool clean(T* tile, int tid) {
        return tile_clean<T, D, D, ROWS, NT>(tile, tid);
    }
};

// Rows of one sequence's K or V and their way into LDS, ROWS at a time.
template <typename T, int D, int ROWS, int NW>
struct RowSource {
    using S = Swizzled<T, D>;
    static constexpr int RUNS = ROWS / S::RPR, NI = RUNS / NW;
    static_assert(RUNS % NW == 0 && 16 % S::RPR == 0, "whole runs a wave, in 16-row groups");
    const T* base;
    int64_t seq, batch;
    int voff[NI];
    __device__ __forceinline__ RowSource(const T* b, int64_t seq_, int64_t batch_, int d, int wave, int lane)
        : base(b), seq(seq_), batch(batch_) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int row = (i * NW + wave) * S::RPR + lane / S::CPR;
            const int col = ((lane % S::CPR) ^ S::turn(row)) * S::E;
            voff[i] = col < d ? (int)(row * seq + col) * (int)sizeof(T) : 0x7ffffff0;
        }
    }
    // DMA of rows [k0, k0 + ROWS), zeros at and past `end` and where a page is bad, in pages of 16 rows or
    // more; pg: the pages of its 16-row groups, or of row k0 alone where a page holds all.
    static constexpr int GROUPS = ROWS / 16;
    __device__ __forceinline__ void fill(T* dst, int k0, int end, const int (&pg)[GROUPS], const CachePages& c,
                                         int wave) const {
        constexpr int kStep = NW * S::RPR;   // rows of the waves' i-th runs
        if (kStep > 16 && (!c.table || c.page_mask >= ROWS - 1)) {
            const int n = pg[0] < 0 ? 0 : max(0, min(ROWS, end - k0));
            const T* src = n == 0 ? base : c.table ? base + (pg[0] * batch + (k0 & c.page_mask) * seq) : base + k0 * seq;
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<T*>(src), (short)0, (int)(n * seq) * (int)sizeof(T), 0x00020000);
#pragma unroll
            for (int i = 0; i < NI; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    rs, (__attribute__((address_space(3))) void*)(dst + (i * NW + wave) * 64 * S::E), 16, voff[i], 0, 0, 0);
            return;
        }
        // A 16-row group lies in one page; its rows are addressed as from row k0 on.
        __amdgpu_buffer_rsrc_t rs;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int run = i * NW + wave;
            if (i * kStep % 16 == 0 || kStep > 16) {
                const int grp = kStep > 16 ? run * S::RPR / 16 : i * kStep / 16, row = k0 + 16 * grp;
                int page = pg[i * kStep / 16];
#pragma unroll
                for (int e = 1; e < kStep / 16; ++e) page = wave * S::RPR / 16 == e ? pg[i * kStep / 16 + e] : page;
                const int n = page < 0 ? 0 : max(0, min(16, end - row));
                const T* src = n == 0 ? base : base + (page * batch + ((c.table ? row & c.page_mask : row) - 16 * grp) * seq);
                rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(src), (short)0,
                                                       n == 0 ? 0 : (int)((16 * grp + n) * seq) * (int)sizeof(T), 0x00020000);
            }
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rs, (__attribute__((address_space(3))) void*)(dst + run * 64 * S::E), 16, voff[i], 0, 0, 0);
        }
    }
    // The pages of rows [k0, k0 + ROWS) before `end`; returns whether one is bad.
    static __device__ __forceinline__ int look_up(const CachePages& c, int k0, int end, int (&pg)[GROUPS]) {
        int bad = 0;
        const bool whole = !c.table || c.page_mask >= ROWS - 1;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const int row = k0 + 16 * i;
            if (i > 0 && whole) {
                pg[i] = pg[0];
            } else {
                pg[i] = row < end ? c.page(row) : -1;
            }
            bad = bad || (pg[i] < 0 && row < end);
        }
        return bad;
    }
    // the same element by element: any alignment, any page size
    __device__ __forceinline__ void fill_slow(T* dst, int k0, int end, const CachePages& c, int d, int tid) const {
#pragma unroll 1
        for (int pos = tid; pos < ROWS * (D / 8); pos += 64 * NW) {
            const int r = pos / (D / 8), col = 8 * (pos % (D / 8));
            const int64_t at = c.at(k0 + r, end, seq, batch);
            const typename Mma<T>::v8 x = global_row<T, false>(base + (at < 0 ? 0 : at), 0, 0, at >= 0, col, d);
            if constexpr (sizeof(T) == 2) {
                *reinterpret_cast<typename Mma<T>::v8*>(dst + S::at(r, col)) = x;
            } else {
                *reinterpret_cast<f32x4*>(dst + S::at(r, col)) = __builtin_shufflevector(x, x, 0, 1, 2, 3);
                *reinterpret_cast<f32x4*>(dst + S::at(r, col + 4)) = __builtin_shufflevector(x, x, 4, 5, 6, 7);
            }
        }
    }
    // Whether a row of [k0, k0 + ROWS) before `end` lies in a bad page, a lane a row: what look_up returns, for any page
    // size.  Every wave looks for itself, so all come to the same answer.
    static __device__ __forceinline__ int bad_rows(const CachePages& c, int k0, int end, int lane) {
        static_assert(ROWS <= 64, "a lane a row");
        if (!c.table) return 0;
        return __builtin_amdgcn_ballot_w64(lane < ROWS && k0 + lane < end && c.at(k0 + lane, end, 0, 0) < 0) != 0;
    }
};

// MT 16-row tiles of a wave: their queries, and the running softmax over KB 16-key blocks at a time.
template <typename T, int D, int MT, int KB, int MOD, bool VEC>
struct RowTiles {
    using M = Mma<T>;
    using S = Swizzled<T, D>;
    using v8 = typename M::v8;
    static constexpr int NDC = D / 32, NDB = D / 16, NCH = KB / 2;
    v8 q[MT][NDC], pb[MT][NCH];
    f32x4 o[MT][NDB], s[MT][KB];
    float m[MT], ref[MT], l[MT];   // l: the lane's share of the row's sum
    float slope[MT];
    int token[MT], pos[MT], qd[MT];
    uint64_t word[MT];             // the token's first mask word
    int g, li;
    float c;

    __device__ __forceinline__ void init(const RowsParams& p, const RowsWork& w, int rfirst, int lane) {
        g = lane >> 4, li = lane & 15;
        c = MOD != 0 ? 1.0f : p.scale_log2e;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int r = rfirst + 16 * t + li;
            const bool real = r < w.nrows;
            token[t] = real ? r / p.group : 0;
            const int h = w.hk * p.group + (real ? r % p.group : 0);
            const T* from = reinterpret_cast<const T*>(p.q) + w.b * p.qs.b + h * p.qs.h;
#pragma unroll
            for (int dc = 0; dc < NDC; ++dc)
                q[t][dc] = global_row<T, VEC>(from, p.qs.s, token[t], real ? p.n : 0, 32 * dc + 8 * g, p.d);
            pos[t] = !w.tree ? p.q_start + token[t] : p.pos ? p.pos[w.b * p.n + token[t]] : w.len + token[t];
            qd[t] = w.docs ? p.q_doc[(int64_t)w.b * p.n + token[t]] : 0;
            slope[t] = has_bias<MOD>(p) ? p.slopes[h] * kLog2e : 0.0f;
            word[t] = 0;
            if (w.tree)
                word[t] = p.mask ? p.mask[((p.mask_shared ? 0 : (int64_t)w.b * p.n) + token[t]) * p.mask_words]
                                 : token[t] < 63 ? (2ull << token[t]) - 1 : ~0ull;
#pragma unroll
            for (int j = 0; j < NDB; ++j) o[t][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
            m[t] = OPS_NEG_INF;
            l[t] = ref[t] = 0.0f;
        }
    }
    // Scores of KB blocks of keys from k0, relative to the references (modified: log2 units, and what 16-bit weights
    // are taken larger by); hidden ones -inf.
    static constexpr float kUp = MOD != 0 ? kProbLog2<T> : 0.0f;
    __device__ __forceinline__ void scores(const RowsParams& p, const RowsWork& w, const T* Ks, int k0, bool masked,
                                           bool badpage) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const float x = MOD != 0 ? 0.0f : -ref[t];
                s[t][b] = (f32x4){x, x, x, x};
            }
        constexpr int PRE = sizeof(T) == 2 ? 1 : 0;   // 32-column steps read ahead
        v8 k[PRE + 1][KB];
        auto load = [&](int dc) {
#pragma unroll
            for (int b = 0; b < KB; ++b) k[dc % (PRE + 1)][b] = S::row_op(Ks, 16 * b, dc, g, li);
        };
        if (PRE) load(0);
#pragma unroll
        for (int dc = 0; dc < NDC; ++dc) {
            if (dc + PRE < NDC) load(dc + PRE);
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int t = 0; t < MT; ++t) s[t][b] = M::mma(k[dc % (PRE + 1)][b], q[t][dc], s[t][b]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (MOD != 0) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const float dist = (float)(pos[t] - k0 - 4 * g);
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    if (has_cap<MOD>(p)) {
                        s[t][b] = capped_over<T, MOD>(s[t][b], p.cap_in, p.cap_log2e, ref[t] - kUp);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][b][r] = __builtin_fmaf(s[t][b][r], p.scale_log2e, kUp - ref[t]);
                    }
                    if (has_bias<MOD>(p)) {
                        f32x4 x;
#pragma unroll
                        for (int r = 0; r < 4; ++r) x[r] = dist - (float)(16 * b + r);
                        if (masked && w.tree) {
                            // drafted keys stand where the program says
                            const RowsParams lp = late_params<RowsParams>();
                            const int bit = k0 + 16 * b + 4 * g - w.len;
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (lp.pos && bit + r >= 0)
                                    x[r] = (float)(pos[t] - lp.pos[w.b * lp.n + min(bit + r, lp.n - 1)]);
                        }
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][b][r] = __builtin_fmaf(-slope[t], fabsf(x[r]), s[t][b][r]);
                    }
                }
            }
        }
        if (masked) {
            // keys k0 .. k0 + 16 KB - 1 as bits
            const RowsParams lp = late_params<RowsParams>();
            const uint64_t there = keys_there(lp, w, k0, badpage);
            uint64_t see[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) see[t] = there & seen_bits(lp, w, t, k0);
            if constexpr (kWindow) {
#pragma unroll
                for (int t = 0; t < MT; ++t)
                    see[t] &= window_bits<16 * KB>(lp, w, pos[t], k0, [&](int b, int r) { return 16 * b + 4 * g + r; });
            }
            if (w.docs) {
#pragma unroll
                for (int b = 0; b < KB; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int x = 16 * b + 4 * g + r;
                        const int kd = lp.k_doc[(int64_t)w.b * lp.sk + min(k0 + x, lp.sk - 1)];
#pragma unroll
                        for (int t = 0; t < MT; ++t)
                            if (kd != qd[t]) see[t] &= ~(1ull << x);
                    }
            }
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    const unsigned bits = (unsigned)(see[t] >> (16 * b + 4 * g));
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (!(bits & (1u << r))) s[t][b][r] = OPS_NEG_INF;
                }
        }
    }
    // Bits of the keys that exist: before the run's end, in good pages (one lane a key).
    __device__ __forceinline__ uint64_t keys_there(const RowsParams& p, const RowsWork& w, int k0, int badpage) const {
        const int lane = 16 * g + li, key = k0 + lane;
        const int n = kWindow ? max(w.kend - k0, 0) : w.kend - k0;   // (windows: a block may start past the end)
        if (!badpage) return n >= 64 ? ~0ull : (1ull << n) - 1;
        const CachePages pages = rows_pages(p, w.b);
        return __builtin_amdgcn_ballot_w64(key < w.kend && pages.at(key, w.kend, 0, 0) >= 0);
    }
    // Bits of the keys that the lane's row of tile t sees, as far as causal, prefix and tree tell.
    __device__ __forceinline__ uint64_t seen_bits(const RowsParams& p, const RowsWork& w, int t, int k0) const {
        if (!w.tree) {
            const int n = (w.docs && qd[t] < 0 ? 0 : p.causal ? max(p.q_start + token[t] + 1, w.prefix) : 0x7fffffff) - k0;
            return n >= 64 ? ~0ull : (1ull << max(n, 0)) - 1;
        }
        const int rel = k0 - w.len;   // the first key's number among the drafted ones
        if (rel <= -64) return ~0ull;
        if (rel < 0) return (mask_word(p, w, t, 0) << -rel) | ((1ull << -rel) - 1);
        const int i = rel >> 6, sh = rel & 63;
        const uint64_t lo = mask_word(p, w, t, i) >> sh;
        return sh == 0 ? lo : lo | (mask_word(p, w, t, i + 1) << (64 - sh));
    }
    __device__ __forceinline__ uint64_t mask_word(const RowsParams& p, const RowsWork& w, int t, int i) const {
        if (i == 0) return word[t];
        if (i >= p.mask_words) return 0;
        if (p.mask) return p.mask[((p.mask_shared ? 0 : (int64_t)w.b * p.n) + token[t]) * p.mask_words + i];
        const int n = token[t] + 1 - 64 * i;   // a chain
        return n >= 64 ? ~0ull : (1ull << max(n, 0)) - 1;
    }
    // the reference of a row moves only when a score passes it by more than kLazy, or at its first key
    __device__ __forceinline__ void softmax() {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            float mt = s[t][0][0];
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) mt = __builtin_elementwise_maximum(mt, s[t][b][r]);
            mt -= kUp;
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
            float sum = 0.0f;
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float x = ops_exp2(MOD != 0 ? s[t][b][r] : __builtin_fmaf(s[t][b][r], c, kProbLog2<T>));
                    pb[t][b / 2][4 * (b & 1) + r] = T(x);
                    sum += x;
                }
            l[t] += sum;
        }
    }
    __device__ __forceinline__ void values(const T* Vs) {
        constexpr int PRE = sizeof(T) == 2 ? 3 : 0;
        v8 a[PRE + 1];
        auto load = [&](int n) { a[n % (PRE + 1)] = S::col_op(Vs, 32 * (n / NDB), 16 * (n % NDB), g, li); };
#pragma unroll
        for (int n = 0; n < PRE; ++n) load(n);
#pragma unroll
        for (int n = 0; n < NCH * NDB; ++n) {
            if (n + PRE < NCH * NDB) load(n + PRE);
#pragma unroll
            for (int t = 0; t < MT; ++t) o[t][n % NDB] = M::mma(a[n % (PRE + 1)], pb[t][n / NDB], o[t][n % NDB]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // maxima in log2 units and whole row sums, before partial sums meet
    __device__ __forceinline__ void close() {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            m[t] *= c;
            l[t] = row4_sum(l[t]);
        }
    }
    // Partial sums, or the rows themselves where the sequence is one run.  specials: V held
    // infinities or NaN in a masked block.
    __device__ __forceinline__ void store(const RowsWork& w, const T* V, int rfirst, int tile0, int lane,
                                          bool specials) {
        const RowsParams p = late_params<RowsParams>();
        const CachePages pages = rows_pages(p, w.b);
        const int mine = min(16 * MT, w.nrows - rfirst);
        auto row_at = [&](int key) -> const T* {
            if (w.out(key)) return nullptr;
            const int64_t at = pages.at(key, w.kend, p.vs.s, p.vs.b);
            return at < 0 ? nullptr : V + at;
        };
        auto row_sees = [&](int key, int r) { return rows_see(p, w, (rfirst + r) / p.group, key); };
        if (w.runs > 1) {
            const int64_t part = ((int64_t)w.run * p.kv_heads + w.hk) * p.nrb + w.rb;
            const int rows = p.block_rows;
            float* const po = p.part_o + (part * rows + 16 * tile0) * D;
            float* const pm = p.part_ml + part * 2 * rows + 16 * tile0;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
#pragma unroll
                for (int j = 0; j < NDB; ++j)
                    *reinterpret_cast<f32x4*>(po + (16 * t + li) * D + 16 * j + 4 * g) = o[t][j];
                if (g == 0) {
                    pm[16 * t + li] = m[t];
                    pm[rows + 16 * t + li] = l[t];
                }
            }
            if (specials) {
                __threadfence();
                add_specials<T, float, true>(w.kbeg, w.kend, mine, p.d, lane, row_at, row_sees,
                                             [&](int r) { return po + r * D; });
            }
            return;
        }
        auto out_row = [&](int r) {
            const int h = w.hk * p.group + (rfirst + r) % p.group;
            return reinterpret_cast<T*>(p.out) + w.b * p.os.b + h * p.os.h + (rfirst + r) / p.group * p.os.s;
        };
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int r = rfirst + 16 * t + li;
            if (r >= w.nrows) continue;
            T* const out = out_row(16 * t + li);
            const float inv = l[t] == 0.0f ? 0.0f : 1.0f / l[t];
#pragma unroll
            for (int j = 0; j < NDB; ++j) store4<T, VEC>(out, 16 * j + 4 * g, p.d, o[t][j] * inv);
            if (p.lse && g == 0)
                p.lse[((int64_t)w.b * p.heads + w.hk * p.group + r % p.group) * p.n + token[t]] =
                    l[t] == 0.0f ? OPS_NEG_INF : (m[t] + __builtin_log2f(l[t]) - kProbLog2<T>) * kLn2;
        }
        if (specials) {
            __threadfence();
            add_specials<T, T, true>(w.kbeg, w.kend, mine, p.d, lane, row_at, row_sees, out_row);
        }
    }
};

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    constexpr int n = N > 63 ? 63 : N;
    __builtin_amdgcn_s_waitcnt(0x0f70 | (n & 15) | (n >> 4 << 14));
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

// ---------------------------------------------------------------------------
// Up to 16 MT rows, a wave 32-key blocks of its own.
// ---------------------------------------------------------------------------
template <typename T, int D, int MT, int MOD, bool VEC>
__device__ __forceinline__ void rows_stream(const RowsParams& p) {
    constexpr int NW = kStreamWaves<D * (int)sizeof(T)>, SK = 32, TILE = SK * D;
    using R = RowTiles<T, D, MT, 2, MOD, VEC>;
    using Src = RowSource<T, D, SK, 1>;
    constexpr int RUNS = Src::RUNS, NDB = R::NDB;
    T* const K0 = lds_array<T, NW * TILE, 0>();
    T* const V0 = lds_array<T, NW * TILE, 1>();
    T* const K1 = lds_array<T, NW * TILE, 2>();
    T* const V1 = lds_array<T, NW * TILE, 3>();
    __shared__ float Ml[NW][MT][2][16];
    __shared__ int any_special[NW];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    RowsWork w;
    if (!rows_work(p, 16 * MT, lane, &w)) return;
    const CachePages pages = rows_pages(p, w.b);
    const T* const K = reinterpret_cast<const T*>(p.k) + w.hk * p.ks.h + (p.table ? 0 : w.b * p.ks.b);
    const T* const V = reinterpret_cast<const T*>(p.v) + w.hk * p.vs.h + (p.table ? 0 : w.b * p.vs.b);
    const Src ksrc(K, p.ks.s, p.ks.b, p.d, 0, lane), vsrc(V, p.vs.s, p.vs.b, p.d, 0, lane);
    const int k_first = SK * wave;   // of the walked keys
    const int nblk = k_first < w.kwalk() ? (w.kwalk() - k_first + SK * NW - 1) / (SK * NW) : 0;
    static_assert(VEC, "DMA only");

    bool special = false;
    R x;
    // pages of the block to fill next are looked up a block ahead
    int page[2];
    int bad0, bad1, bad2;
    auto look_up = [&](int blk) {
        const int k0 = w.key(k_first + blk * SK * NW);
        return Src::look_up(pages, k0, blk < nblk ? w.kend : k0, page);
    };
    auto fill = [&](const Src& src, T* dst, int blk) {
        const int k0 = w.key(k_first + blk * SK * NW);
        src.fill(dst + wave * TILE, k0, blk < nblk ? w.kend : k0, page, pages, 0);
    };
    bad0 = look_up(0);
    if (nblk > 0) {
        fill(ksrc, K0, 0);
        fill(vsrc, V0, 0);
    }
    bad1 = look_up(1);
    x.init(p, w, w.rfirst, lane);
    if (nblk > 0) {
        // Q's loads are through before more DMA starts: only DMA is counted from here
        wait_vmcnt<0>();
        fill(ksrc, K1, 1);
        fill(vsrc, V1, 1);
    }
    bad2 = look_up(2);
    auto block = [&](int i, T* kb, T* vb) {
        T* const Ks = kb + wave * TILE;
        T* const Vs = vb + wave * TILE;
        const int k0 = w.key(k_first + i * SK * NW);
        const int bad = bad0;
        bad0 = bad1;
        bad1 = bad2;
        wait_vmcnt<3 * RUNS>();
        const int masked = bad || rows_masked(p, w, k0, SK);
        x.scores(p, w, Ks, k0, masked, bad);
        reread();
        fill(ksrc, kb, i + 2);
        x.softmax();
        wait_vmcnt<3 * RUNS>();
        if (masked) {
            special = Swizzled<T, D>::template clean<SK, 64>(Vs, lane) || special;
            reread();
        }
        x.values(Vs);
        reread();
        fill(vsrc, vb, i + 2);
        bad2 = look_up(i + 3);
    };
    for (int i = 0; i < nblk; i += 2) {
        block(i, K0, V0);
        if (i + 1 < nblk) block(i + 1, K1, V1);
    }
    x.close();
    const bool any = __builtin_amdgcn_ballot_w64(special) != 0;
    if (lane == 0) any_special[wave] = any;
    if constexpr (NW > 1) {
        // Join the waves' sums: the upper half leaves its own in LDS, the lower half adds them, and again.
        // Each slot array is one wave's or more; the DMA into it has landed.
        constexpr int SLOT = MT * NDB * 64;
        static_assert(SLOT * 16 <= NW * TILE * (int)sizeof(T), "a wave's sums fit an array");
        wait_vmcnt<0>();
#pragma unroll
        for (int half = NW / 2; half >= 1; half /= 2) {
            __syncthreads();
            auto slot = [&](int i) { return reinterpret_cast<f32x4*>(i == 0 ? K0 : V0); };
            if (wave >= half && wave < 2 * half) {
                f32x4* const to = slot(wave - half);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
#pragma unroll
                    for (int j = 0; j < NDB; ++j) to[(t * NDB + j) * 64 + lane] = x.o[t][j];
                    if (x.g == 0) {
                        Ml[wave - half][t][0][x.li] = x.m[t];
                        Ml[wave - half][t][1][x.li] = x.l[t];
                    }
                }
            }
            __syncthreads();
            if (wave < half) {
                const f32x4* const from = slot(wave);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const float m2 = Ml[wave][t][0][x.li], l2 = Ml[wave][t][1][x.li];
                    const float mn = fmaxf(x.m[t], m2), ref = mn == OPS_NEG_INF ? 0.0f : mn;
                    const float c1 = ops_exp2(x.m[t] - ref), c2 = ops_exp2(m2 - ref);
                    x.m[t] = mn;
                    x.l[t] = x.l[t] * c1 + l2 * c2;
#pragma unroll
                    for (int j = 0; j < NDB; ++j) x.o[t][j] = x.o[t][j] * c1 + from[(t * NDB + j) * 64 + lane] * c2;
                }
            }
        }
    }
    if (wave != 0) return;
    int specials = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) specials |= any_special[i];
    x.store(w, V, w.rfirst, 0, lane, specials != 0);
}

// ---------------------------------------------------------------------------
// Many rows: the waves share the keys.
// ---------------------------------------------------------------------------
template <typename T, int D, int MT, int MOD, bool VEC>
__device__ __forceinline__ void rows_shared(const RowsParams& p) {
    constexpr int NW = 8, SK = sizeof(T) == 4 || D > 128 ? 32 : 64, TILE = SK * D, KB = SK / 16;
    constexpr int RING = TILE * (int)sizeof(T) > 16384 ? 2 : 3;   // stages in LDS
    using R = RowTiles<T, D, MT, KB, MOD, VEC>;
    using Src = RowSource<T, D, SK, NW>;
    T* const K0 = lds_array<T, TILE, 0>();
    T* const V0 = lds_array<T, TILE, 1>();
    T* const K1 = lds_array<T, TILE, 2>();
    T* const V1 = lds_array<T, TILE, 3>();
    constexpr int THIRD = (RING > 2) ? TILE : 8;
    T* const K2 = (RING > 2) ? lds_array<T, THIRD, 4>() : K0;
    T* const V2 = (RING > 2) ? lds_array<T, THIRD, 5>() : V0;
    __shared__ int Special;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    RowsWork w;
    if (!rows_work(p, 16 * MT * NW, lane, &w)) return;
    const CachePages pages = rows_pages(p, w.b);
    const T* const K = reinterpret_cast<const T*>(p.k) + w.hk * p.ks.h + (p.table ? 0 : w.b * p.ks.b);
    const T* const V = reinterpret_cast<const T*>(p.v) + w.hk * p.vs.h + (p.table ? 0 : w.b * p.vs.b);
    const Src ksrc(K, p.ks.s, p.ks.b, p.d, wave, lane), vsrc(V, p.vs.s, p.vs.b, p.d, wave, lane);
    const int nst = (w.kwalk() + SK - 1) / SK;
    const int rfirst = w.rfirst + 16 * MT * wave;
    const int act = rfirst < w.nrows;

    // whether the stages on their way have bad pages; those of the stage to fill next are looked up a stage ahead
    int bad_now = 0, bad_1 = 0, bad_2 = 0, bad_next = 0;
    int page[SK / 16];
    auto look_up = [&](int st) {
        const int k0 = w.key(st * SK);
        if (VEC) bad_next = Src::look_up(pages, k0, st < nst ? w.kend : k0, page);
    };
    auto fill = [&](int st, T* k, T* v) -> int {
        const int k0 = w.key(st * SK);
        const int bad = bad_next;
        if constexpr (VEC) {
            const int end = st < nst ? w.kend : k0;
            ksrc.fill(k, k0, end, page, pages, wave);
            vsrc.fill(v, k0, end, page, pages, wave);
            look_up(st + 1);
        } else if (k0 < w.kend) {
            ksrc.fill_slow(k, k0, w.kend, pages, p.d, tid);
            vsrc.fill_slow(v, k0, w.kend, pages, p.d, tid);
        }
        return bad;
    };
    look_up(0);
    // All waves' share of a stage has landed, and all are done with the stage before; younger: DMA issued since.
    auto arrive = [&](auto younger) {
        if constexpr (VEC) {
            wait_vmcnt<decltype(younger)::value>();
            __builtin_amdgcn_s_barrier();
            reread();
        } else {
            __syncthreads();
        }
    };
    if (tid == 0) Special = 0;
    R x;
    x.init(p, w, rfirst, lane);
    __syncthreads();
    // the two waves of a SIMD out of step: one multiplies while the other is in its softmax
    if (wave < NW / 2) __builtin_amdgcn_s_setprio(1);
    bad_now = fill(0, K0, V0);
    if (RING > 2) bad_1 = fill(1, K1, V1);
    auto step = [&](int st, T* k, T* v, T* kn, T* vn) {
        const int k0 = w.key(st * SK);
        // the same on all waves: a barrier hangs on it
        const int bad = VEC ? bad_now : Src::bad_rows(pages, k0, w.kend, lane);
        arrive(std::integral_constant<int, (RING - 2) * 2 * Src::NI>{});
        const int filled = fill(st + RING - 1, kn, vn);
        if (RING > 2) bad_2 = filled;
        else bad_1 = filled;
        const int masked = bad || rows_masked(p, w, k0, SK);
        if (act) {
            x.scores(p, w, k, k0, masked, bad);
            x.softmax();
        }
        if (masked) {
            if (Swizzled<T, D>::template clean<SK, 64 * NW>(v, tid)) Special = 1;
            __syncthreads();
        }
        if (act) x.values(v);
        bad_now = bad_1;
        bad_1 = bad_2;
    };
    if constexpr (RING == 3) {
        for (int st = 0; st < nst; st += 3) {
            step(st, K0, V0, K2, V2);
            if (st + 1 < nst) step(st + 1, K1, V1, K0, V0);
            if (st + 2 < nst) step(st + 2, K2, V2, K1, V1);
        }
    } else {
        for (int st = 0; st < nst; st += 2) {
            step(st, K0, V0, K1, V1);
            if (st + 1 < nst) step(st + 1, K1, V1, K0, V0);
        }
    }
    __syncthreads();
    x.close();
    if (act) x.store(w, V, rfirst, MT * wave, lane, Special != 0);
}

// Joins the partial sums of a row, D / 4 lanes a run (some 4 us for 512 rows of 9 runs: a launch's time).  WIDE: a workgroup a row, the runs dealt to
// its groups of lanes, whose sums meet in LDS; else (few runs) a group of lanes a row.
template <typename T, int D, bool VEC, bool WIDE>
__device__ __forceinline__ void rows_merge(const RowsParams& p) {
    constexpr int L = D / 4, N = 256 / L, G = WIDE ? N : 1;
    __shared__ f32x4 sums[G][L];
    __shared__ float ls[G];
    const int nrows = p.n * p.group, rows = p.block_rows, tid = threadIdx.x;
    const int grp = WIDE ? tid / L : 0, lane = tid % L;
    // past the last row: the last one again, so that all lanes take part in what follows
    const int64_t last = (int64_t)p.batch * p.kv_heads * nrows - 1, at = (int64_t)blockIdx.x * N + tid / L;
    const int64_t id = WIDE ? blockIdx.x : min(at, last);
    const int kv = id / nrows, r = id % nrows;
    const int b = kv / p.kv_heads, hk = kv % p.kv_heads, h = hk * p.group + r % p.group, token = r / p.group;
    const Runs runs = runs_of_sequence(p, b, tid & 63);
    if (runs.count == 1) return;   // written by its run
    const int64_t next = (int64_t)p.kv_heads * p.nrb * rows;   // rows from one run's partial sums to the next's
    const int64_t part = ((int64_t)runs.first * p.kv_heads + hk) * p.nrb + r / rows;
    const float* const ml = p.part_ml + part * 2 * rows + r % rows;
    const float* const po = p.part_o + (part * rows + r % rows) * D + 4 * lane;
    float mx = OPS_NEG_INF;
    if constexpr (WIDE) {
        for (int s = tid & 63; s < runs.count; s += 64) mx = fmaxf(mx, ml[s * 2 * next]);
#pragma unroll
        for (int s = 1; s < 64; s *= 2) mx = fmaxf(mx, __shfl_xor(mx, s));
    } else {
#pragma unroll 4
        for (int s = 0; s < runs.count; ++s) mx = fmaxf(mx, ml[s * 2 * next]);
    }
    const float ref = mx == OPS_NEG_INF ? 0.0f : mx;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
#pragma unroll 4
    for (int s = grp; s < runs.count; s += G) {
        const float c = ops_exp2(ml[s * 2 * next] - ref);
        l += c * ml[s * 2 * next + rows];
        o += c * *reinterpret_cast<const f32x4*>(po + s * next * D);
    }
    if constexpr (WIDE) {
        sums[grp][lane] = o;
        if (lane == 0) ls[grp] = l;
        __syncthreads();
        if (grp != 0) return;
#pragma unroll
        for (int i = 1; i < G; ++i) {
            o += sums[i][lane];
            l += ls[i];
        }
    }
    store4<T, VEC>(reinterpret_cast<T*>(p.out) + b * p.os.b + h * p.os.h + token * p.os.s, 4 * lane, p.d,
                   o * (l == 0.0f ? 0.0f : 1.0f / l));
    if (p.lse && lane == 0)
        p.lse[((int64_t)b * p.heads + h) * p.n + token] =
            l == 0.0f ? OPS_NEG_INF : (mx + __builtin_log2f(l) - kProbLog2<T>) * kLn2;
}

#define PASTE_(a, b, c, d) a##b##c##d
#define PASTE(a, b, c, d) PASTE_(a, b, c, d)
#define KERNEL(F, BODY, D, MT, MOD, VEC, TAG, THREADS, WAVES)                                                  \
    extern "C" __global__ __launch_bounds__(THREADS, WAVES) void PASTE(F, OPS_NAME, _d##D##_t##MT, TAG)(RowsParams p) { \
        BODY<OPS_T, D, MT, MOD, VEC>(p);                                                                       \
    }
// plain scores, capped (c), with a bias (b) or both (cb); any alignment and page size (s)
// windows: plain scores, or looked up (m)
#ifdef OPS_WINDOW
#define KINDS(F, BODY, D, MT, THREADS, WAVES)                            \
    KERNEL(F, BODY, D, MT, 0, true, , THREADS, WAVES)                    \
    KERNEL(F, BODY, D, MT, kAny, true, m, THREADS, WAVES)
#else
#define KINDS(F, BODY, D, MT, THREADS, WAVES)                            \
    KERNEL(F, BODY, D, MT, 0, true, , THREADS, WAVES)                    \
    KERNEL(F, BODY, D, MT, kCap, true, c, THREADS, WAVES)                \
    KERNEL(F, BODY, D, MT, kBias, true, b, THREADS, WAVES)               \
    KERNEL(F, BODY, D, MT, kCap | kBias, true, cb, THREADS, WAVES)
#endif
#define STREAM(D, MT, WAVES) KINDS(fa_rows_stream_, rows_stream, D, MT, (64 * kStreamWaves<D * (int)sizeof(OPS_T)>), WAVES)
#define SHARED(D, MT, WAVES) KINDS(fa_rows_shared_, rows_shared, D, MT, 512, WAVES)
#define MERGE(D, VEC, WIDE, TAG)                                                                                  \
    extern "C" __global__ __launch_bounds__(256) void PASTE(fa_rows_merge_, OPS_NAME, _d##D, TAG)(RowsParams p) { \
        rows_merge<OPS_T, D, VEC, WIDE>(p);                                                                       \
    }
#define COMMON(D)                                                                                               \
    KERNEL(fa_rows_shared_, rows_shared, D, 1, kAny, false, s, 512, 2)                                          \
    MERGE(D, true, false, )                                                                                     \
    MERGE(D, true, true, w)                                                                                     \
    MERGE(D, false, true, s)
COMMON(64)
COMMON(128)
COMMON(256)
STREAM(64, 1, 2)
STREAM(128, 1, 2)
#ifdef OPS_16BIT
STREAM(64, 2, 2)
STREAM(256, 1, 2)
SHARED(64, 2, 2)
SHARED(128, 2, 2)
#endif
SHARED(64, 1, 2)
SHARED(128, 1, 2)
SHARED(256, 1, 2)
