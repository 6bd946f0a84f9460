// fa_norm.hip -- gfx950 kernels of the norms of queries and keys with rotary
// positions in the same pass (fa_norm_rotary, fa_norm_rotary_backward,
// fa_norm_cache_append).
//
//     y = R(pos) (x r w),   r = 1 / sqrt(mean x^2 + eps)
// and backward, with g = R^T dy,
//     dw = sum over rows of g x r,   dx = r (w g - x r^2 mean(w g x))
//
// Bound by memory: every value is read and written once.  A head row is kept by L neighbouring lanes (a power of
// two), each with one unit of columns (W > 1: 16 bytes of a column run and, in the half layout, the 16 bytes half the
// rotary columns further; W = 1: up to four pairs or copied columns), so that the sums over a row are a few
// exchanges between lanes and pairs never leave a lane.  A workgroup takes the rows of a few tokens of one tensor;
// their sines and cosines are formed once, a pair a thread, from angles reduced in 64 bits, and shared through LDS:
// the more tokens a workgroup has, the fewer of them there are to fill the GPU (plan_norm).
// bf16, 8192 tokens of 32 + 8 heads of 128 columns: 31 us (5.4 TB/s; 41 between passes over different inputs); backward
// 2 x 4096 tokens of 16 + 4 heads 31 us (4.1 TB/s, since two sums a row come before the first store) and 4.7 us for the
// weights' sums; a token of 32 sequences into a cache 5.7 us, a launch and one chain of loads.  Where runs of columns are no
// whole 16 bytes it is bound by loads of single columns: bf16, 8192 tokens of 40 heads of 80 columns, 40 of them rotary in two
// halves 101 us, interleaved 32.

#include "fa_ops_common.h"

template <typename T, int W>
struct NormRun {
    typedef T type __attribute__((ext_vector_type(W == 1 ? 2 : W)));
};

// N floats of LDS, aligned to 16 bytes or their own size
template <int N>
__device__ __forceinline__ void load_floats(float (&to)[N], const float* from) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int e = 0; e < N; e += 4) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(from + e);
#pragma unroll
            for (int r = 0; r < 4; ++r) to[e + r] = x[r];
        }
    } else if constexpr (N == 2) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const f32x2 x = *reinterpret_cast<const f32x2*>(from);
        to[0] = x[0];
        to[1] = x[1];
    } else {
        to[0] = from[0];
    }
}

// Where a lane's rows lie in one tensor: element offset of the present row, and what it grows by.
struct NormWalk {
    int64_t at, step, head_wrap, seq_wrap;
    __device__ __forceinline__ NormWalk(const OpsStrides& st, int b, int i, int seq, int heads, int t, int head, int dt, int dh) {
        at = b * st.b + (i + t) * st.s + head * st.h;
        step = dt * st.s + dh * st.h;
        head_wrap = st.s - heads * st.h;
        seq_wrap = st.b - seq * st.s;
    }
    __device__ __forceinline__ void advance(bool head, int seqs) {
        at += step;
        if (head) at += head_wrap;
        if (seqs) at += seqs * seq_wrap;
    }
};

// FULL: rotary columns alone, a unit for every lane (the half layout: of two runs).  INNER: pairs inside a run.
template <typename T, int W, int NU, bool BACK, bool INNER, bool FULL>
__device__ __forceinline__ void norm_body(const NormParams& p) {
    typedef typename NormRun<T, W>::type run;
    constexpr bool kTwo = !INNER;   // units of rotary columns have two runs
    constexpr int RB = kTwo ? NU : 1;
    __shared__ __attribute__((aligned(16))) float cosines[kNormTokens * 128];
    __shared__ __attribute__((aligned(16))) float sines[kNormTokens * 128];

    const int tid = threadIdx.x;
    int n = 0;
    unsigned blk = blockIdx.x;
    while (n + 1 < p.nt && blk >= (unsigned)p.t[n].blocks) blk -= p.t[n++].blocks;
    const NormTensor& x = p.t[n];
    const int64_t all = (int64_t)p.batch * p.seq, tok0 = (int64_t)blk * x.tokens;
    const int tokens = (int)min((int64_t)x.tokens, all - tok0);
    const int half = p.rot / 2;
    const bool norm = x.norm;

    // the lane's units: first those of the rotary columns, then runs of copied ones
    const int L = p.lanes, R = kNormThreads / L, slot = tid / L;
    const int nrot = INNER ? p.rot / W : half / W;
    int c0[NU], c1[RB], pair[NU];
    bool there[NU], two[NU];
#pragma unroll
    for (int k = 0; k < NU; ++k) {
        const int unit = (tid & (L - 1)) + k * L;
        there[k] = FULL || unit < p.units;
        two[k] = FULL || (there[k] && unit < nrot);
        c0[k] = !there[k] ? 0 : !two[k] ? p.rot + (unit - nrot) * W : W == 1 && p.interleaved ? 2 * unit : unit * W;
        if (kTwo) c1[k] = !two[k] ? c0[k] : W == 1 && p.interleaved ? c0[k] + 1 : c0[k] + half;
        pair[k] = !two[k] ? 0 : INNER ? unit * (W / 2) : unit * W;
    }

    // rows slot, slot + R, ... of the workgroup's; the next one is on its way while one is worked on
    const int rows = tokens * x.heads, steps = (rows + R - 1) / R, dt = R / x.heads, dh = R % x.heads;
    int t = slot / x.heads, head = slot % x.heads;
    int b = tok0 / p.seq, i = tok0 % p.seq;
    NormWalk wx(x.xs, b, i, p.seq, x.heads, t, head, dt, dh);
    NormWalk wo(x.outs, b, i, p.seq, x.heads, t, head, dt, dh);
    NormWalk wd(BACK ? x.dys : x.xs, b, i, p.seq, x.heads, t, head, dt, dh);
    i += t;
    auto wraps = [&] {   // sequences that the row has passed
        int k = 0;
        while (i >= p.seq) {
            i -= p.seq;
            ++k;
        }
        b += k;
        return k;
    };
    {
        const int k = wraps();
        wx.at += k * wx.seq_wrap;
        wo.at += k * wo.seq_wrap;
        if (BACK) wd.at += k * wd.seq_wrap;
    }
    auto advance = [&] {
        t += dt;
        i += dt;
        head += dh;
        const bool wrap = head >= x.heads;
        if (wrap) {
            head -= x.heads;
            ++t;
            ++i;
        }
        const int k = wraps();
        wx.advance(wrap, k);
        if (BACK || !x.cache) wo.advance(wrap, k);
        if (BACK) wd.advance(wrap, k);
    };
    struct Row {
        run xa[NU], xb[RB], da[BACK ? NU : 1], db[BACK ? RB : 1];
        T* to;   // nullptr: not stored
        int t;
    };
    // Fills one row of a tensor; lanes without it get zeros.
    auto fetch = [&](const T* from, int k, run& a, run& bb) {
        if constexpr (W == 1) {
            a[0] = there[k] ? from[c0[k]] : T(0.0f);
            bb[0] = two[k] ? from[c1[k]] : T(0.0f);
        } else {
            a = run{};
            if (there[k]) a = *reinterpret_cast<const run*>(from + c0[k]);
            if constexpr (kTwo) {
                bb = run{};
                if (two[k]) bb = *reinterpret_cast<const run*>(from + c1[k]);
            }
        }
    };
    auto load = [&](Row& r, bool real) {
        r.to = nullptr;
        r.t = 0;
#pragma unroll
        for (int k = 0; k < NU; ++k) {
            r.xa[k] = run{};
            if (kTwo) r.xb[k] = run{};
            if (BACK) r.da[k] = run{};
            if (BACK && kTwo) r.db[k] = run{};
        }
        if (!real) return;
        const T* const from = reinterpret_cast<const T*>(x.x) + wx.at;
        const T* const grad = reinterpret_cast<const T*>(x.dy) + wd.at;
#pragma unroll
        for (int k = 0; k < NU; ++k) {
            fetch(from, k, r.xa[k], r.xb[kTwo ? k : 0]);
            if constexpr (BACK) fetch(grad, k, r.da[k], r.db[kTwo ? k : 0]);
        }
        r.t = t;
        T* const out = reinterpret_cast<T*>(x.out);
        if (!BACK && x.cache) {
            const int len = p.lens[b];
            const int64_t row = (int64_t)len + i;
            if (len < 0 || row >= p.capacity) return;
            if (p.table) {
                const int page = p.table[(int64_t)b * p.pages_per_seq + (row >> p.page_shift)];
                if ((unsigned)page < (unsigned)p.n_pages)
                    r.to = out + page * x.outs.b + (row & ((1 << p.page_shift) - 1)) * x.outs.s + head * x.outs.h;
            } else {
                r.to = out + b * x.outs.b + row * x.outs.s + head * x.outs.h;
            }
        } else if (out) {
            r.to = out + wo.at;
        }
    };
    Row cur;
    load(cur, slot < rows);

    // weights (in the type: registers are short backward), and sums of their gradients
    run wa[NU], wb[RB];
    float ga[NU][W], gb[RB][W];
#pragma unroll
    for (int k = 0; k < NU; ++k)
#pragma unroll
        for (int e = 0; e < W; ++e) {
            const T* const weight = reinterpret_cast<const T*>(x.w);
            const bool given = norm && weight;
            wa[k][e] = given && there[k] ? weight[c0[k] + e] : T(1.0f);
            ga[k][e] = 0.0f;
            if (kTwo) {
                wb[k][e] = given && two[k] ? weight[c1[k] + e] : T(1.0f);
                gb[k][e] = 0.0f;
            }
        }
    if (norm) {
        for (int j = tid; j < tokens * half; j += kNormThreads) {
            const int tt = j / half, c = j % half;
            const double a = (double)p.pos[tok0 + tt] * p.turns[c];
            float s, cc;
            sincospif(2.0f * (float)(a - rint(a)), &s, &cc);
            cosines[j] = cc * p.gain;
            sines[j] = BACK ? -s * p.gain : s * p.gain;
        }
        __syncthreads();
    }

    // turns the pairs of unit k by the row's angles
    auto turn = [&](float (&a)[W], float (&bb)[W], int at, int k) {
        if (!FULL && !two[k]) return;
        if constexpr (INNER) {
            float c[W / 2 > 0 ? W / 2 : 1], s[W / 2 > 0 ? W / 2 : 1];
            load_floats(c, cosines + at + pair[k]);
            load_floats(s, sines + at + pair[k]);
#pragma unroll
            for (int e = 0; e < W / 2; ++e) {
                const float u = a[2 * e], v = a[2 * e + 1];
                a[2 * e] = u * c[e] - v * s[e];
                a[2 * e + 1] = u * s[e] + v * c[e];
            }
        } else {
            float c[W], s[W];
            load_floats(c, cosines + at + pair[k]);
            load_floats(s, sines + at + pair[k]);
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float u = a[e], v = bb[e];
                a[e] = u * c[e] - v * s[e];
                bb[e] = u * s[e] + v * c[e];
            }
        }
    };
    auto row_sum = [&](float s) {
        for (int m = 1; m < L; m *= 2) s += __shfl_xor(s, m);
        return s;
    };
    auto store = [&](T* to, int k, const float (&a)[W], const float (&bb)[W]) {
        if constexpr (W == 1) {
            if (there[k]) to[c0[k]] = T(a[0]);
            if (two[k]) to[c1[k]] = T(bb[0]);
        } else {
            run ya, yb;
#pragma unroll
            for (int e = 0; e < W; ++e) {
                ya[e] = T(a[e]);
                if (kTwo) yb[e] = T(bb[e]);
            }
            if (there[k]) *reinterpret_cast<run*>(to + c0[k]) = ya;
            if constexpr (kTwo) {
                if (two[k]) *reinterpret_cast<run*>(to + c1[k]) = yb;
            }
        }
    };
    const float inv_d = 1.0f / (float)p.d;
    float none[W];
    // (all lanes of a row come here together; rows that are none are zeros and have no place)
    auto process = [&](const Row& r) {
        float a[NU][W], bb[RB][W];
        float ss = 0.0f;
        const int at = r.t * half;
#pragma unroll
        for (int k = 0; k < NU; ++k)
#pragma unroll
            for (int e = 0; e < W; ++e) {
                a[k][e] = float(r.xa[k][e]);
                ss = __builtin_fmaf(a[k][e], a[k][e], ss);
                if (kTwo) {
                    bb[k][e] = float(r.xb[k][e]);
                    ss = __builtin_fmaf(bb[k][e], bb[k][e], ss);
                }
            }
        if constexpr (!BACK) {
            if (norm) {
                const float rs = rsqrtf(__builtin_fmaf(row_sum(ss), inv_d, p.eps));
#pragma unroll
                for (int k = 0; k < NU; ++k) {
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        a[k][e] *= rs * float(wa[k][e]);
                        if (kTwo) bb[k][e] *= rs * float(wb[k][e]);
                    }
                    turn(a[k], kTwo ? bb[kTwo ? k : 0] : none, at, k);
                }
            }
        } else {
            float da[NU][W], db[RB][W], sg = 0.0f;
#pragma unroll
            for (int k = 0; k < NU; ++k) {
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    da[k][e] = float(r.da[k][e]);
                    if (kTwo) db[k][e] = float(r.db[k][e]);
                }
                turn(da[k], kTwo ? db[kTwo ? k : 0] : none, at, k);
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    sg = __builtin_fmaf(da[k][e] * float(wa[k][e]), a[k][e], sg);
                    if (kTwo) sg = __builtin_fmaf(db[k][e] * float(wb[k][e]), bb[k][e], sg);
                }
            }
            for (int m = 1; m < L; m *= 2) {
                ss += __shfl_xor(ss, m);
                sg += __shfl_xor(sg, m);
            }
            const float rs = rsqrtf(__builtin_fmaf(ss, inv_d, p.eps));
            float mean = sg * rs * rs * inv_d;
            // Squares past f32's range: zeros, though the sum that the mean comes from may have passed it as well; NaN only
            // where the row itself is not finite.
            if (__builtin_amdgcn_ballot_w64(rs == 0.0f) != 0) {
                float zero = 0.0f;
#pragma unroll
                for (int k = 0; k < NU; ++k)
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        zero = __builtin_fmaf(a[k][e], rs, zero);
                        if (kTwo) zero = __builtin_fmaf(bb[k][e], rs, zero);
                    }
                zero = row_sum(zero);
                if (rs == 0.0f) mean = zero;
            }
#pragma unroll
            for (int k = 0; k < NU; ++k)
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    ga[k][e] = __builtin_fmaf(da[k][e], a[k][e] * rs, ga[k][e]);
                    a[k][e] = rs * __builtin_fmaf(-a[k][e], mean, da[k][e] * float(wa[k][e]));
                    if (kTwo) {
                        gb[k][e] = __builtin_fmaf(db[k][e], bb[k][e] * rs, gb[k][e]);
                        bb[k][e] = rs * __builtin_fmaf(-bb[k][e], mean, db[k][e] * float(wb[k][e]));
                    }
                }
        }
        if (r.to) {
#pragma unroll
            for (int k = 0; k < NU; ++k) store(r.to, k, a[k], kTwo ? bb[kTwo ? k : 0] : none);
        }
    };
    for (int j = 1; j <= steps; ++j) {
        Row next;
        if (j < steps) {
            advance();
            load(next, j * R + slot < rows);
        }
        process(cur);
        cur = next;
    }

    if constexpr (BACK) {
        // sums of the workgroup's rows: over the rows of a wave by exchanges, over the waves in LDS
        if (!x.part) return;
        __shared__ float sums[4][256];
        const int wave = tid >> 6;
#pragma unroll
        for (int k = 0; k < NU; ++k)
#pragma unroll
            for (int e = 0; e < W; ++e) {
                for (int m = L; m < 64; m *= 2) {
                    ga[k][e] += __shfl_xor(ga[k][e], m);
                    if (kTwo) gb[k][e] += __shfl_xor(gb[k][e], m);
                }
                if ((tid & 63) < L) {
                    if (there[k]) sums[wave][c0[k] + e] = ga[k][e];
                    if constexpr (kTwo) {
                        if (two[k]) sums[wave][c1[k] + e] = gb[k][e];
                    }
                }
            }
        __syncthreads();
        if (tid < p.d) x.part[(int64_t)blk * p.d + tid] = sums[0][tid] + sums[1][tid] + sums[2][tid] + sums[3][tid];
    }
}

// Sums of the workgroups' weight gradients: 8 columns of a tensor a workgroup, the partial sums dealt to 128 threads each
// (1536 workgroups: 3.9 us, a launch's time).
extern "C" __global__ __launch_bounds__(1024) void fa_norm_weights(NormParams p) {
    constexpr int C = kNormColumns, G = 1024 / C;
    __shared__ float sums[16][C];
    const int per = (p.d + C - 1) / C, n = blockIdx.x / per, c = blockIdx.x % per * C + threadIdx.x % C;
    const int grp = threadIdx.x / C;
    const NormTensor& x = p.t[n];
    float s = 0.0f;
    if (c < p.d && x.dw) {
#pragma unroll 8
        for (int i = grp; i < x.blocks; i += G) s += x.part[(int64_t)i * p.d + c];
    }
#pragma unroll
    for (int m = C; m < 64; m *= 2) s += __shfl_xor(s, m);
    if ((threadIdx.x & 63) < C) sums[threadIdx.x / 64][threadIdx.x % C] = s;
    __syncthreads();
    if (grp != 0 || c >= p.d || !x.dw) return;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += sums[i][threadIdx.x];
    x.dw[c] = s;
}

#define NORM_KERNEL(NAME, T, W, NU, BACK, INNER, FULL)                                    \
    extern "C" __global__ __launch_bounds__(kNormThreads, NU == 1 ? 4 : 2) void NAME(NormParams p) { \
        norm_body<T, W, NU, BACK, INNER, FULL>(p);                                         \
    }
// half layout or pairs inside runs (i), a unit for every lane (f), three units a lane (3: not the half layout of 16-bit
// types, whose 48 columns a lane do not fit the registers backward); any alignment and width (0)
#define NORM_KERNELS(F, N, T, BACK)                                              \
    NORM_KERNEL(F##_##N##_f, T, 16 / (int)sizeof(T), 1, BACK, false, true)       \
    NORM_KERNEL(F##_##N##_fi, T, 16 / (int)sizeof(T), 1, BACK, true, true)       \
    NORM_KERNEL(F##_##N##_1, T, 16 / (int)sizeof(T), 1, BACK, false, false)      \
    NORM_KERNEL(F##_##N##_1i, T, 16 / (int)sizeof(T), 1, BACK, true, false)      \
    NORM_KERNEL(F##_##N##_3i, T, 16 / (int)sizeof(T), 3, BACK, true, false)      \
    NORM_KERNEL(F##_##N##_0, T, 1, 4, BACK, false, false)
#define NORM_TYPE(N, T)                \
    NORM_KERNELS(fa_norm, N, T, false) \
    NORM_KERNELS(fa_norm_back, N, T, true)
NORM_TYPE(bf16, __bf16)
NORM_TYPE(f16, _Float16)
NORM_TYPE(f32, float)
NORM_KERNEL(fa_norm_f32_3, float, 4, 3, false, false, false)
NORM_KERNEL(fa_norm_back_f32_3, float, 4, 3, true, false, false)
