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
// their sines and cosines are formed once, a pair a thread, from angles reduced in 64 bits, and shared through LDS.

#include "fa_ops_common.h"

template <typename T, int W>
struct NormRun {
    typedef T type __attribute__((ext_vector_type(W == 1 ? 2 : W)));
};

// W (at least 2) floats of LDS, 8-byte aligned at least
template <int N>
__device__ __forceinline__ void load_floats(float (&to)[N], const float* from) {
#pragma unroll
    for (int e = 0; e < N; ++e) to[e] = from[e];
}

template <typename T, int W, int NU, bool BACK>
__device__ __forceinline__ void norm_body(const NormParams& p) {
    typedef typename NormRun<T, W>::type run;
    constexpr int PAIRS = W;   // pairs of a unit, at most
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
    const bool inner = W > 1 && p.interleaved;   // pairs inside a run

    if (x.norm) {
        for (int i = tid; i < tokens * half; i += kNormThreads) {
            const int t = i / half, pair = i % half;
            const double a = (double)p.pos[tok0 + t] * p.turns[pair];
            float s, c;
            sincospif(2.0f * (float)(a - rint(a)), &s, &c);
            cosines[t * half + pair] = c * p.gain;
            sines[t * half + pair] = BACK ? -s * p.gain : s * p.gain;
        }
        __syncthreads();
    }

    // the lane's units: first those of the rotary columns, then runs of copied ones
    const int L = p.lanes, R = kNormThreads / L, slot = tid / L;
    const int nrot = inner ? p.rot / W : half / W;
    int c0[NU], c1[NU], pair[NU];
    bool there[NU], rotary[NU], two[NU];
    float wa[NU][W], wb[NU][W], ga[NU][W], gb[NU][W];   // weights, and sums of their gradients
#pragma unroll
    for (int k = 0; k < NU; ++k) {
        const int unit = (tid & (L - 1)) + k * L;
        there[k] = unit < p.units;
        rotary[k] = there[k] && unit < nrot;
        two[k] = rotary[k] && !inner;
        c0[k] = !there[k] ? 0 : !rotary[k] ? p.rot + (unit - nrot) * W : W == 1 && p.interleaved ? 2 * unit : unit * W;
        c1[k] = !two[k] ? c0[k] : W == 1 && p.interleaved ? c0[k] + 1 : c0[k] + half;
        pair[k] = !rotary[k] ? 0 : inner ? unit * (W / 2) : unit * W;
        const T* const weight = reinterpret_cast<const T*>(x.w);
#pragma unroll
        for (int e = 0; e < W; ++e) {
            wa[k][e] = x.norm && x.w && there[k] ? float(weight[c0[k] + e]) : 1.0f;
            wb[k][e] = x.norm && x.w && two[k] ? float(weight[c1[k] + e]) : 1.0f;
            ga[k][e] = gb[k][e] = 0.0f;
        }
    }

    struct Row {
        run xa[NU], xb[NU], da[BACK ? NU : 1], db[BACK ? NU : 1];
        T* to;
        int t;
    };
    auto fetch = [&](run* a, run* b, const T* from, int k) {
        if constexpr (W == 1) {
            a[k][0] = there[k] ? from[c0[k]] : T(0.0f);
            b[k][0] = two[k] ? from[c1[k]] : T(0.0f);
        } else {
            a[k] = b[k] = run{};
            if (there[k]) a[k] = *reinterpret_cast<const run*>(from + c0[k]);
            if (two[k]) b[k] = *reinterpret_cast<const run*>(from + c1[k]);
        }
    };
    const int b0 = tok0 / p.seq, i0 = tok0 % p.seq;
    // row `head` of token tok0 + t; to = nullptr: it has no place
    auto load = [&](int t, int head) {
        Row r;
        int b = b0, i = i0 + t;
        while (i >= p.seq) {
            i -= p.seq;
            ++b;
        }
        const T* const from = reinterpret_cast<const T*>(x.x) + b * x.xs.b + i * x.xs.s + head * x.xs.h;
        const T* const grad = BACK ? reinterpret_cast<const T*>(x.dy) + b * x.dys.b + i * x.dys.s + head * x.dys.h : from;
#pragma unroll
        for (int k = 0; k < NU; ++k) {
            fetch(r.xa, r.xb, from, k);
            if (BACK) fetch(r.da, r.db, grad, k);
        }
        r.t = t;
        r.to = reinterpret_cast<T*>(x.out);
        if (!r.to) return r;
        r.to += head * x.outs.h;
        if (!BACK && x.cache) {
            const int len = p.lens[b];
            const int64_t row = (int64_t)len + i;
            if (len < 0 || row >= p.capacity) {
                r.to = nullptr;
            } else if (p.table) {
                const int page = p.table[(int64_t)b * p.pages_per_seq + (row >> p.page_shift)];
                if ((unsigned)page >= (unsigned)p.n_pages) r.to = nullptr;
                else r.to += page * x.outs.b + (row & ((1 << p.page_shift) - 1)) * x.outs.s;
            } else {
                r.to += b * x.outs.b + row * x.outs.s;
            }
        } else {
            r.to += b * x.outs.b + i * x.outs.s;
        }
        return r;
    };
    // turns the pairs of unit k by the row's angles
    auto turn = [&](float (&a)[W], float (&b)[W], int t, int k) {
        if (!rotary[k]) return;
        float cs[PAIRS], sn[PAIRS];
        const int at = t * half + pair[k];
        if constexpr (W > 1) {
            if (inner) {
                float c2[W / 2], s2[W / 2];
                load_floats(c2, cosines + at);
                load_floats(s2, sines + at);
#pragma unroll
                for (int e = 0; e < W / 2; ++e) {
                    const float u = a[2 * e], v = a[2 * e + 1];
                    a[2 * e] = u * c2[e] - v * s2[e];
                    a[2 * e + 1] = u * s2[e] + v * c2[e];
                }
                return;
            }
        }
        load_floats(cs, cosines + at);
        load_floats(sn, sines + at);
#pragma unroll
        for (int e = 0; e < W; ++e) {
            const float u = a[e], v = b[e];
            a[e] = u * cs[e] - v * sn[e];
            b[e] = u * sn[e] + v * cs[e];
        }
    };
    auto row_sum = [&](float s) {
        for (int m = 1; m < L; m *= 2) s += __shfl_xor(s, m);
        return s;
    };
    auto store = [&](const Row& r, int k, const float (&a)[W], const float (&b)[W]) {
        if constexpr (W == 1) {
            if (there[k]) r.to[c0[k]] = T(a[0]);
            if (two[k]) r.to[c1[k]] = T(b[0]);
        } else {
            run ya, yb;
#pragma unroll
            for (int e = 0; e < W; ++e) {
                ya[e] = T(a[e]);
                yb[e] = T(b[e]);
            }
            if (there[k]) *reinterpret_cast<run*>(r.to + c0[k]) = ya;
            if (two[k]) *reinterpret_cast<run*>(r.to + c1[k]) = yb;
        }
    };
    const float inv_d = 1.0f / (float)p.d;
    // (all lanes of a row come here together; `real`: it is one)
    auto process = [&](const Row& r, bool real) {
        float a[NU][W], b[NU][W];
        float ss = 0.0f;
#pragma unroll
        for (int k = 0; k < NU; ++k)
#pragma unroll
            for (int e = 0; e < W; ++e) {
                a[k][e] = float(r.xa[k][e]);
                b[k][e] = float(r.xb[k][e]);
                ss = __builtin_fmaf(a[k][e], a[k][e], ss);
                ss = __builtin_fmaf(b[k][e], b[k][e], ss);
            }
        if constexpr (!BACK) {
            if (x.norm) {
                const float rs = 1.0f / sqrtf(__builtin_fmaf(row_sum(ss), inv_d, p.eps));
#pragma unroll
                for (int k = 0; k < NU; ++k) {
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        a[k][e] *= rs * wa[k][e];
                        b[k][e] *= rs * wb[k][e];
                    }
                    turn(a[k], b[k], r.t, k);
                }
            }
            if (real && r.to) {
#pragma unroll
                for (int k = 0; k < NU; ++k) store(r, k, a[k], b[k]);
            }
        } else {
            float da[NU][W], db[NU][W], sg = 0.0f;
#pragma unroll
            for (int k = 0; k < NU; ++k) {
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    da[k][e] = float(r.da[k][e]);
                    db[k][e] = float(r.db[k][e]);
                }
                turn(da[k], db[k], r.t, k);
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    sg = __builtin_fmaf(da[k][e] * wa[k][e], a[k][e], sg);
                    sg = __builtin_fmaf(db[k][e] * wb[k][e], b[k][e], sg);
                }
            }
            const float rs = 1.0f / sqrtf(__builtin_fmaf(row_sum(ss), inv_d, p.eps));
            const float mean = row_sum(sg) * rs * rs * inv_d;
#pragma unroll
            for (int k = 0; k < NU; ++k)
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    if (real) {
                        ga[k][e] = __builtin_fmaf(da[k][e], a[k][e] * rs, ga[k][e]);
                        gb[k][e] = __builtin_fmaf(db[k][e], b[k][e] * rs, gb[k][e]);
                    }
                    a[k][e] = rs * (da[k][e] * wa[k][e] - a[k][e] * mean);
                    b[k][e] = rs * (db[k][e] * wb[k][e] - b[k][e] * mean);
                }
            if (real && r.to) {
#pragma unroll
                for (int k = 0; k < NU; ++k) store(r, k, a[k], b[k]);
            }
        }
    };

    // rows slot, slot + R, ... of the workgroup's; the next one is on its way while one is worked on
    const int rows = tokens * x.heads, steps = (rows + R - 1) / R, dt = R / x.heads, dh = R % x.heads;
    int t = slot / x.heads, head = slot % x.heads;
    auto clamped = [&](int i) {   // past the last row: row 0, whose results are dropped
        return i * R + slot < rows ? load(t, head) : load(0, 0);
    };
    auto advance = [&] {
        t += dt;
        head += dh;
        if (head >= x.heads) {
            head -= x.heads;
            ++t;
        }
    };
    Row cur = clamped(0);
    for (int i = 0; i < steps; ++i) {
        advance();
        Row next = cur;
        if (i + 1 < steps) next = clamped(i + 1);
        process(cur, i * R + slot < rows);
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
                    gb[k][e] += __shfl_xor(gb[k][e], m);
                }
                if ((tid & 63) < L) {
                    if (there[k]) sums[wave][c0[k] + e] = ga[k][e];
                    if (two[k]) sums[wave][c1[k] + e] = gb[k][e];
                }
            }
        __syncthreads();
        if (tid < p.d) x.part[(int64_t)blk * p.d + tid] = sums[0][tid] + sums[1][tid] + sums[2][tid] + sums[3][tid];
    }
}

// Sums of the workgroups' weight gradients: 16 columns of a tensor a workgroup, the partial sums dealt to 64 threads
// each.
extern "C" __global__ __launch_bounds__(1024) void fa_norm_weights(NormParams p) {
    __shared__ float sums[64][17];
    const int per = (p.d + 15) / 16, n = blockIdx.x / per, c = blockIdx.x % per * 16 + threadIdx.x % 16;
    const int grp = threadIdx.x / 16;
    const NormTensor& x = p.t[n];
    float s = 0.0f;
    if (c < p.d && x.dw)
        for (int i = grp; i < x.blocks; i += 64) s += x.part[(int64_t)i * p.d + c];
    sums[grp][threadIdx.x % 16] = s;
    __syncthreads();
    if (grp != 0 || c >= p.d || !x.dw) return;
    s = 0.0f;
    for (int i = 0; i < 64; ++i) s += sums[i][threadIdx.x];
    x.dw[c] = s;
}

#define NORM_KERNEL(NAME, T, W, NU, BACK) \
    extern "C" __global__ __launch_bounds__(kNormThreads) void NAME(NormParams p) { norm_body<T, W, NU, BACK>(p); }
#define NORM_KERNELS(N, T)                                               \
    NORM_KERNEL(fa_norm_##N##_1, T, 16 / (int)sizeof(T), 1, false)       \
    NORM_KERNEL(fa_norm_##N##_0, T, 1, 4, false)                         \
    NORM_KERNEL(fa_norm_back_##N##_1, T, 16 / (int)sizeof(T), 1, true)   \
    NORM_KERNEL(fa_norm_back_##N##_0, T, 1, 4, true)
NORM_KERNELS(bf16, __bf16)
NORM_KERNELS(f16, _Float16)
NORM_KERNELS(f32, float)
