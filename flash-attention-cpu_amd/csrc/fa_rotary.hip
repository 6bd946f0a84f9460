// fa_rotary.hip -- gfx950 kernels of rotary positions (fa_rotary) and of the
// cache append that rotates on the way (fa_cache_append).
//
// Bound by memory: every value is read and written once.  A thread owns a token's unit
// of columns (WIDE: 16 bytes of a column run and, in the half layout, the 16 bytes half the
// rotary columns further; else one pair or one copied column), finds the
// sines and cosines of its pairs once and runs over the heads of all tensors with
// them.  Angles are position * turns in 64 bits, of which only the fraction
// goes into sin and cos.  (bf16, 8192 tokens of 32 + 8 heads of 128 columns: 37 us, 4.5 TB/s; f32, 2 x 1000 tokens of
// 16 + 16 heads of 80 columns, 40 of them rotary: 10 us.)

#include "fa_ops_common.h"

template <typename T, bool WIDE>
__device__ __forceinline__ void rotary_body(const RotParams& p) {
    constexpr int W = WIDE ? 16 / (int)sizeof(T) : 1;   // columns of a run
    typedef T run __attribute__((ext_vector_type(W == 1 ? 2 : W)));
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int unit = id % p.cols;
    const int ht = id / p.cols % p.hthreads;
    const int64_t tok = id / p.cols / p.hthreads;
    if (tok >= (int64_t)p.batch * p.seq) return;
    const int b = tok / p.seq, i = tok % p.seq;

    // units: first those of the rotary columns, then runs of copied ones
    const int half = p.rot / 2;
    const int nrot = WIDE ? (p.interleaved ? p.rot / W : half / W) : half;
    const bool rotary = unit < nrot;
    int c0, c1;   // columns of the unit's first and second run
    if (!rotary) {
        c0 = c1 = p.rot + (unit - nrot) * W;
    } else if (p.interleaved) {
        c0 = WIDE ? unit * W : 2 * unit;
        c1 = c0 + 1;
    } else {
        c0 = unit * W;
        c1 = c0 + half;
    }
    float cs[W], sn[W];
    if (rotary) {
        const double at = (double)p.pos[tok];
#pragma unroll
        for (int e = 0; e < W; ++e) {
            if (WIDE && p.interleaved && e >= W / 2) break;
            const int pair = p.interleaved && WIDE ? unit * (W / 2) + e : unit * W + e;
            const double a = at * p.turns[pair];
            float s, c;
            sincospif(2.0f * (float)(a - rint(a)), &s, &c);
            cs[e] = c * p.gain;
            sn[e] = s * p.gain * p.sign;
        }
    }
    for (int n = 0; n < p.nt; ++n) {
        const RotTensor& x = p.t[n];
        const T* src = reinterpret_cast<const T*>(x.src) + b * x.in.b + i * x.in.s;
        T* dst = reinterpret_cast<T*>(x.dst);
        if (x.cache) {
            const int len = p.lens[b];
            const int64_t row = (int64_t)len + i;
            if (len < 0 || row >= p.capacity) continue;
            if (p.table) {
                const int page = p.table[(int64_t)b * p.pages_per_seq + (row >> p.page_shift)];
                if ((unsigned)page >= (unsigned)p.n_pages) continue;
                dst += page * x.out.b + (row & ((1 << p.page_shift) - 1)) * x.out.s;
            } else {
                dst += b * x.out.b + row * x.out.s;
            }
        } else {
            dst += b * x.out.b + i * x.out.s;
        }
        for (int h = ht; h < x.heads; h += p.hthreads) {
            const T* from = src + h * x.in.h;
            T* to = dst + h * x.out.h;
            if constexpr (WIDE) {
                const run u = *reinterpret_cast<const run*>(from + c0);
                if (!rotary) {
                    *reinterpret_cast<run*>(to + c0) = u;
                } else if (p.interleaved) {
                    run y = u;
                    if (x.rotate) {
#pragma unroll
                        for (int e = 0; e < W / 2; ++e) {
                            const float a = float(u[2 * e]), c = float(u[2 * e + 1]);
                            y[2 * e] = T(a * cs[e] - c * sn[e]);
                            y[2 * e + 1] = T(a * sn[e] + c * cs[e]);
                        }
                    }
                    *reinterpret_cast<run*>(to + c0) = y;
                } else {
                    const run v = *reinterpret_cast<const run*>(from + c1);
                    run y = u, z = v;
                    if (x.rotate) {
#pragma unroll
                        for (int e = 0; e < W; ++e) {
                            const float a = float(u[e]), c = float(v[e]);
                            y[e] = T(a * cs[e] - c * sn[e]);
                            z[e] = T(a * sn[e] + c * cs[e]);
                        }
                    }
                    *reinterpret_cast<run*>(to + c0) = y;
                    *reinterpret_cast<run*>(to + c1) = z;
                }
            } else if (!rotary) {
                to[c0] = from[c0];
            } else {
                const T u = from[c0], v = from[c1];
                if (x.rotate) {
                    to[c0] = T(float(u) * cs[0] - float(v) * sn[0]);
                    to[c1] = T(float(u) * sn[0] + float(v) * cs[0]);
                } else {
                    to[c0] = u;
                    to[c1] = v;
                }
            }
        }
    }
}

#define ROTARY_KERNELS(N, T)                                                                                   \
    extern "C" __global__ __launch_bounds__(256) void fa_rotary_##N##_1(RotParams p) { rotary_body<T, true>(p); } \
    extern "C" __global__ __launch_bounds__(256) void fa_rotary_##N##_0(RotParams p) { rotary_body<T, false>(p); }
ROTARY_KERNELS(bf16, __bf16)
ROTARY_KERNELS(f16, _Float16)
ROTARY_KERNELS(f32, float)
