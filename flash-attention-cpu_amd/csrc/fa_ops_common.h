// fa_ops_common.h -- device helpers of the score, cache and rotary kernels:
// matrix-core operands that look alike for bf16, f16 and f32, tiles of rows in
// LDS, the modified score and its masks.
//
// Operands.  All products run on 16 x 16 x 32 steps: lane l (g = l / 16,
// li = l % 16) holds A[li][8g .. 8g + 7] and B[8g .. 8g + 7][li], and C[4g + r][li]
// in register r.  bf16 and f16 have that as one instruction; f32 takes eight
// 16 x 16 x 4 products, the e-th over the columns 8g + e of the four g, which adds
// up the same terms.
#ifndef FA_OPS_COMMON_H
#define FA_OPS_COMMON_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "fa_ops_params.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

#define OPS_NEG_INF (-__builtin_huge_valf())

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;
// The reference that exponentials are taken against may trail the true
// maximum of a row by this much (log2 units) before the sums are rescaled.
constexpr float kLazy = 8.0f;

template <typename T>
struct Mma;
template <>
struct Mma<__bf16> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    typedef __bf16 v4 __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ f32x4 mma(v8 a, v8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mma<_Float16> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v4 __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ f32x4 mma(v8 a, v8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mma<float> {
    typedef f32x8 v8;
    typedef f32x4 v4;
    static __device__ __forceinline__ f32x4 mma(v8 a, v8 b, f32x4 c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};

// Probabilities of f16 products are taken 2^7 times larger: those down to 2^-21
// then round as normal numbers, and with the lazy maximum they stay below 2^15.
template <typename T>
constexpr float kProbLog2 = std::is_same<T, _Float16>::value ? 7.0f : 0.0f;

__device__ __forceinline__ float ops_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Elements of padding of an LDS row of D: rows an odd number of 32-byte units
// apart, so that 16 row reads of 16 bytes and the transposed reads spread over the banks.
template <typename T>
constexpr int kPad = sizeof(T) == 2 ? 16 : 8;

// A operand of rows row0 + li, columns 32 dc + 8g (LD: elements per LDS row).
template <typename T, int LD>
__device__ __forceinline__ typename Mma<T>::v8 row_op(const T* tile, int row0, int dc, int g, int li) {
    return *reinterpret_cast<const typename Mma<T>::v8*>(tile + (row0 + li) * LD + 32 * dc + 8 * g);
}

// A operand of the transposed tile: row li is column col0 + li, and its elements are the rows
// row0 + 4g + e (e < 4) and row0 + 16 + 4g + e - 4: the rows whose C registers
// of two 16-row blocks a lane holds.  16-bit types by the transposing LDS read: in a
// group of 16 lanes, lane i gets element i % 4 of what lane 4r + i / 4 addresses.
template <typename T, int LD>
__device__ __forceinline__ typename Mma<T>::v8 col_op(const T* tile, int row0, int col0, int g, int li) {
    if constexpr (sizeof(T) == 2) {
        typedef __attribute__((address_space(3))) s16x4* lds4;
        const T* a = tile + (row0 + 4 * g + (li >> 2)) * LD + col0 + 4 * (li & 3);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4) const_cast<T*>(a));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4) const_cast<T*>(a + 16 * LD));
        return __builtin_bit_cast(typename Mma<T>::v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
        typename Mma<T>::v8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = tile[(row0 + (e < 4 ? 0 : 12) + 4 * g + e) * LD + col0 + li];
        return v;
    }
}

// Rows row0 + li of a matrix in global memory as an operand: columns 32 dc + 8g.
// Zero outside [0, rows) x [0, d).
template <typename T>
__device__ __forceinline__ typename Mma<T>::v8 global_row(const T* base, int64_t stride, int row, int rows, int col,
                                                          int d, bool vec) {
    typename Mma<T>::v8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = T(0.0f);
    if (row < rows && col < d) {
        const T* p = base + row * stride + col;
        if (vec) {
            v = *reinterpret_cast<const typename Mma<T>::v8*>(p);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (col + e < d) v[e] = p[e];
        }
    }
    return v;
}

// The C layout's four consecutive columns of one row, to global memory.
template <typename T>
__device__ __forceinline__ void store4(T* row, int col, int d, bool wide, f32x4 x) {
    typename Mma<T>::v4 y;
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = T(x[r]);
    if (wide && col + 4 <= d) {
        *reinterpret_cast<typename Mma<T>::v4*>(row + col) = y;
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (col + r < d) row[col + r] = y[r];
    }
}

// Max / sum over the four lanes (g = 0 .. 3) that hold a row of C^T.
__device__ __forceinline__ float row4_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float row4_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// log2(e) * softcap * tanh(scale x / softcap); t: the tanh.
// 16-bit: 1 - 2 / (e^2y + 1), within 2e-7 absolutely.  f32 takes the library's tanh,
// whose relative error is small also near 0.
template <typename T>
__device__ __forceinline__ float capped(float x, float cap_in, float cap_log2e, float* t) {
    if constexpr (sizeof(T) == 2) {
        *t = 1.0f - 2.0f * __builtin_amdgcn_rcpf(ops_exp2(x * cap_in) + 1.0f);
    } else {
        *t = tanhf(x * (cap_in * (0.5f * kLn2)));
    }
    return cap_log2e * *t;
}

__device__ __forceinline__ bool not_finite(float x) {
    return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u;
}

template <typename T>
__device__ __forceinline__ bool any_not_finite(typename Mma<T>::v8 v) {
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) bad = bad || not_finite(float(v[e]));
    return bad;
}

// LDS reads do not move over this, nor are their values kept in registers for a second use.
__device__ __forceinline__ void reread() { asm volatile("" ::: "memory"); }

// acc[j] += op(i, j) * w[i] over the 32-row chunks i, where a weight of exactly 0
// means "not seen": operand values of rows that are not seen must not reach the
// sum, not even as 0 * inf.  Used on tiles with hidden pairs.  Values are
// nearly always finite: that is checked first, and the plain product taken.  Otherwise the
// finite values are summed, and infinities and NaN looked for among the seen ones,
// one kind after another.
template <typename T, int NB, int NCH, typename Op>
__device__ __forceinline__ void mma_seen(f32x4 (&acc)[NB], const typename Mma<T>::v8 (&w)[NCH], Op op) {
    using v8 = typename Mma<T>::v8;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            bad = bad || any_not_finite<T>(op(i, j));
            reread();
        }
    if (__builtin_amdgcn_ballot_w64(bad) == 0) {
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                acc[j] = Mma<T>::mma(op(i, j), w[i], acc[j]);
                reread();
            }
        return;
    }
    for (int kind = 0; kind < 4; ++kind) {   // finite, +inf, -inf, NaN
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            f32x4 sum = kind == 0 ? acc[j] : (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
            f32x4 neg = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                reread();
                v8 a = op(i, j), b = w[i], c = w[i];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = float(a[e]), y = float(w[i][e]);
                    if (kind == 0) {
                        if (not_finite(x)) a[e] = T(0.0f);
                    } else {
                        const bool hit = kind == 3 ? x != x : x == (kind == 1 ? 1.0f : -1.0f) * __builtin_huge_valf();
                        a[e] = T(hit ? 1.0f : 0.0f);
                        b[e] = T(y > 0.0f ? 1.0f : 0.0f);   // infinities keep the weight's sign
                        c[e] = T(y < 0.0f ? 1.0f : 0.0f);
                    }
                }
                sum = Mma<T>::mma(a, b, sum);
                if (kind != 0) neg = Mma<T>::mma(a, c, neg);
            }
            if (kind == 0) {
                acc[j] = sum;
            } else {
                const float special = kind == 1   ? __builtin_huge_valf()
                                      : kind == 2 ? -__builtin_huge_valf()
                                                  : __builtin_nanf("");
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (sum[r] > 0.0f) acc[j][r] += special;
                    if (neg[r] > 0.0f) acc[j][r] -= special;
                }
            }
        }
    }
}

// Visibility of key j to the query at position pos (score attention).
struct ScoreMask {
    int causal, prefix, sk;
    __device__ __forceinline__ bool seen(int key, int pos) const {
        return key < sk && (!causal || key <= pos || key < prefix);
    }
};

#endif  // FA_OPS_COMMON_H
