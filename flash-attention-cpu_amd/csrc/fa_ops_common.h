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

extern "C" __global__ void OPS_STAMP_KERNEL() {}

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

// Kernels of calls with a sliding window are code objects of their own (the same sources built with OPS_WINDOW): what
// they need besides would take scalar registers from the others.
#ifdef OPS_WINDOW
constexpr bool kWindow = true;
#else
constexpr bool kWindow = false;
#endif

// What happens to scores, fixed for a kernel: bits kCap and kBias, or kAny: looked up in the parameters.
constexpr int kCap = 1, kBias = 2, kAny = 4;
template <int MOD, typename P>
__device__ __forceinline__ bool has_cap(const P& p) {
    return MOD == kAny ? p.cap_log2e != 0.0f : (MOD & kCap) != 0;
}
template <int MOD, typename P>
__device__ __forceinline__ bool has_bias(const P& p) {
    return MOD == kAny ? p.slopes != nullptr : (MOD & kBias) != 0;
}

// The kernel's parameters, read again where this stands: code that runs seldom (masked tiles, the
// stores at the end) uses these, so that what only it needs does not occupy scalar
// registers in the main loop.
template <typename P>
__device__ __forceinline__ P late_params() {
    auto k = (const __attribute__((address_space(4))) char*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(k));
    P p;
    __builtin_memcpy(&p, (const char*)k, sizeof(P));
    return p;
}

// A scalar load of what all lanes want: a vector load would come back only after all of the
// wave's DMA.
template <typename V>
__device__ __forceinline__ V load_uniform(const V* p) {
    return *(const __attribute__((address_space(4))) V*)p;
}

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

// Kernels come in two kinds: VEC, where rows are 16-byte aligned and d is a multiple of 8, and
// one that takes any alignment and width element by element.

// Rows row0 + li of a matrix in global memory as an operand: columns 32 dc + 8g.
// Zero outside [0, rows) x [0, d).
template <typename T, bool VEC>
__device__ __forceinline__ typename Mma<T>::v8 global_row(const T* base, int64_t stride, int row, int rows, int col,
                                                          int d) {
    typename Mma<T>::v8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = T(0.0f);
    if (row < rows && col < d) {
        const T* p = base + row * stride + col;
        if constexpr (VEC) {
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
template <typename T, bool VEC>
__device__ __forceinline__ void store4(T* row, int col, int d, f32x4 x) {
    typename Mma<T>::v4 y;
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = T(x[r]);
    if constexpr (VEC) {
        if (col < d) *reinterpret_cast<typename Mma<T>::v4*>(row + col) = y;
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
// 16-bit: 1 - 2 / (e^2y + 1), within 2e-7 absolutely, so the score is within 2e-7 of the cap: enough up to
// kFastCap.  f32, and 16-bit types with larger caps, take the library's tanh, whose relative error is small
// also near 0; the latter in the kernels of any alignment only (kAny), where the host sends them.
template <typename T, int MOD>
__device__ __forceinline__ bool fast_cap(float cap_log2e) {
    return sizeof(T) == 2 && (MOD != kAny || cap_log2e <= kFastCap * kLog2e);
}
template <typename T, int MOD>
__device__ __forceinline__ f32x4 capped(f32x4 x, float cap_in, float cap_log2e, f32x4* t) {
    if (fast_cap<T, MOD>(cap_log2e)) {
#pragma unroll
        for (int r = 0; r < 4; ++r) (*t)[r] = 1.0f - 2.0f * __builtin_amdgcn_rcpf(ops_exp2(x[r] * cap_in) + 1.0f);
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) (*t)[r] = tanhf(x[r] * (cap_in * (0.5f * kLn2)));
    }
    return *t * cap_log2e;
}

// The same less ref, where the tanh itself is not wanted.
template <typename T, int MOD>
__device__ __forceinline__ f32x4 capped_over(f32x4 x, float cap_in, float cap_log2e, float ref) {
    if (fast_cap<T, MOD>(cap_log2e)) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            x[r] = __builtin_fmaf(-2.0f * cap_log2e, __builtin_amdgcn_rcpf(ops_exp2(x[r] * cap_in) + 1.0f), cap_log2e - ref);
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = cap_log2e * tanhf(x[r] * (cap_in * (0.5f * kLn2))) - ref;
    }
    return x;
}

__device__ __forceinline__ bool not_finite(float x) {
    return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u;
}

// LDS reads do not move over this, nor are their values kept in registers for a second use.
__device__ __forceinline__ void reread() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Tiles that hold hidden pairs: a hidden pair has the weight 0, and values of rows that a
// query does not see must not reach its sum, not even as 0 * inf.  So before
// such a tile is multiplied, its infinities and NaN are replaced by zeros in LDS; where there
// were any, the kernel adds them once its sums are written, to the rows that see them.

// Whether a chunk of 16 bytes holds an infinity or NaN.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ bool chunk_special(u32x4 u) {
    if constexpr (sizeof(T) == 2) {
        // half words: magnitude + (2^15 - infinity) reaches 2^15 where not finite
        constexpr unsigned kAdd = (0x8000u - (std::is_same<T, __bf16>::value ? 0x7f80u : 0x7c00u)) * 0x10001u;
        unsigned any = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) any |= (u[e] & 0x7fff7fffu) + kAdd;
        return (any & 0x80008000u) != 0;
    } else {
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) bad = bad || (u[e] & 0x7f800000u) == 0x7f800000u;
        return bad;
    }
}
template <typename T>
__device__ __forceinline__ void clean_chunk(T* at) {
#pragma unroll 1
    for (int e = 0; e < 16 / (int)sizeof(T); ++e)
        if (not_finite(float(at[e]))) at[e] = T(0.0f);
}

// Cleans ROWS rows of D elements (LD apart), NT threads; returns whether the thread found something.
template <typename T, int LD, int D, int ROWS, int NT>
__device__ __forceinline__ bool tile_clean(T* tile, int tid) {
    constexpr int E = 16 / (int)sizeof(T), CPR = D / E;
    bool found = false;
#pragma unroll 1
    for (int pos = tid; pos < ROWS * CPR; pos += NT) {
        T* const at = tile + pos / CPR * LD + E * (pos % CPR);
        if (chunk_special<T>(*reinterpret_cast<const u32x4*>(at))) {
            found = true;
            clean_chunk<T>(at);
        }
    }
    return found;
}

// Adds what tile_clean took out: rows [from, to) of src (a row's address: at(row), nullptr: none) that hold
// infinities or NaN, to the rows r < n of the wave that see them.  POSITIVE weights: as they are, else as NaN.
template <typename T, typename O, bool POSITIVE, typename At, typename See, typename Out>
__device__ __forceinline__ void add_specials(int from, int to, int n, int d, int lane, At at, See see, Out out) {
#pragma unroll 1
    for (int row = from; row < to; ++row) {
        const T* x = at(row);
        if (!x) continue;
#pragma unroll 1
        for (int c = lane; c - lane < d; c += 64) {
            const float y = c < d ? float(x[c]) : 0.0f;
            if (__builtin_amdgcn_ballot_w64(not_finite(y)) == 0) continue;
#pragma unroll 1
            for (int r = 0; r < n; ++r) {
                if (!see(row, r)) continue;
                O* to_ = out(r);
                if (not_finite(y)) to_[c] = O(POSITIVE ? float(to_[c]) + y : __builtin_nanf(""));
            }
        }
    }
}

// N elements of LDS, one array per (N, ID) in a kernel: distinct arrays, so that the
// compiler sees that a DMA into one does not change what is read from another.
template <typename T, int N, int ID>
__device__ __forceinline__ T* lds_array() {
    __shared__ __attribute__((aligned(16))) T buf[N];
    return buf;
}

// The calling wave's outstanding loads and DMA have arrived.
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// Fills ROWS x D tiles (rows of LD elements) from a matrix in global memory, zero
// outside [0, rows) x [0, d): by DMA, lane L of run R = i NW + wave at 16-byte chunk 64 R + L of the
// tile's image (pad chunks included) with offsets fixed for the whole kernel -- the buffer's range ends at the
// last row, and lanes past it, past column d or in the pad read zeros --
// or, where rows are not 16-byte aligned, element by element.
template <typename T, int D, int ROWS, int NW, bool VEC>
struct TileFill {
    static constexpr int LD = D + kPad<T>, E = 16 / (int)sizeof(T), RCH = LD / E;
    static constexpr int TOTAL = ROWS * RCH, RUNS = (TOTAL + 63) / 64, NI = (RUNS + NW - 1) / NW;
    static constexpr int SIZE = RUNS * 64 * E;   // elements of a tile's buffer: whole runs
    int voff[NI];
    int wave, lane, d;
    int64_t stride;
    __device__ __forceinline__ TileFill(int64_t stride_, int d_, int wave_, int lane_)
        : wave(wave_), lane(lane_), d(d_), stride(stride_) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int pos = (i * NW + wave) * 64 + lane, r = pos / RCH, col = pos % RCH * E;
            voff[i] = pos < TOTAL && col < d ? (int)(r * stride + col) * (int)sizeof(T) : 0x7ffffff0;
        }
    }
    __device__ __forceinline__ void operator()(T* dst, const T* base, int row0, int rows) const {
        const T* src = base + row0 * stride;
        if constexpr (VEC) {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<T*>(src), (short)0, (int)(min(ROWS, rows - row0) * stride) * (int)sizeof(T), 0x00020000);
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int run = i * NW + wave;
                if ((i + 1) * NW <= RUNS || run < RUNS)
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(
                        rs, (__attribute__((address_space(3))) void*)(dst + run * 64 * E), 16, voff[i], 0, 0, 0);
            }
        } else {
#pragma unroll 1
            for (int pos = wave * 64 + lane; pos < ROWS * (D / 8); pos += 64 * NW) {
                const int r = pos / (D / 8), col = 8 * (pos % (D / 8));
                *reinterpret_cast<typename Mma<T>::v8*>(dst + r * LD + col) =
                    global_row<T, false>(src, stride, r, rows - row0, col, d);
            }
        }
    }
    // Whether what the lane itself filled, and what has arrived, holds an infinity or NaN; CLEAN: they become zeros.
    template <bool CLEAN>
    __device__ __forceinline__ bool special(T* dst) const {
        bool found = false;
        auto look = [&](T* at) {
            if (chunk_special<T>(*reinterpret_cast<const u32x4*>(at))) {
                found = true;
                if (CLEAN) clean_chunk<T>(at);
            }
        };
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int run = i * NW + wave;
                if ((i + 1) * NW <= RUNS || run < RUNS) look(dst + (run * 64 + lane) * E);
            }
        } else {
#pragma unroll 1
            for (int pos = wave * 64 + lane; pos < ROWS * (D / 8); pos += 64 * NW)
#pragma unroll
                for (int c = 0; c < 8; c += E) look(dst + pos / (D / 8) * LD + 8 * (pos % (D / 8)) + c);
        }
        return found;
    }
};

#endif  // FA_OPS_COMMON_H
