// fa_cache4.hip -- gfx950 kernels of the key / value cache held in 4 bits:
// append, rows read back, and attention of query rows over it (fa_cache4_*).
//
// A row's columns come in groups of 32.  A group has a step S / 16 and an offset O, both f16, and its code c
// stands for the value O + (1 + c / 16) S:  c in the upper bits of the fraction of an f16 in [1, 2) makes that one
// multiply-add of two values, and no subtraction of a constant is needed.
//
// Keys lie in rows of d / 8 words, 8 columns a word; values in words of 8 rows of one column, d such words for the
// 8 rows.  Both are then operands of 16 x 16 x 32 matrix products as they come from memory, a word's eight codes
// being the eight elements that a lane holds, and nothing goes through LDS or is transposed.
// Entry e of a word stands at bits 4 (e / 2) + 16 (e % 2), so that pairs of neighbours leave it together.
//
// Built once a type: OPS_T the type of queries, outputs and rows (16 bits), OPS_NAME its name in the kernels'.

#define ROWS_EVEN
#include "fa_rows.h"

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// A sequence's row among all rows of its head's kind in memory ([blocks, kv_heads, rows]: fewer than 2^32), if there is one.
struct Place {
    unsigned at;
    bool there;
};
__device__ __forceinline__ Place cache4_place(const Cache4Params& p, int b, int h, int64_t row) {
    if (row < 0 || row >= p.capacity) return {0, false};
    const unsigned head = (unsigned)h * (unsigned)p.block_rows, block = (unsigned)p.kv_heads * (unsigned)p.block_rows;
    if (!p.table) return {(unsigned)b * block + head + (unsigned)row, true};
    const int page = p.table[(int64_t)b * p.pages_per_seq + ((int)row >> p.page_shift)];
    if ((unsigned)page >= (unsigned)p.n_pages) return {0, false};
    return {(unsigned)page * block + head + ((unsigned)row & ((1u << p.page_shift) - 1)), true};
}

// The neighbour at lane ^ M, M = 1 or 2
template <int M, typename V>
__device__ __forceinline__ V neighbour(V x) {
    constexpr int kPerm = M == 1 ? 0xb1 : 0x4e;
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kPerm, 0xf, 0xf, true));
}
// a / b, rounded as a division is, from the inverse of b rounded right
__device__ __forceinline__ float divided(float a, float b, float inv) {
    const float q = a * inv;
    return __builtin_fmaf(__builtin_fmaf(-q, b, a), inv, q);
}

__device__ __forceinline__ unsigned half_bits(_Float16 x) { return __builtin_bit_cast(unsigned short, x); }
__device__ __forceinline__ _Float16 bits_half(unsigned x) { return __builtin_bit_cast(_Float16, (unsigned short)x); }

// x / d of numbers below 2^16, d given as its inverse
__device__ __forceinline__ int small_div(int x, float inv) { return (int)(((float)x + 0.5f) * inv); }

// ---------------------------------------------------------------------------
// Append: a workgroup takes a few runs of 8 rows of one head of K or V.  A thread quantises 8 columns of a row, four
// neighbours a group.  Keys are words then; values meet in LDS, where a thread a column makes a word of
// 8 rows, with what is there already of rows that are not new.
// Bound by vector instructions, some 220 for 8 columns: 83 make the group's step and its inverse and the codes (24 of them
// the eight quotients), 54 widen the columns and find the smallest and largest, 51 put words of V together, 44 and a table's
// look-up move the pieces on their way along and find the place of the next: 12 of the 18 us below.  A quotient is the
// group's inverse and one correction, which rounds it as a division does: the inverse of an 11-bit number is rounded
// right by one step from the approximate one, since it lies no nearer than 2^-36 to the middle of two f32 numbers, and from
// a right inverse the corrected quotient is right.  4 x 2048 rows of K and V, 8 heads of 128 columns, bf16: 18 us (34 MB
// read, 10 MB written: 2.4 TB/s).
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void cache4_append(const Cache4Params& p) {
    __shared__ __attribute__((aligned(16))) unsigned char codes[256 * 8];   // [run][8 rows][d]
    __shared__ int fresh[8];       // rows of a run that are new
    __shared__ unsigned where[8];   // and its place among the runs in memory
    typedef T run8 __attribute__((ext_vector_type(8)));
    const int tid = threadIdx.x, words = p.d / 8, per = 256 / p.d;   // runs of 8 rows a workgroup
    const float inv_d = 1.0f / (float)p.d, inv_words = 1.0f / (float)words;
    unsigned id = blockIdx.x;
    const int part = id % p.nparts;
    id /= p.nparts;
    const int h = id % p.kv_heads;
    id /= p.kv_heads;
    const bool isv = id & 1;
    const int b = id >> 1;
    const int len = p.lens[b];
    if (len < 0) return;
    const T* const src = reinterpret_cast<const T*>(isv ? p.v : p.k) + (isv ? b * p.vs.b + h * p.vs.h : b * p.ks.b + h * p.ks.h);
    const int64_t seq = isv ? p.vs.s : p.ks.s;
    const bool mine = tid < per * p.d;
    const int run = small_div(tid, inv_d), col = tid - run * p.d, r = small_div(col, inv_words), word = col - r * words;
    const int groups = words / 4;

    // what a thread takes of the workgroup's u-th few runs: its place in the cache, and its columns
    struct Piece {
        Place at;
        run8 y;
    };
    auto first_of = [&](int u) { return len / 8 + ((int64_t)part * p.loops + u) * per; };
    auto fetch = [&](Piece& x, int u) {
        const int64_t row = (first_of(u) + run) * 8 + r, token = row - len;
        x.at = {0, false};
        x.y = run8{};
        if (mine && token >= 0 && token < p.n) {
            x.at = cache4_place(p, b, h, row);
            const T* const from = src + token * seq + 8 * word;
            if (p.vec) {
                x.y = *reinterpret_cast<const run8*>(from);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x.y[e] = from[e];
            }
        }
    };
    auto keep = [&](const Piece& piece, int u) {
        const Place at = piece.at;
        float x[8], lo = INFINITY, hi = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = float(piece.y[e]);
            lo = fminf(lo, x[e]);
            hi = fmaxf(hi, x[e]);
        }
        int bad = chunk_special<T>(__builtin_bit_cast(u32x4, piece.y));
        lo = fminf(lo, neighbour<1>(lo));
        hi = fmaxf(hi, neighbour<1>(hi));
        bad |= neighbour<1>(bad);
        lo = fminf(lo, neighbour<2>(lo));
        hi = fmaxf(hi, neighbour<2>(hi));
        bad |= neighbour<2>(bad);
        if (__builtin_amdgcn_ballot_w64(lo < -kCache4Max || hi > kCache4Max) != 0) {
            lo = __builtin_amdgcn_fmed3f(lo, -kCache4Max, kCache4Max);
            hi = __builtin_amdgcn_fmed3f(hi, -kCache4Max, kCache4Max);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __builtin_amdgcn_fmed3f(x[e], -kCache4Max, kCache4Max);
        }
        // as the header defines them, each operation rounded once
        constexpr float kTop = 65504.0f;
        const float size = fminf(divided((hi - lo) * 16.0f, 15.0f, 1.0f / 15.0f), kTop);
        const _Float16 big = bad ? bits_half(0x7e00) : _Float16(size);
        const _Float16 off = bad ? bits_half(0x7e00) : _Float16(fmaxf(lo - float(big), -kTop));
        const float o = bad ? 0.0f : float(off), step = bad ? 0.0f : float(big) * 0.0625f;
        const float near = __builtin_amdgcn_rcpf(step);
        // (no step: an inverse of 0 gives codes of 0)
        const float inv = step == 0.0f ? 0.0f : __builtin_fmaf(__builtin_fmaf(-near, step, 1.0f), near, near);
        // Codes plus 16 as bytes, rounded to even: entries 0, 4, 1, 5 of the word's, and 2, 6, 3, 7.
        unsigned even = 0, odd = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float z = __builtin_amdgcn_fmed3f(divided(x[e] - o, step, inv), 16.0f, 31.0f);
            unsigned& to = e / 2 % 2 == 0 ? even : odd;
            to = __builtin_amdgcn_cvt_pk_u8_f32(z, e / 4 + 2 * (e % 2), to);
        }
        even &= 0x0f0f0f0fu;
        odd &= 0x0f0f0f0fu;
        if (!isv) {
            if (!at.there) return;
            p.k4[(uint64_t)at.at * (unsigned)words + (unsigned)word] = even | odd << 4;
            if (word % 4 == 0)
                reinterpret_cast<unsigned*>(p.kscale)[(uint64_t)at.at * (unsigned)groups + (unsigned)word / 4] =
                    half_bits(big) | half_bits(off) << 16;
            return;
        }
        __syncthreads();
        if (tid < per) fresh[tid] = 0;
        __syncthreads();
        if (at.there) {
            if (word == 0) {
                atomicOr(&fresh[run], 1 << r);
                where[run] = at.at >> 3;   // (all rows of a run lie in one page)
            }
            *reinterpret_cast<u32x2*>(codes + (run * 8 + r) * p.d + 8 * word) = (u32x2){even, odd};
            if (word % 4 == 0) {
                unsigned short* const s = p.vscale + ((uint64_t)(at.at >> 3) * (unsigned)groups + (unsigned)word / 4) * 16 + r;
                s[0] = half_bits(big);
                s[8] = half_bits(off);
            }
        }
        __syncthreads();
        const int have = mine ? fresh[run] : 0;
        if (have == 0) return;
        const int byte = (col & ~7) + (col / 2 % 2) * 4 + (col / 4 % 2) + 2 * (col % 2);   // of the column's codes
        unsigned* const word8 = p.v4 + (uint64_t)where[run] * (unsigned)p.d + (unsigned)col;
        unsigned w = have == 0xff ? 0u : *word8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int sh = 4 * (e / 2) + 16 * (e % 2);
            const unsigned c = (unsigned)codes[(run * 8 + e) * p.d + byte] << sh, keep = ~(15u << sh);
            if (have >> e & 1) w = (w & keep) | c;
        }
        *word8 = w;
    };
    // three pieces on their way while one is worked on
    Piece now, second, third, last;
    fetch(now, 0);
    if (p.loops > 1) fetch(second, 1);
    if (p.loops > 2) fetch(third, 2);
    for (int u = 0; u < p.loops; ++u) {
        if (u + 3 < p.loops) fetch(last, u + 3);
        keep(now, u);
        now = second;
        second = third;
        third = last;
    }
}

// Rows of the cache in the type: 8 columns of a row a thread, a head of K or V a workgroup.  Bound by memory and the
// launch: 4 x 2048 rows of K and V, 8 heads of 128 columns, bf16: 12 us (10 MB read, 34 MB written: 3.6 TB/s).  A thread
// takes four rows, whose loads are under way together.
template <typename T>
__device__ __forceinline__ void cache4_read(const Cache4Params& p) {
    typedef T run8 __attribute__((ext_vector_type(8)));
    const int tid = threadIdx.x, words = p.d / 8, groups = p.d / 32, per = 256 / words;   // rows a workgroup
    unsigned id = blockIdx.x;
    const int part = id % p.nparts;
    id /= p.nparts;
    const int h = id % p.kv_heads;
    id /= p.kv_heads;
    const bool isv = id & 1;
    const int b = id >> 1;
    const int r = small_div(tid, 1.0f / (float)words), word = tid - r * words;
    if (r >= per || !(isv ? p.vo : p.ko)) return;
    constexpr int N = kCache4ReadRows;   // rows of a thread, whose loads overlap
    const int64_t i0 = (int64_t)part * per * N + r;
    Place at[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int64_t i = i0 + u * per;
        at[u] = i < p.n ? cache4_place(p, b, h, p.rows[(int64_t)b * p.n + i]) : Place{0, false};
    }
    u32x4 w[N][2];
    unsigned sc[N];   // S and O
#pragma unroll
    for (int u = 0; u < N; ++u) {
        w[u][0] = w[u][1] = (u32x4){0, 0, 0, 0};
        sc[u] = 0;
        if (!at[u].there) continue;
        if (!isv) {
            w[u][0][0] = p.k4[(uint64_t)at[u].at * (unsigned)words + (unsigned)word];
            sc[u] = reinterpret_cast<const unsigned*>(p.kscale)[(uint64_t)at[u].at * (unsigned)groups + (unsigned)word / 4];
        } else {
            const unsigned run = at[u].at >> 3;
            const unsigned short* const s =
                p.vscale + ((uint64_t)run * (unsigned)groups + (unsigned)word / 4) * 16 + (at[u].at & 7);
            sc[u] = s[0] | (unsigned)s[8] << 16;
            const u32x4* const from = reinterpret_cast<const u32x4*>(p.v4 + (uint64_t)run * (unsigned)p.d + 8 * word);
            w[u][0] = from[0];
            w[u][1] = from[1];
        }
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int64_t i = i0 + u * per;
        if (i >= p.n) break;
        const float big = float(bits_half(sc[u] & 0xffff)), off = float(bits_half(sc[u] >> 16));
        const int e8 = at[u].at & 7, sh = 4 * (e8 / 2) + 16 * (e8 % 2);
        run8 y;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const unsigned c = isv ? w[u][e / 4][e % 4] >> sh : w[u][0][0] >> (4 * (e / 2) + 16 * (e % 2));
            // (no such row: 0)
            y[e] = T(__builtin_fmaf(1.0f + (float)(c & 15) * 0.0625f, big, off));
        }
        T* const to = reinterpret_cast<T*>(isv ? p.vo : p.ko) +
                      (isv ? b * p.vs.b + h * p.vs.h + i * p.vs.s : b * p.ks.b + h * p.ks.h + i * p.ks.s) + 8 * word;
        if (p.vec) {
            *reinterpret_cast<run8*>(to) = y;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) to[e] = y[e];
        }
    }
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
// Eight values of a word: codes to the fraction of f16 numbers in [1, 2), times S, plus O.  big(i), off(i): those of
// pair i.  A value is rounded to f16's 11 bits (from a multiply-add in one step), as the weights of values are.  Half a
// step of a code is 1 / 30 of its group's range, that rounding 2^-11 of the value: 136 times less or better where a
// group's values lie around zero, but more than half a step where they lie over 68 ranges from it.  Values in f32 would
// take the matrix product at a sixteenth of the rate; the codes themselves as an operand, with S and O applied to the sums
// of every group of columns, would take 8 vector instructions a group of 16 keys and query tile instead of 4, and values and
// weights in two f16 parts each 15 to 20 % of the time.  Rows of f16 are off by 4.0e-4 of their size (2.9e-4 in two parts),
// of which the rounding of the output alone is 2.1e-4; rows of bf16 by 1.7e-3, all of it the output's.
template <typename B, typename O>
__device__ __forceinline__ h8 dequant(unsigned w, unsigned one, B big, O off) {
    h8 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        unsigned bits = 4 * i < 6 ? w << (6 - 4 * i) : w >> (4 * i - 6);
        // (bits & mask) | one: the compiler makes two instructions of it, since it takes both constants for literals
        asm("v_and_or_b32 %0, %0, %1, %2" : "+v"(bits) : "s"(0x03c003c0u), "v"(one));
        const h2 t = __builtin_bit_cast(h2, bits);
        const h2 y = __builtin_elementwise_fma(t, big(i), off(i));
        v[2 * i] = y[0];
        v[2 * i + 1] = y[1];
    }
    return v;
}

// A row's token: its number, position and first mask word.  (The following are what RowTiles of fa_cache.hip has as members,
// for trees alone; its kernels take 3 % longer through functions like these: 176 us instead of 171 for 8 trees of 64
// tokens over up to 16384 rows.)
struct RowToken {
    int token, pos;
    uint64_t word;
};
__device__ __forceinline__ RowToken row_token(const RowsParams& p, const RowsWork& w, int token) {
    const int64_t at = (int64_t)w.b * p.n + token;
    return {token, p.pos ? p.pos[at] : w.len + token,
            p.mask ? p.mask[(p.mask_shared ? token : at) * p.mask_words] : bits_before(token + 1)};
}
__device__ __forceinline__ uint64_t mask_word(const RowsParams& p, const RowsWork& w, const RowToken& r, int i) {
    if (i == 0) return r.word;
    if (i >= p.mask_words) return 0;
    if (p.mask) return p.mask[((p.mask_shared ? 0 : (int64_t)w.b * p.n) + r.token) * p.mask_words + i];
    return bits_before(r.token + 1 - 64 * i);   // a chain
}
// Bits of the keys from k0 that the row sees, as far as the tree tells.
__device__ __forceinline__ uint64_t seen_bits(const RowsParams& p, const RowsWork& w, const RowToken& r, int k0) {
    const int rel = k0 - w.len;   // the first key's number among the drafted ones
    if (rel <= -64) return ~0ull;
    if (rel < 0) return (mask_word(p, w, r, 0) << -rel) | ((1ull << -rel) - 1);
    const int i = rel >> 6, sh = rel & 63;
    const uint64_t lo = mask_word(p, w, r, i) >> sh;
    return sh == 0 ? lo : lo | (mask_word(p, w, r, i + 1) << (64 - sh));
}
// Bits of the 32 keys from k0 that exist: before the run's end, in good pages (one lane a key).
__device__ __forceinline__ uint64_t keys_there(const RowsParams& p, const RowsWork& w, int k0, int lane, int badpage) {
    if (!badpage) return bits_before(w.kend - k0);
    const CachePages pages = rows_pages(p, w.b);
    return __builtin_amdgcn_ballot_w64(k0 + lane < w.kend && pages.at(k0 + lane, w.kend, 0, 0) >= 0);
}

template <int N>
struct Words {
    unsigned w[N];
};
// N words at a byte offset of a buffer (zeros past its end)
template <int N>
__device__ __forceinline__ Words<N> buffer_words(__amdgpu_buffer_rsrc_t rs, int at) {
    Words<N> r;
    if constexpr (N == 4) {
        const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rs, at, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = x[i];
    } else if constexpr (N == 2) {
        const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(rs, at, 0, 0);
        r.w[0] = x[0];
        r.w[1] = x[1];
    } else {
        r.w[0] = __builtin_amdgcn_raw_buffer_load_b32(rs, at, 0, 0);
    }
    return r;
}

// The matrix product over f16, whose other operands are the values that codes stand for.
using M4 = Mma<_Float16>;

// Waves walk blocks of 32 keys of their own, two blocks in registers or on their way while one is used.  MT 16-row
// tiles of queries; SMALL: pages of less than 32 rows, whose rows are found lane by lane.
// A lane (g = l / 16, li = l % 16) has of K the rows 8 (li / 4) + 4 b + li % 4, b < 2, of a block, so that the scores
// it gets are those of keys 8 g .. 8 g + 7, the eight rows of a word of V.
//
// Bound by vector instructions: a block of 32 keys of 128 columns takes some 290 a wave, most of them to make values of codes (12
// for 8 of them), so 16 rows of queries cost as much as one, and a second tile of them little.  bf16, 8 x 32 / 8
// heads, one token over up to 32768 rows: 51 us, 5.2 TB/s of the cache's bytes (a cache of 16 bits holds 3.2 times as many),
// with the vector units busy two thirds of the time and three waves a SIMD (two: 5 us more).  Few rows (f16, 4 x 25
// tokens of 16 / 2 heads over 3000 rows, 20 us) are a chain of first loads, a few blocks a wave and the join in LDS.
template <typename T, int NDC, int MT, int MOD, bool SMALL>
__device__ __forceinline__ void rows4(const RowsParams& p) {
    constexpr int NW = kRows4Waves, SK = 32, D = 32 * NDC;
    constexpr int KW = NDC % 4 == 0 ? 4 : NDC % 2 == 0 ? 2 : 1, NK = NDC / KW;   // words of a load of K, and loads a row
    constexpr int VW = NDC % 2 == 0 ? 4 : 2, NV = D / (16 * VW);                  // columns of a load of V, and loads
    constexpr int NO = D / 16, PD = D <= 64 ? 64 : D <= 128 ? 128 : 256;          // PD: a row of partial sums
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, li = lane & 15;
    RowsWork w;
    if (!rows_work(p, 16 * MT, lane, &w)) return;
    const CachePages pages = rows_pages(p, w.b);
    const int page_rows = p.block4;   // rows of a block of memory
    const unsigned* const K = reinterpret_cast<const unsigned*>(p.k);
    const unsigned* const KS = reinterpret_cast<const unsigned*>(p.k_scale);
    const unsigned* const V = reinterpret_cast<const unsigned*>(p.v);
    const unsigned* const VS = reinterpret_cast<const unsigned*>(p.v_scale);
    const int nblk = SK * wave < w.kwalk() ? (w.kwalk() - SK * wave + SK * NW - 1) / (SK * NW) : 0;
    auto key_of = [&](int i) { return w.key(SK * wave + i * SK * NW); };   // first key of the wave's i-th block

    // byte offsets of the lane's loads in a block of 32 rows
    int kat[2], kpat[2], vat, vpat;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int row = 8 * (li >> 2) + 4 * b + (li & 3);
        kat[b] = row * (D / 2) + g * 4 * KW;
        kpat[b] = row * NDC * 4 + (g * KW / 4) * 4;
    }
    vat = g * D * 4 + li * 4 * VW;
    vpat = g * NDC * 32 + (VW == 4 ? (li >> 3) * 32 : 0);
    struct Block {
        Words<KW> k[2][NK];
        unsigned ks[2][NK];
        Words<VW> v[NV];
        Words<4> big[NV], off[NV];
    };
    // the page of a block of 32 keys (0 without pages; SMALL: of each of its runs of 8), -1: bad or past the end
    struct Pages {
        int p[SMALL ? 4 : 1];
    };
    auto look_up = [&](int i) {
        Pages r;
#pragma unroll
        for (int e = 0; e < (SMALL ? 4 : 1); ++e) {
            r.p[e] = -1;
            if (i < nblk && key_of(i) + 8 * e < w.kend) r.p[e] = pages.page(key_of(i) + 8 * e);
        }
        return r;
    };
    auto any_bad = [&](const Pages& pg, int k0) {
        int bad = 0;
#pragma unroll
        for (int e = 0; e < (SMALL ? 4 : 1); ++e) bad |= pg.p[e] < 0 && k0 + 8 * e < w.kend;
        return bad;
    };
    // Of a block of 32 keys: the rows before it in memory, and those that are there.
    struct Source {
        int64_t at;
        int n;
    };
    const int64_t head_rows = ((int64_t)(p.table ? 0 : w.b) * p.kv_heads + w.hk) * page_rows;
    const int64_t page_stride = (int64_t)p.kv_heads * page_rows;
    auto source = [&](int i, int page) -> Source {
        if (page < 0 || i >= nblk) return {0, 0};
        const int k0 = key_of(i);
        return {head_rows + (p.table ? page * page_stride + (k0 & pages.page_mask) : (int64_t)k0), min(SK, w.kend - k0)};
    };
    auto buffer = [&](const unsigned* base, int64_t word, int words) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned*>(base + word), (short)0, 4 * words, 0x00020000);
    };
    // SMALL: the rows before row `row` of its head, in run `run` of 8 of the block, where it is one
    auto lane_rows = [&](const Pages& pg, int row, int run, bool* real) -> int64_t {
        int page = pg.p[0];
        if constexpr (SMALL) page = run == 0 ? pg.p[0] : run == 1 ? pg.p[1] : run == 2 ? pg.p[2] : pg.p[3];
        *real = page >= 0 && row < w.kend;
        return head_rows + page * page_stride + (row & pages.page_mask);
    };
    auto load_k = [&](Block& x, int i, const Source& src, const Pages& pg) {
        if constexpr (SMALL) {
            const int k0 = key_of(i);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                bool real;
                const int64_t at = lane_rows(pg, k0 + 8 * (li >> 2) + 4 * b + (li & 3), li >> 2, &real);
#pragma unroll
                for (int q = 0; q < NK; ++q) {
                    x.k[b][q] = {};
                    x.ks[b][q] = 0;
                    if (!real) continue;
#pragma unroll
                    for (int e = 0; e < KW; ++e) x.k[b][q].w[e] = K[at * (D / 8) + q * 4 * KW + g * KW + e];
                    x.ks[b][q] = KS[at * NDC + q * KW + g * KW / 4];
                }
            }
        } else {
            const int n = src.n;
            const __amdgpu_buffer_rsrc_t rk = buffer(K, src.at * (D / 8), n * (D / 8)), rs = buffer(KS, src.at * NDC, n * NDC);
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int q = 0; q < NK; ++q) {
                    x.k[b][q] = buffer_words<KW>(rk, kat[b] + q * 16 * KW);
                    x.ks[b][q] = buffer_words<1>(rs, kpat[b] + q * 4 * KW).w[0];
                }
        }
    };
    auto load_v = [&](Block& x, int i, const Source& src, const Pages& pg) {
        if constexpr (SMALL) {
            const int k0 = key_of(i);
            bool real;
            const int64_t at = lane_rows(pg, k0 + 8 * g, g, &real) >> 3;
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                x.v[q] = {};
                x.big[q] = x.off[q] = {};
                if (!real) continue;
#pragma unroll
                for (int e = 0; e < VW; ++e) x.v[q].w[e] = V[at * D + q * 16 * VW + li * VW + e];
                const unsigned* const s = VS + (at * NDC + (q * 16 + li) * VW / 32) * 8;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x.big[q].w[e] = s[e];
                    x.off[q].w[e] = s[4 + e];
                }
            }
        } else {
            const int n = (src.n + 7) >> 3;   // runs of 8 rows
            const int64_t at = src.at >> 3;
            const __amdgpu_buffer_rsrc_t rv = buffer(V, at * D, n * D), rs = buffer(VS, at * NDC * 8, n * NDC * 8);
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                x.v[q] = buffer_words<VW>(rv, vat + q * 64 * VW);
                x.big[q] = buffer_words<4>(rs, vpat + q * 16 * VW);
                x.off[q] = buffer_words<4>(rs, vpat + q * 16 * VW + 16);
            }
        }
    };

    Block A, B;
    Pages page2 = look_up(0);
    int bad0 = any_bad(page2, key_of(0));   // of the block to work on, and of the next
    load_k(A, 0, source(0, page2.p[0]), page2);
    load_v(A, 0, source(0, page2.p[0]), page2);
    page2 = look_up(1);
    int bad1 = any_bad(page2, key_of(1));
    load_k(B, 1, source(1, page2.p[0]), page2);
    load_v(B, 1, source(1, page2.p[0]), page2);
    page2 = look_up(2);

    // Queries as f16.  bf16 rows are brought into its range by a power of two, exactly but for entries 2^29 below the
    // row's largest; qs takes it back.
    h8 q[MT][NDC];
    f32x4 o[MT][NO], s[MT][2];
    float m[MT], ref[MT], l[MT], qs[MT], c[MT], slope[MT];
    RowToken tok[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int r = w.rfirst + 16 * t + li;
        const bool real = r < w.nrows;
        const int token = real ? r / p.group : 0, h = w.hk * p.group + (real ? r % p.group : 0);
        tok[t] = row_token(p, w, token);
        slope[t] = has_bias<MOD>(p) ? p.slopes[h] * kLog2e : 0.0f;
        const T* const from = reinterpret_cast<const T*>(p.q) + w.b * p.qs.b + h * p.qs.h + token * p.qs.s;
        typename Mma<T>::v8 x[NDC];
        float mx = 0.0f;
#pragma unroll
        for (int j = 0; j < NDC; ++j) {
            const int col = j / KW * 32 * KW + g * 8 * KW + j % KW * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[j][e] = T(0.0f);
            if (real) {
                if (p.vec4) {
                    x[j] = *reinterpret_cast<const typename Mma<T>::v8*>(from + col);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[j][e] = from[col + e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(float(x[j][e])));
        }
        qs[t] = 1.0f;
        float up = 1.0f;
        if constexpr (std::is_same<T, __bf16>::value) {
            mx = row4_max(mx);
            const unsigned ex = __float_as_uint(mx) >> 23;
            if (ex > 0 && ex < 255) {
                const unsigned e = max(ex, 15u);
                up = __uint_as_float((268u - e) << 23);   // the largest to 2^14 .. 2^15
                qs[t] = __uint_as_float((e - 14u) << 23);
            }
        }
#pragma unroll
        for (int j = 0; j < NDC; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) q[t][j][e] = _Float16(float(x[j][e]) * up);
        // (never 0, which would make NaN of the -inf of keys that a row does not see: scores, below 2^40, are nothing either way)
        c[t] = MOD != 0 ? 1.0f : fmaxf(p.scale_log2e * qs[t], 0x1p-126f);
#pragma unroll
        for (int j = 0; j < NO; ++j) o[t][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        m[t] = OPS_NEG_INF;
        l[t] = ref[t] = 0.0f;
    }
    constexpr float kProb = kProbLog2<_Float16>, kUp = MOD != 0 ? kProb : 0.0f;
    int special = 0;
    const unsigned one = 0x3c003c00u;   // two f16 ones

    auto block = [&](int i, Block& x) {
        const int k0 = key_of(i), bad = bad0;
        const Source next = source(i + 2, page2.p[0]);
        // S^T of the block, relative to the rows' references
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const float r = MOD != 0 ? 0.0f : -ref[t];
            s[t][0] = s[t][1] = (f32x4){r, r, r, r};
        }
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int j = 0; j < KW; ++j)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const h2 so = __builtin_bit_cast(h2, x.ks[b][n]);
                    const h8 k = dequant(x.k[b][n].w[j], one, [&](int) { return (h2){so[0], so[0]}; },
                                         [&](int) { return (h2){so[1], so[1]}; });
#pragma unroll
                    for (int t = 0; t < MT; ++t) s[t][b] = M4::mma(k, q[t][n * KW + j], s[t][b]);
                }
        __builtin_amdgcn_sched_barrier(0);
        load_k(x, i + 2, next, page2);
        const int masked = bad || rows_masked(p, w, k0, SK);
        if constexpr (MOD != 0) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const float dist = (float)(tok[t].pos - k0 - 8 * g);
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    s[t][b] *= qs[t];
                    if (has_cap<MOD>(p)) {
                        s[t][b] = capped_over<_Float16, MOD>(s[t][b], p.cap_in, p.cap_log2e, ref[t] - kUp);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][b][r] = __builtin_fmaf(s[t][b][r], p.scale_log2e, kUp - ref[t]);
                    }
                    if (has_bias<MOD>(p)) {
                        f32x4 y;
#pragma unroll
                        for (int r = 0; r < 4; ++r) y[r] = dist - (float)(4 * b + r);
                        if (masked && p.pos) {
                            // drafted keys stand where the program says
                            const int bit = k0 + 8 * g + 4 * b - w.len;
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (bit + r >= 0)
                                    y[r] = (float)(tok[t].pos - p.pos[w.b * p.n + min(bit + r, p.n - 1)]);
                        }
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][b][r] = __builtin_fmaf(-slope[t], fabsf(y[r]), s[t][b][r]);
                    }
                }
            }
        }
        if (masked) {
            const RowsParams lp = late_params<RowsParams>();
            const uint64_t there = keys_there(lp, w, k0, lane, bad);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                uint64_t see = there & seen_bits(lp, w, tok[t], k0);
                if constexpr (kWindow) see &= window_bits<SK>(lp, w, tok[t].pos, k0, [&](int b, int r) { return 8 * g + 4 * b + r; });
                const unsigned bits = (unsigned)(see >> (8 * g));
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (!(bits & (1u << (4 * b + r)))) s[t][b][r] = OPS_NEG_INF;
            }
            // rows that are not there, or are no numbers, weigh nothing: what those that see them get comes at the end
            const unsigned mine = (unsigned)(there >> (8 * g));
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const unsigned sh = 16 * (e % 2), keep = ~(0xffffu << sh);
                    const unsigned hb = x.big[n].w[e / 2] >> sh & 0x7c00u, ho = x.off[n].w[e / 2] >> sh & 0x7c00u;
                    const bool nan = hb == 0x7c00u || ho == 0x7c00u, there_ = mine >> e & 1;
                    if (nan && there_) special = 1;
                    if (nan || !there_) {
                        x.big[n].w[e / 2] &= keep;
                        x.off[n].w[e / 2] &= keep;
                    }
                }
        }
        // softmax: the reference of a row moves only when a score passes it by more than kLazy, or at its first key
        h8 pb[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            float mt = s[t][0][0];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) mt = __builtin_elementwise_maximum(mt, s[t][b][r]);
            mt -= kUp;
            const bool seen = m[t] != OPS_NEG_INF;
            const float limit = seen ? kLazy : OPS_NEG_INF;
            if (__builtin_amdgcn_ballot_w64(mt * c[t] > limit) != 0) {
                mt = row4_max(mt);
                const bool grow = mt * c[t] > limit;
                const float delta = grow ? mt : 0.0f;
#pragma unroll
                for (int b = 0; b < 2; ++b) s[t][b] -= delta;
                if (grow) m[t] = ref[t] = ref[t] + delta;
                if (__builtin_amdgcn_ballot_w64(grow && seen) != 0) {
                    const float corr = grow && seen ? ops_exp2(-delta * c[t]) : 1.0f;
                    l[t] *= corr;
#pragma unroll
                    for (int j = 0; j < NO; ++j) o[t][j] *= corr;
                }
            }
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float y = ops_exp2(MOD != 0 ? s[t][b][r] : __builtin_fmaf(s[t][b][r], c[t], kProb));
                    pb[t][4 * b + r] = _Float16(y);   // (11 bits; the row's sum takes them unrounded)
                    l[t] += y;
                }
        }
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                const h8 v = dequant(x.v[n].w[j], one, [&](int e) { return __builtin_bit_cast(h2, x.big[n].w[e]); },
                                     [&](int e) { return __builtin_bit_cast(h2, x.off[n].w[e]); });
#pragma unroll
                for (int t = 0; t < MT; ++t) o[t][n * VW + j] = M4::mma(v, pb[t], o[t][n * VW + j]);
            }
        __builtin_amdgcn_sched_barrier(0);
        load_v(x, i + 2, next, page2);
        bad0 = bad1;
        bad1 = any_bad(page2, key_of(i + 2));
        page2 = look_up(i + 3);
    };
    for (int i = 0; i < nblk; i += 2) {
        block(i, A);
        if (i + 1 < nblk) block(i + 1, B);
    }

#pragma unroll
    for (int t = 0; t < MT; ++t) {
        m[t] *= c[t];   // log2 units
        l[t] = row4_sum(l[t]);
    }
    // Join the waves' sums: the upper half leaves its own in LDS, the lower half adds them, and again.
    __shared__ f32x4 sums[NW / 2][MT * NO * 64];
    __shared__ float Ml[NW / 2][MT][2][16];
    __shared__ int any_special;
    if (threadIdx.x == 0) any_special = 0;
    __syncthreads();
    if (special) any_special = 1;
#pragma unroll
    for (int half = NW / 2; half >= 1; half /= 2) {
        __syncthreads();
        if (wave >= half && wave < 2 * half) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
#pragma unroll
                for (int j = 0; j < NO; ++j) sums[wave - half][(t * NO + j) * 64 + lane] = o[t][j];
                if (g == 0) {
                    Ml[wave - half][t][0][li] = m[t];
                    Ml[wave - half][t][1][li] = l[t];
                }
            }
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const float m2 = Ml[wave][t][0][li], l2 = Ml[wave][t][1][li];
                const float mn = fmaxf(m[t], m2), top = mn == OPS_NEG_INF ? 0.0f : mn;
                const float c1 = ops_exp2(m[t] - top), c2 = ops_exp2(m2 - top);
                m[t] = mn;
                l[t] = l[t] * c1 + l2 * c2;
#pragma unroll
                for (int j = 0; j < NO; ++j) o[t][j] = o[t][j] * c1 + sums[wave][(t * NO + j) * 64 + lane] * c2;
            }
        }
    }
    if (wave != 0) return;

    // Partial sums, or the rows themselves where the sequence is one run.  The lane's columns: 4 VW in a row of each load.
    const RowsParams lp = late_params<RowsParams>();
    const int64_t part = ((int64_t)w.run * lp.kv_heads + w.hk) * lp.nrb + w.rb;
    float* const po = lp.part_o + part * lp.block_rows * PD;
    float* const pm = lp.part_ml + part * 2 * lp.block_rows;
    auto out_row = [&](int r) {
        const int h = w.hk * lp.group + (w.rfirst + r) % lp.group;
        return reinterpret_cast<T*>(lp.out) + w.b * lp.os.b + h * lp.os.h + (w.rfirst + r) / lp.group * lp.os.s;
    };
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int r = 16 * t + li;
        if (w.runs > 1) {
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int j = 0; j < VW; ++j) po[r * PD + n * 16 * VW + 4 * VW * g + VW * e + j] = o[t][n * VW + j][e];
            if (g == 0) {
                pm[r] = m[t] - (kProb - kProbLog2<T>);   // as the joining kernel of the type takes them
                pm[lp.block_rows + r] = l[t];
            }
            continue;
        }
        if (w.rfirst + r >= w.nrows) continue;
        const float inv = l[t] == 0.0f ? 0.0f : 1.0f / l[t];
        T* const out = out_row(r);
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < VW; ++e) {   // the e-th four of the columns
                f32x4 y;
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = o[t][n * VW + (4 * e + j) % VW][(4 * e + j) / VW] * inv;
                const int col = n * 16 * VW + 4 * VW * g + 4 * e;
                if (lp.vec4) store4<T, true>(out, col, D, y);
                else store4<T, false>(out, col, D, y);
            }
        if (lp.lse && g == 0)
            lp.lse[((int64_t)w.b * lp.heads + w.hk * lp.group + (w.rfirst + r) % lp.group) * lp.n + tok[t].token] =
                l[t] == 0.0f ? OPS_NEG_INF : (m[t] + __builtin_log2f(l[t]) - kProb) * kLn2;
    }
    if (!any_special) return;
    // values that are no numbers, to the rows that see them
    __threadfence();
    const int mine = min(16 * MT, w.nrows - w.rfirst);
#pragma unroll 1
    for (int key = w.kbeg; key < w.kend; ++key) {
        if (w.out(key)) continue;
        const int page = pages.page(key);
        if (page < 0) continue;
        const int64_t at = ((int64_t)(lp.table ? page : w.b) * lp.kv_heads + w.hk) * page_rows + (lp.table ? key & pages.page_mask : key);
#pragma unroll 1
        for (int col = lane; col < D; col += 64) {
            const unsigned short* const sv =
                reinterpret_cast<const unsigned short*>(VS) + (at / 8 * NDC + col / 32) * 16 + at % 8;
            const unsigned code = V[at / 8 * D + col] >> (4 * (at % 8 / 2) + 16 * (at % 2)) & 15;
            const float y = __builtin_fmaf(1.0f + (float)code * 0.0625f, float(bits_half(sv[0])), float(bits_half(sv[8])));
            if (!not_finite(y)) continue;
#pragma unroll 1
            for (int r = 0; r < mine; ++r) {
                if (!rows_see(lp, w, (w.rfirst + r) / lp.group, key)) continue;
                if (w.runs > 1) po[r * PD + col] += y;
                else out_row(r)[col] = T(float(out_row(r)[col]) + y);
            }
        }
    }
}

#define PASTE_(a, b, c, d) a##b##c##d
#define PASTE(a, b, c, d) PASTE_(a, b, c, d)
#define KERNEL(NDC, MT, MOD, SMALL, TAG, WAVES)                                                         \
    extern "C" __global__ __launch_bounds__(64 * kRows4Waves, WAVES)                                    \
    void PASTE(fa_rows4_, OPS_NAME, _c##NDC##_t##MT, TAG)(RowsParams p) {                               \
        rows4<OPS_T, NDC, MT, MOD, SMALL>(p);                                                           \
    }
// plain scores, or looked up (m); pages of less than 32 rows (p)
#define KINDS(NDC, MT, WAVES, MWAVES)           \
    KERNEL(NDC, MT, 0, false, , WAVES)          \
    KERNEL(NDC, MT, kAny, false, m, MWAVES)     \
    KERNEL(NDC, MT, kAny, true, p, MWAVES)
KINDS(2, 1, 4, 3)
KINDS(2, 2, 2, 2)
KINDS(4, 1, 3, 2)
KINDS(4, 2, 2, 2)
KINDS(8, 1, 1, 1)
// other widths
#define WIDTHS(NDC, WAVES)                  \
    KERNEL(NDC, 1, kAny, false, m, WAVES)   \
    KERNEL(NDC, 1, kAny, true, p, WAVES)
WIDTHS(1, 4)
WIDTHS(3, 2)
WIDTHS(5, 1)
WIDTHS(6, 1)
WIDTHS(7, 1)
#ifndef OPS_WINDOW
extern "C" __global__ __launch_bounds__(256) void PASTE(fa_cache4_append_, OPS_NAME, , )(Cache4Params p) {
    cache4_append<OPS_T>(p);
}
extern "C" __global__ __launch_bounds__(256) void PASTE(fa_cache4_read_, OPS_NAME, , )(Cache4Params p) {
    cache4_read<OPS_T>(p);
}
#endif
