// fa_rows.h -- what the kernels for query rows over a cache have in common
// (fa_cache.hip, fa_cache4.hip): pages, the runs that the keys of all sequences are cut into, and
// what a row sees.
//
// In a window (OPS_WINDOW) only the keys from the first row's window on and the sinks are walked, the sinks last, as if
// they followed the others (RowsWork::key): bf16, 16 x 32 / 8 heads, one token over 32768 rows in pages, window 4096:
// 51 us for 269 MB (5.3 TB/s), and 5 us to join the runs.
#ifndef FA_ROWS_H
#define FA_ROWS_H

#include "fa_ops_common.h"

// The pages of a sequence.
struct CachePages {
    const int32_t* table;   // nullptr: rows one after another
    int shift, page_mask, n_pages;
    // page of a row, -1: bad (0 without pages)
    __device__ __forceinline__ int page(int row) const {
        if (!table) return 0;
        const int pg = load_uniform(table + (row >> shift));
        return (unsigned)pg < (unsigned)n_pages ? pg : -1;
    }
    // element offset of a row, or -1
    __device__ __forceinline__ int64_t at(int row, int end, int64_t seq, int64_t batch) const {
        if (row >= end) return -1;
        if (!table) return row * seq;
        const int pg = table[row >> shift];
        return (unsigned)pg < (unsigned)n_pages ? pg * batch + (row & page_mask) * seq : -1;
    }
};

__device__ __forceinline__ CachePages rows_pages(const RowsParams& p, int b) {
    return {p.table ? p.table + (int64_t)b * p.pages_per_seq : nullptr, p.page_shift, (1 << p.page_shift) - 1, p.n_pages};
}

// What a workgroup of either kernel works on.
struct RowsWork {
    int run, rb, b, hk;
    int runs;   // of the sequence
    int len, prefix, open, kbeg, kend, nrows, rfirst;
    // windows: kfirst and klast, the run's ends among the keys that are walked: first those from `near` on (near_keys of
    // them), then the sinks; keys [out_lo, out_hi) lie between kbeg and kend but are not the run's
    int kfirst, klast, near, near_keys, out_lo, out_hi;
    int low;          // a window's: keys before this and not before p.sinks are hidden from some row
    int tree, docs;
    // how many keys are walked, and the i-th (a multiple of 16) of them
    __device__ __forceinline__ int kwalk() const { return kWindow ? klast - kfirst : kend - kbeg; }
    __device__ __forceinline__ int key(int i) const {
        if (!kWindow) return kbeg + i;
        const int k = kfirst + i;
        return k < near_keys ? near + k : k - near_keys;
    }
    __device__ __forceinline__ bool out(int k) const { return kWindow && k >= out_lo && k < out_hi; }
};

// Keys that any query of sequence b sees: those before `total`.  In a window, those from `near` on and, after them, those
// before `sinks`, all three but `total` multiples of 64, so that blocks of keys start where they do without.  (Sinks
// last: their scores may be so far below the others, by a bias, that those would lose their low bits against a reference
// that starts there.)
struct Walk {
    int total, near, sinks;
    __device__ __forceinline__ int near_keys() const { return (total - near + 63) & ~63; }
    __device__ __forceinline__ int walked() const { return sinks ? near_keys() + sinks : total - near; }
};
__device__ __forceinline__ Walk rows_walk(const RowsParams& p, int b) {
    Walk w = {0, 0, 0};
    int first;   // position of the first query
    if (p.lens) {
        const int len = p.lens[b];
        w.total = len < 0 ? 0 : (int)min((int64_t)len + p.n, (int64_t)p.sk);
        first = min(len, kWindowMaxPos);
    } else {
        w.total = p.causal ? max(min(max(p.q_start + p.n, p.prefix ? p.prefix[b] : 0), p.sk), 0) : p.sk;
        first = p.q_start;
    }
    if (kWindow) {
        if (!p.lens) w.total = min(w.total, max(max(first + p.n - 1 + p.window, p.sinks), 0));
        w.near = max(min(first - p.window + 1, w.total), 0) & ~63;
        w.sinks = min((p.sinks + 63) & ~63, w.near);
    }
    return w;
}
__device__ __forceinline__ int rows_total(const RowsParams& p, int b) { return rows_walk(p, b).walked(); }

// The runs of a sequence: their length in steps, how many, and the first one's number.
struct Runs {
    int b, steps, count, first;
};
// All sequences' steps are shared out over p.share runs, and a sequence takes as many whole runs as hold
// its own, one at least.  Every wave finds them for itself, a lane a sequence, 64 sequences at a
// time: f(sequence, its runs, the end of its runs' numbers) on every lane.
template <typename F>
__device__ __forceinline__ int each_runs(const RowsParams& p, int lane, F f) {
    auto steps_of = [&](int i) { return (rows_total(p, i) + p.step - 1) / p.step; };
    int64_t all = 0;
    for (int i = lane; i < p.batch; i += 64) all += steps_of(i);
#pragma unroll
    for (int s = 1; s < 64; s *= 2) all += __shfl_xor(all, s);
    const int steps = (int)max((int64_t)1, (all + p.share - 1) / p.share);
    int before = 0;   // runs of the sequences of earlier chunks
    for (int base = 0; base < p.batch; base += 64) {
        const int i = base + lane;
        const int n = i < p.batch ? max(1, (steps_of(i) + steps - 1) / steps) : 0;
        int end = n;
#pragma unroll
        for (int s = 1; s < 64; s *= 2) {
            const int x = __shfl_up(end, s);
            end += lane >= s ? x : 0;
        }
        end += before;
        if (f(base, n, end)) break;
        before = __builtin_amdgcn_readlane(end, 63);
    }
    return steps;
}
// The runs of a call of one sequence.
__device__ __forceinline__ Runs runs_of_one(const RowsParams& p) {
    const int all = (rows_total(p, 0) + p.step - 1) / p.step, steps = max(1, (all + p.share - 1) / p.share);
    return {0, steps, max(1, (all + steps - 1) / steps), 0};
}
// The sequence that run `run` (the same on all lanes) belongs to; b < 0: no such run.
__device__ __forceinline__ Runs runs_of_run(const RowsParams& p, int run, int lane) {
    if (p.batch == 1) {
        Runs r = runs_of_one(p);
        if (run >= r.count) r.b = -1;
        return r;
    }
    Runs r = {-1, 0, 0, 0};
    if (p.share == 1) {   // a run each: with many sequences every workgroup would look through all of them
        if (run < p.batch) r = {run, (rows_total(p, run) + p.step - 1) / p.step, 1, run};
        return r;
    }
    r.steps = each_runs(p, lane, [&](int base, int n, int end) {
        const uint64_t hit = __builtin_amdgcn_ballot_w64(n > 0 && run >= end - n && run < end);
        if (hit == 0) return false;
        const int at = __builtin_ctzll(hit);
        r.b = base + at;
        r.count = __builtin_amdgcn_readlane(n, at);
        r.first = __builtin_amdgcn_readlane(end, at) - r.count;
        return true;
    });
    return r;
}
// Those of sequence b, each lane its own.
__device__ __forceinline__ Runs runs_of_sequence(const RowsParams& p, int b, int lane) {
    if (p.batch == 1) return runs_of_one(p);
    Runs r = {b, 0, 0, 0};
    r.steps = each_runs(p, lane, [&](int base, int n, int end) {
        const int count = __shfl(n, b - base), last = __shfl(end, b - base);
        if (b >= base && b < base + 64) {
            r.count = count;
            r.first = last - count;
        }
        return false;
    });
    return r;
}

// (16 sequences of 33 steps, 17 of them a run's share: 31 + 2 steps each, or 17 + 16; bf16, 16 decode steps in a window of
// 4096 keys)
#if defined(ROWS_EVEN) || defined(OPS_WINDOW)
constexpr bool kEvenRuns = true;
#else
constexpr bool kEvenRuns = false;
#endif

// Returns whether there is work.
__device__ __forceinline__ bool rows_work(const RowsParams& p, int rows, int lane, RowsWork* out) {
    RowsWork& w = *out;
    // the row blocks of one run of keys side by side on one XCD where the counts allow
    int rk;
    if ((p.num_runs * p.kv_heads & 7) == 0) {
        const int t = blockIdx.x >> 3;
        w.rb = t % p.nrb;
        rk = t / p.nrb * 8 + (blockIdx.x & 7);
    } else {
        w.rb = blockIdx.x % p.nrb;
        rk = blockIdx.x / p.nrb;
    }
    w.run = rk / p.kv_heads;
    w.hk = rk % p.kv_heads;
    const Runs r = runs_of_run(p, w.run, lane);
    w.b = __builtin_amdgcn_readfirstlane(r.b);
    if (w.b < 0) return false;
    w.runs = __builtin_amdgcn_readfirstlane(r.count);
    w.tree = p.lens != nullptr;
    w.docs = p.q_doc != nullptr;
    // all of the filled rows, then the drafted ones; every row sees those before `open`
    w.len = w.tree ? load_uniform(p.lens + w.b) : 0;
    w.prefix = p.prefix ? load_uniform(p.prefix + w.b) : 0;
    if (w.tree) {
        w.open = min(max(w.len, 0), p.sk);
    } else {
        w.open = w.docs ? 0 : p.causal ? max(p.q_start + 1, w.prefix) : p.sk;
    }
    if (kWindow) {
        int last = p.q_start + p.n - 1;   // position of the last query
        if (w.tree) {
            last = p.pos ? w.len : (int)min((int64_t)w.len + p.n - 1, (int64_t)kWindowMaxPos);
            for (int i = lane; p.pos && i < p.n; i += 64) last = max(last, p.pos[(int64_t)w.b * p.n + i]);
#pragma unroll
            for (int s = 1; s < 64; s *= 2) last = max(last, __shfl_xor(last, s));
            last = min(__builtin_amdgcn_readfirstlane(last), kWindowMaxPos);
        } else {
            w.open = min(w.open, max(p.q_start + p.window, 0));
        }
        w.low = last - p.window + 1;
    }
    const Walk walk = rows_walk(p, w.b);
    const int total = __builtin_amdgcn_readfirstlane(walk.walked());
    int64_t per = (int64_t)__builtin_amdgcn_readfirstlane(r.steps) * p.step;
    // a sequence's runs of one length, rather than all but its last
    if (kEvenRuns) per = (int64_t)((total + p.step * w.runs - 1) / (p.step * w.runs)) * p.step;
    w.kbeg = (int)min((w.run - __builtin_amdgcn_readfirstlane(r.first)) * per, (int64_t)total);
    w.kend = (int)min(w.kbeg + per, (int64_t)total);
    if (kWindow) {
        w.kfirst = w.kbeg;
        w.klast = w.kend;
        w.near = __builtin_amdgcn_readfirstlane(walk.near);
        const int end = __builtin_amdgcn_readfirstlane(walk.total), nk = __builtin_amdgcn_readfirstlane(walk.near_keys());
        w.near_keys = nk;
        w.out_lo = w.out_hi = 0;
        if (w.kfirst < nk) {
            w.kbeg = w.near + w.kfirst;
            w.kend = w.near + min(w.klast, end - w.near);
            if (w.klast > nk) {   // sinks too
                w.out_lo = w.klast - nk;
                w.out_hi = w.kbeg;
                w.kbeg = 0;
            }
        } else {
            w.kbeg = w.kfirst - nk;
            w.kend = w.klast - nk;
        }
    }
    w.nrows = p.n * p.group;
    w.rfirst = w.rb * rows;
    return true;
}

// Whether the keys of a block need the mask: [k0, k0 + n).
__device__ __forceinline__ int rows_masked(const RowsParams& p, const RowsWork& w, int k0, int n) {
    return k0 + n > min(w.open, w.kend) || (kWindow && k0 < w.low && k0 + n > p.sinks);
}

// Position of a token for windows, which drafted tokens do not stand before their sequence's filled rows for.
__device__ __forceinline__ int window_position(const RowsParams& p, const RowsWork& w, int tok) {
    if (!w.tree) return p.q_start + tok;
    return min(p.pos ? max(p.pos[(int64_t)w.b * p.n + tok], w.len) : w.len + tok, kWindowMaxPos);
}
// Whether the window hides key `key` from a token that stands at `pos`.
__device__ __forceinline__ bool window_hides(const RowsParams& p, const RowsWork& w, int pos, int key) {
    if (key < p.sinks) return false;
    if (!w.tree) return key <= pos - p.window || key >= pos + p.window;
    const int bit = key - w.len;
    return pos - (bit >= 0 ? window_position(p, w, min(bit, p.n - 1)) : key) >= p.window;
}

// Whether token `tok` sees key `key` < kend, as far as masks tell.
__device__ __forceinline__ bool rows_see(const RowsParams& p, const RowsWork& w, int tok, int key) {
    if (kWindow && window_hides(p, w, window_position(p, w, tok), key)) return false;
    if (!w.tree) {
        if (p.causal && !(key <= p.q_start + tok || key < w.prefix)) return false;
        if (!w.docs) return true;
        const int id = p.q_doc[(int64_t)w.b * p.n + tok];
        return id >= 0 && p.k_doc[(int64_t)w.b * p.sk + key] == id;
    }
    if (key < w.len) return true;
    const int bit = key - w.len;
    if (!p.mask) return bit <= tok;
    const int64_t row = (p.mask_shared ? 0 : (int64_t)w.b * p.n) + tok;
    return (p.mask[row * p.mask_words + (bit >> 6)] >> (bit & 63)) & 1;
}

__device__ __forceinline__ uint64_t bits_before(int n) { return n >= 64 ? ~0ull : (1ull << max(n, 0)) - 1; }

// Bits of the N keys from k0 that the window leaves a row at position pos; drafted keys that stand where the program says: of the keys
// at(b, r), b < N / 16, whose scores the lane holds.
template <int N, typename At>
__device__ __forceinline__ uint64_t window_bits(const RowsParams& p, const RowsWork& w, int pos, int k0, At at_) {
    const int at = w.tree ? min(max(pos, w.len), kWindowMaxPos) : pos;
    uint64_t bits = ~bits_before(at - p.window + 1 - k0);
    if (!w.tree) bits &= bits_before(at + p.window - k0);
    bits |= bits_before(p.sinks - k0);
    if (w.tree && p.pos && k0 + N > w.len) {
#pragma unroll 1
        for (int b = 0; b < N / 16; ++b)
#pragma unroll 1
            for (int r = 0; r < 4; ++r) {
                const int x = at_(b, r);
                if (k0 + x < w.len) continue;
                bits = window_hides(p, w, at, k0 + x) ? bits & ~(1ull << x) : bits | 1ull << x;
            }
    }
    return bits;
}

#endif  // FA_ROWS_H
