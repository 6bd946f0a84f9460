// fa_ops_host.h -- host side of attention with modified scores, rotary
// positions, norms and the key / value caches (included by fa_host.cpp, whose device
// state and stream workspaces it uses).
//
// Their kernels are code objects of their own next to fa_kernels.hsaco, each loaded
// by the first call that needs it (0.4 to 3.4 ms; a capture does not mind), so that
// programs without them load none.  Every argument is checked before anything is queued.

#include "fa_ops_params.h"

namespace {

// Code objects: those of score attention and of the cache one a type (FA_DTYPE_*), those of a cache in 4 bits for bf16
// and f16; calls in a window have their own.
enum OpsModule {
    kRotaryModule,
    kNormModule,
    kScoreModule,
    kCacheModule = kScoreModule + 3,
    kCache4Module = kCacheModule + 3,
    kScoreWindowModule = kCache4Module + 2,
    kCacheWindowModule = kScoreWindowModule + 3,
    kCache4WindowModule = kCacheWindowModule + 3,
    kOpsModules = kCache4WindowModule + 2
};
OpsModule of_type(OpsModule m, int dtype) { return static_cast<OpsModule>(m + dtype); }

struct OpsState {
    std::once_flag once[kOpsModules];
    int status[kOpsModules] = {};
    hipModule_t module[kOpsModules] = {};
    std::mutex mu;
    std::unordered_map<std::string, hipFunction_t> fns[kOpsModules];
};

OpsState g_ops[kMaxDevices];

#define OPS_STRING_(x) #x
#define OPS_STRING(x) OPS_STRING_(x)
constexpr char kStampKernel[] = OPS_STRING(OPS_STAMP_KERNEL);

constexpr size_t kOpsMaxSeq = size_t(1) << 30;      // tokens: positions and their sums stay in 32 bits
constexpr size_t kOpsMaxD = 256;
constexpr int64_t kOpsMaxRowStride = int64_t(1) << 22;   // elements: a tile's byte offsets stay in 32 bits
constexpr int64_t kOpsMaxStride = int64_t(1) << 44;
constexpr size_t kTreeMaxTokens = 256;
constexpr size_t kOpsMaxGrid = size_t(1) << 23;   // workgroups: threads of a launch stay in 32 bits
constexpr size_t kOpsMaxTokens = size_t(1) << 31;   // of a rotary launch: a thread for each at least

int ops_module(int dev, OpsModule which) {
    static const char* const files[kOpsModules] = {
        "fa_rotary.hsaco",       "fa_norm.hsaco",          "fa_score_f32.hsaco",    "fa_score_bf16.hsaco",
        "fa_score_f16.hsaco",    "fa_cache_f32.hsaco",     "fa_cache_bf16.hsaco",   "fa_cache_f16.hsaco",
        "fa_cache4_bf16.hsaco",  "fa_cache4_f16.hsaco",    "fa_score_w_f32.hsaco",  "fa_score_w_bf16.hsaco",
        "fa_score_w_f16.hsaco",  "fa_cache_w_f32.hsaco",   "fa_cache_w_bf16.hsaco", "fa_cache_w_f16.hsaco",
        "fa_cache4_w_bf16.hsaco", "fa_cache4_w_f16.hsaco"};
    OpsState& s = g_ops[dev];
    std::call_once(s.once[which], [&] {
        std::string path = module_path();
        const size_t pos = path.rfind('/');
        path = (pos == std::string::npos ? std::string() : path.substr(0, pos + 1)) + files[which];
        FILE* f = std::fopen(path.c_str(), "rb");
        if (f) std::fclose(f);
        hipFunction_t of_this_build;
        if (!f || hipModuleLoad(&s.module[which], path.c_str()) != hipSuccess ||
            hipModuleGetFunction(&of_this_build, s.module[which], kStampKernel) != hipSuccess) {
            (void)hipGetLastError();
            s.status[which] = FA_ERR_MODULE;
        }
    });
    return s.status[which];
}

template <typename P>
int ops_launch(int dev, OpsModule which, const char* name, size_t grid, unsigned block, P* p, hipStream_t stream) {
    if (grid == 0) return FA_OK;
    OpsState& s = g_ops[dev];
    hipFunction_t fn = nullptr;
    {
        std::lock_guard<std::mutex> lock(s.mu);
        auto it = s.fns[which].find(name);
        if (it != s.fns[which].end()) {
            fn = it->second;
        } else {
            if (hipModuleGetFunction(&fn, s.module[which], name) != hipSuccess) {
                (void)hipGetLastError();
                return FA_ERR_MODULE;
            }
            s.fns[which].emplace(name, fn);
        }
    }
    void* args[] = {p};
    if (hipModuleLaunchKernel(fn, static_cast<unsigned>(grid), 1, 1, block, 1, 1, 0, stream, args, nullptr) !=
        hipSuccess) {
        (void)hipGetLastError();
        return FA_ERR_LAUNCH;
    }
    return FA_OK;
}

// Device and module of a call; *dev is the current device.
int ops_begin(int* dev, OpsModule which) {
    int rc = current_device(dev);
    if (rc == FA_OK) rc = ensure_loaded(*dev);
    if (rc == FA_OK) rc = ops_module(*dev, which);
    return rc;
}

// A call's scratch memory: the stream's workspace, which is the call's until this object goes, or an
// allocation around the call above its limit.
struct OpsWorkspace {
    void* ptr = nullptr;
    bool own = false;
    WorkspaceCall call;
    int get(int dev, hipStream_t stream, size_t bytes) {
        if (bytes <= kWorkspaceCacheMax) {
            call = WorkspaceCall(dev, stream);
            return stream_workspace(dev, stream, bytes, &ptr);
        }
        if (bytes > free_device_bytes() || hipMallocAsync(&ptr, bytes, stream) != hipSuccess) {
            (void)hipGetLastError();
            return FA_ERR_ALLOC;
        }
        own = true;
        return FA_OK;
    }
    int done(hipStream_t stream, int rc) {
        if (own && hipFreeAsync(ptr, stream) != hipSuccess) {
            (void)hipGetLastError();
            if (rc == FA_OK) rc = FA_ERR_ALLOC;
        }
        return rc;
    }
};

size_t elem_size(int dtype) { return dtype == FA_DTYPE_F32 ? 4 : 2; }
const char* dtype_name(int dtype) { return dtype == FA_DTYPE_F32 ? "f32" : dtype == FA_DTYPE_BF16 ? "bf16" : "f16"; }
bool valid_dtype(int dtype) { return dtype == FA_DTYPE_F32 || dtype == FA_DTYPE_BF16 || dtype == FA_DTYPE_F16; }
int ops_pad_d(size_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// A tensor's layout: strides resolved, and what they allow.
struct OpsLayout {
    OpsStrides st{};
    bool aligned16 = true;   // rows start 16-byte aligned (given the pointer)
    bool aligned4 = true;    // rows start at multiples of 4 elements
};

int resolve_layout(const fa_strides& in, size_t batch, size_t seq, size_t heads, size_t d, size_t esize, bool writable,
                   OpsLayout* out) {
    int64_t b = in.batch, s = in.seq, h = in.head;
    if (b < 0 || s < 0 || h < 0) return FA_ERR_INVALID_ARG;
    const int64_t row = static_cast<int64_t>(d);
    if (b == 0 && s == 0 && h == 0) {
        s = row;
        h = static_cast<int64_t>(seq) * row;
        if (h > 0 && static_cast<int64_t>(heads) > kOpsMaxStride / h) return FA_ERR_UNSUPPORTED;
        b = static_cast<int64_t>(heads) * h;
    }
    // strides of single entries are never used, whatever they are
    if (seq <= 1) s = row;
    if (heads <= 1) h = 0;
    if (batch <= 1) b = 0;
    if (b > kOpsMaxStride || h > kOpsMaxStride || s >= kOpsMaxRowStride) return FA_ERR_UNSUPPORTED;
    if (s < row) return FA_ERR_INVALID_ARG;
    if (writable) {
        // no two rows overlap: each dimension steps over all of the smaller ones
        struct Dim {
            int64_t stride;
            size_t n;
        } dims[3] = {{b, batch}, {s, seq}, {h, heads}};
        std::sort(dims, dims + 3, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
        int64_t extent = row;
        for (const Dim& x : dims) {
            if (x.n <= 1) continue;
            if (x.stride < extent) return FA_ERR_INVALID_ARG;
            // a stride of 2^44 over 2^30 entries would pass 64 bits; none is larger than 2^44
            extent = x.n > static_cast<size_t>(kOpsMaxStride / x.stride) ? 2 * kOpsMaxStride
                                                                          : x.stride * static_cast<int64_t>(x.n);
        }
    }
    out->st = {b, s, h};
    const int64_t unit = static_cast<int64_t>(16 / esize);
    out->aligned16 = b % unit == 0 && s % unit == 0 && h % unit == 0 && row % unit == 0;
    out->aligned4 = b % 4 == 0 && s % 4 == 0 && h % 4 == 0;
    return FA_OK;
}

// 16-byte loads of 8-column chunks / stores of 4 columns.
bool vec_ok(const void* ptr, const OpsLayout& l, size_t d) { return l.aligned16 && d % 8 == 0 && aligned16(ptr); }
bool ovec_ok(const void* ptr, const OpsLayout& l, size_t esize) {
    return l.aligned4 && (reinterpret_cast<uintptr_t>(ptr) & (4 * esize - 1)) == 0;
}

struct ScoreScale {
    float scale, scale_log2e, cap_in, cap_log2e;
};
int resolve_scale(float scale, float softcap, size_t d, ScoreScale* out) {
    if (!(softcap >= 0.0f) || !std::isfinite(softcap)) return FA_ERR_INVALID_ARG;
    if (!(scale > 0.0f) || !std::isfinite(scale)) scale = 1.0f / std::sqrt(static_cast<float>(d));
    constexpr float log2e = 1.44269504088896341f;
    out->scale = scale;
    out->scale_log2e = scale * log2e;
    out->cap_in = softcap > 0.0f ? 2.0f * log2e * scale / softcap : 0.0f;
    out->cap_log2e = softcap * log2e;
    // a cap, or its ratio to the scale, at the ends of f32's range
    if (softcap > 0.0f && (!std::isnormal(out->cap_in) || !std::isnormal(out->cap_log2e))) return FA_ERR_UNSUPPORTED;
    return FA_OK;
}

// Large caps of 16-bit types need the longer tanh, which only the kernels of any alignment have (bf16, 32 x 2048^2 causal,
// 64 columns: 46 us with a cap of 400, 200 with one of 1000, whose scores the short tanh would leave 2e-4 off).
bool cap_ok(int dtype, float softcap) { return dtype == FA_DTYPE_F32 || softcap <= kFastCap; }

// Tag of the kernel for what happens to the scores.
const char* score_tag(const fa_score_config& c, bool vec, bool window) {
    if (window) return !vec ? "s" : c.softcap > 0.0f || c.slopes ? "m" : "";
    return !vec ? "s" : c.softcap > 0.0f ? (c.slopes ? "cb" : "c") : c.slopes ? "b" : "";
}

// How a score kernel's four waves share a block of rows: two 16-row tiles a wave where that still makes
// workgroups enough (what a wave reads from LDS serves both tiles); on small grids two groups of
// waves on the same rows, each with half of the walked rows.
struct ScoreTiles {
    int mt, groups, rows;   // rows of a block
    const char* tag;
};
ScoreTiles score_tiles(const fa_score_config& c, int D, bool vec, size_t rows, size_t slices, int num_cus) {
    const size_t cus = static_cast<size_t>(num_cus), blocks = (rows + 63) / 64 * slices;
    // causal workgroups differ in length, so that a single round of them ends late (2048^2, d128: 32 heads 60 us
    // with one tile a wave, 70 with two; 48 heads 86 and 73)
    if (vec && c.dtype != FA_DTYPE_F32 && D <= 128 && (rows + 127) / 128 * slices >= (c.causal ? 3 : 2) * cus)
        return {2, 1, 128, ""};
    // measured (bf16, causal): 16 x 1024^2 d64 (256 blocks) 15.9 us against 18.7, 32 x 1024^2 (512) 19.3 against 19.6,
    // 32 x 1024^2 d128 all visible (512) 38.2 against 27.2
    if (vec && D <= 128 && 2 * blocks <= 3 * cus) return {1, 2, 32, "k"};
    return {1, 1, 64, ""};
}

// Plan of the dK / dV kernel: tiles a wave, and the workgroups that share the heads of a group.
struct DkvPlan {
    ScoreTiles tiles;
    int splits;
    size_t blocks, floats;
};
DkvPlan plan_dkv(const fa_score_config& c, int D, bool vec, int size, int num_cus) {
    DkvPlan r{};
    const size_t nkv = c.batch * c.kv_heads, group = c.heads / c.kv_heads;
    size_t s = 1;
    // (in a window all are of one length, and one round of them will do)
    while (s < group && (c.seq_len_k + 63) / 64 * nkv * s < (size ? 2 : 4) * static_cast<size_t>(num_cus)) {
        ++s;
        while (group % s != 0) ++s;
    }
    r.tiles = score_tiles(c, D, vec, c.seq_len_k, nkv * s, num_cus);
    if (D == 128 && r.tiles.mt == 2) r.tiles = {1, 1, 64, ""};   // two tiles' K, V, dK and dV leave one wave a SIMD: slower
    r.blocks = (c.seq_len_k + r.tiles.rows - 1) / r.tiles.rows;
    r.splits = static_cast<int>(s);
    r.floats = s > 1 ? 2 * s * nkv * c.seq_len_k * D : 0;
    return r;
}

// A window's size and sinks as kernels take them (size 0: hides nothing); farthest: the largest distance there is; past:
// how far beyond it kernels may reckon.
int resolve_window(const fa_window* w, bool docs, int64_t farthest, int past, int* size, int* sinks) {
    *size = *sinks = 0;
    if (!w) return FA_OK;
    if (w->size < 1 || w->sinks < 0) return FA_ERR_INVALID_ARG;
    if (w->sinks > 0 && docs) return FA_ERR_UNSUPPORTED;   // the first keys are another document's
    if (w->size > farthest) return FA_OK;
    if (farthest + past > kWindowMaxPos) return FA_ERR_UNSUPPORTED;   // positions plus or minus a window stay in 32 bits
    *size = static_cast<int>(w->size);
    *sinks = static_cast<int>(std::min<int64_t>(w->sinks, kWindowMaxPos));
    return FA_OK;
}
// The most keys that n consecutive queries of a window walk.
size_t window_keys(size_t keys, int size, int sinks, size_t n, bool both_sides) {
    if (size == 0) return keys;
    return std::min(keys, (both_sides ? 2 : 1) * static_cast<size_t>(size) + sinks + n + 128);
}

// In a window: key blocks that hold sinks, and the workgroups that take the queries that see them from afar.  These
// are shorter than those of the other key blocks, which run first and all end at about the same time: a head of the
// group each, and two thirds of the stages that a window reaches (2 x 16 / 4 heads x 4096^2, 128 columns, window 512,
// 64 sinks, bf16: dK and dV).
struct FarPlan {
    int stages, chunks, splits, blocks;
    size_t floats;
};
FarPlan plan_far(const fa_score_config& c, int D, const DkvPlan& dkv, int size, int sinks) {
    FarPlan r{};
    if (size == 0 || sinks == 0 || c.seq_len_k == 0 || c.seq_len_q == 0) return r;
    const size_t step = dkv.tiles.groups == 1 && (c.dtype == FA_DTYPE_F32 || D > 128) ? 32 : 64;   // queries of a stage
    const size_t nst = (c.seq_len_q + step - 1) / step;
    r.blocks = static_cast<int>((std::min<size_t>(sinks, c.seq_len_k) + dkv.tiles.rows - 1) / dkv.tiles.rows);
    const size_t reach = window_keys(c.seq_len_q, size, 0, dkv.tiles.rows, !c.causal || c.prefix) / step + 1;
    // Where sinks are many, key blocks are of like length without; and the partial sums get 64 MiB at most.
    if (4 * static_cast<size_t>(r.blocks) > dkv.blocks) return FarPlan{};
    r.splits = static_cast<int>(c.heads / c.kv_heads);
    for (size_t stages = std::max(2 * reach / 3, size_t(4)); stages < nst; stages *= 2) {
        r.stages = static_cast<int>(stages);
        r.chunks = static_cast<int>((nst + stages - 1) / stages);
        r.floats = size_t(2) * (r.chunks * size_t(r.splits) + 1) * c.batch * c.kv_heads * r.blocks * dkv.tiles.rows * D;
        if (r.floats <= size_t(16) << 20) return r;
    }
    return FarPlan{};
}

size_t doc_tiles(size_t n) { return (n + kDocTile - 1) / kDocTile; }

// Plan of the rows kernels: streaming waves for few rows, else workgroups that share their
// keys; the keys of all sequences shared out over as many runs as fill the GPU once.
struct RowsPlan {
    bool stream;
    int mt, threads, rows, nrb, step, share, runs;
    size_t floats;
};
// Shares the keys of all sequences out over runs; up to `whole` keys a sequence are one.  D: columns of a row of
// partial sums.
void share_keys(RowsPlan* plan, size_t batch, size_t kv_heads, size_t rows, size_t keys, size_t resident, size_t whole,
                int D) {
    RowsPlan& r = *plan;
    r.nrb = static_cast<int>((rows + r.rows - 1) / r.rows);
    const size_t units = kv_heads * r.nrb;   // workgroups a run
    // One round of resident workgroups where the sequences' last, shorter runs (one a sequence)
    // leave room, else several rounds of shorter runs.
    const size_t slots = std::max<size_t>(1, resident / units);
    size_t share = batch == 1 ? slots : 2 * (batch - 1) <= slots ? slots - (batch - 1) : 4 * slots;
    share = std::min(share, batch * std::max<size_t>(1, (keys + r.step - 1) / r.step));
    if (batch * units >= 4 * resident) share = 1;   // sequences enough: one run each
    if (keys <= whole) share = 1;
    r.share = static_cast<int>(share);
    // each sequence rounds its share up to whole runs; eight runs and heads more or less fall
    // on the eight XCDs evenly
    size_t runs = share == 1 ? batch : share + batch - 1;
    while (runs * kv_heads % 8 != 0 && runs >= 8) ++runs;
    r.runs = static_cast<int>(runs);
    r.floats = share > 1 ? runs * units * r.rows * (D + 2) : 0;
}
RowsPlan plan_rows(int dtype, int D, bool vec, size_t batch, size_t kv_heads, size_t rows, size_t keys, int num_cus) {
    RowsPlan r{};
    const bool f32 = dtype == FA_DTYPE_F32;
    const int row_bytes = D * static_cast<int>(elem_size(dtype));
    // A streaming wave reads a block's K and V for 16 or 32 rows only; with more rows it reads them again (8 sequences
    // of 8000 keys, bf16: 64 rows of 128 columns 102 us streamed, 60 shared, of 256 columns 312 and 107; 16 rows of 128
    // columns 45 and 57; 64 rows of 64 columns 42 and 47)
    r.stream = vec && rows <= (row_bytes <= 128 ? 64 : 16) && row_bytes <= 512;
    size_t resident = static_cast<size_t>(num_cus);
    if (r.stream) {
        r.mt = rows <= 16 ? 1 : 2;
        const int waves = row_bytes <= 256 ? kStreamWaves<256> : kStreamWaves<512>;
        r.threads = 64 * waves;
        r.rows = 16 * r.mt;
        r.step = 32 * waves;
        if (row_bytes <= 128) resident *= 2;   // LDS holds one workgroup a CU, two of short rows
    } else {
        // Two tiles a wave halve what is read from LDS and L2, but start and end later: where each CU gets 16 stages or
        // more (d128: 8 sequences of 16384 keys, 256 rows 308 us with one, 210 with two; 4 of 3000, 200 rows 32 and 39)
        const size_t stages = batch * keys * kv_heads * ((rows + 127) / 128) / 64;
        r.mt = !vec || f32 || D > 128 || rows <= 128 || stages < 16 * resident ? 1 : 2;
        r.threads = 512;
        r.rows = 128 * r.mt;
        r.step = f32 || D > 128 ? 32 : 64;
    }
    // Few keys: one run each, which saves the merge, some 4 us, unless walking them costs as much (measured: 8
    // sequences of 250 keys, bf16, 7 rows of 64 columns 13.1 us split, 9.7 whole; 3 of 250, f32, 8 rows of 80 17.6
    // and 23.6)
    share_keys(&r, batch, kv_heads, rows, keys, resident, static_cast<size_t>(r.step) * (f32 || D > 128 ? 1 : 4), D);
    return r;
}

OpsModule cache_module(int dtype, const RowsParams& p) { return of_type(p.window ? kCacheWindowModule : kCacheModule, dtype); }

// Launches a rows kernel, and the one that joins its partial sums (of D columns).
int launch_rows(int dev, hipStream_t stream, int dtype, OpsModule module, const char* kernel, const RowsPlan& plan, int D,
                bool vec, RowsParams* p) {
    const size_t rows = static_cast<size_t>(p->n) * p->group;
    p->nrb = plan.nrb;
    p->block_rows = plan.rows;
    p->num_runs = plan.runs;
    p->share = plan.share;
    p->step = plan.step;
    const size_t grid = static_cast<size_t>(plan.runs) * p->kv_heads * plan.nrb;
    const size_t mgrid = static_cast<size_t>(p->batch) * p->kv_heads * rows;
    if (grid > kOpsMaxGrid / 2 || (plan.floats && mgrid > kOpsMaxGrid)) return FA_ERR_UNSUPPORTED;
    int rc;
    OpsWorkspace ws;
    if (plan.floats) {
        if ((rc = ws.get(dev, stream, plan.floats * sizeof(float))) != FA_OK) return rc;
        p->part_o = static_cast<float*>(ws.ptr);
        p->part_ml = p->part_o + grid * plan.rows * D;
    }
    rc = ops_launch(dev, module, kernel, grid, plan.threads, p, stream);
    if (rc == FA_OK && plan.floats) {
        // eight runs a sequence or more: a workgroup a row
        const bool wide = !vec || plan.share > 8 * p->batch;
        char name[64];
        std::snprintf(name, sizeof(name), "fa_rows_merge_%s_d%d%s", dtype_name(dtype), D, !vec ? "s" : wide ? "w" : "");
        const size_t per = wide ? 1 : 1024 / D;
        rc = ops_launch(dev, cache_module(dtype, *p), name, (mgrid + per - 1) / per, 256, p, stream);
    }
    return ws.done(stream, rc);
}

int run_rows(int dev, hipStream_t stream, int dtype, int D, bool vec, RowsParams* p, size_t keys) {
    vec = vec && (!p->table || p->page_shift >= 4);   // DMA moves runs of rows of one page
    const OpsModule module = cache_module(dtype, *p);
    const int rc = ops_module(dev, module);
    if (rc != FA_OK) return rc;
    const RowsPlan plan =
        plan_rows(dtype, D, vec, p->batch, p->kv_heads, static_cast<size_t>(p->n) * p->group, keys, g_dev[dev].num_cus);
    char name[64];
    std::snprintf(name, sizeof(name), "fa_rows_%s_%s_d%d_t%d%s", plan.stream ? "stream" : "shared", dtype_name(dtype), D,
                  plan.mt, !vec ? "s" : p->window ? (p->cap_log2e != 0.0f || p->slopes ? "m" : "")
                                  : p->cap_log2e != 0.0f ? (p->slopes ? "cb" : "c") : p->slopes ? "b" : "");
    return launch_rows(dev, stream, dtype, module, name, plan, D, vec, p);
}

// Short query blocks, and few workgroups over many keys, run on the rows kernel, which splits the keys.  keys: those
// that any query of the call walks; walk: those that 32 of them do (in a window fewer).
bool score_takes_rows(const fa_score_config& c, size_t keys, size_t walk, int num_cus) {
    const size_t group = c.heads / c.kv_heads, cus = static_cast<size_t>(num_cus);
    if (c.seq_len_q * group <= 64) return true;
    // a workgroup of 32 rows takes some 0.6 us per 64 keys: above 2048 keys longer than the split and its merge, at
    // 256 columns above 1024 (1 head, 1900^2 causal: bf16 53 us whole, 35 split, f32 277 and 97; 2 heads of 128
    // columns, 1500^2: bf16 21 and 30, f32 72 and 78)
    const size_t blocks = c.batch * c.heads * ((c.seq_len_q + 31) / 32);
    if (keys < (c.d_head > 128 ? 1024 : 2048) || 2 * blocks > cus) return false;
    // The rows kernel takes every block of rows through all of the call's keys, shared out over all CUs, a score kernel's
    // workgroup only its own through what the window leaves: the split has to save the time of the merge, here in keys of
    // a walk.  It always does without a window.  With one, 128 blocks, whole and split: 1 head of 128 columns, 4096^2,
    // window 100 bf16 12 and 44 us, f32 22 and 108; 8 heads of 128, 512 queries at the end of 8192 keys, window 1700
    // bf16 30 and 36, f32 91 and 71, window 3000 bf16 45 and 41; 1 head of 256, 4000^2, bf16, window 1500 56 and 62,
    // window 2000 69 and 62.
    const bool f32 = c.dtype == FA_DTYPE_F32;
    const size_t merge = f32 ? 256 : c.d_head > 128 ? 576 : 1280, split = keys * blocks / cus;
    return walk >= merge + (f32 ? split : 2 * split / 3);   // (a key takes 16-bit rows kernels two thirds of that)
}

int check_score(const fa_score_config* c) {
    if (!c || !valid_dtype(c->dtype)) return FA_ERR_INVALID_ARG;
    if (c->batch == 0 || c->heads == 0 || c->d_head == 0) return FA_OK;
    if (c->kv_heads == 0 || c->heads % c->kv_heads != 0) return FA_ERR_INVALID_ARG;
    if ((c->q_doc == nullptr) != (c->k_doc == nullptr)) return FA_ERR_INVALID_ARG;
    if (c->d_head > kOpsMaxD || c->seq_len_q > kOpsMaxSeq || c->seq_len_k > kOpsMaxSeq || c->batch > kOpsMaxSeq ||
        c->heads > kOpsMaxSeq || c->q_start > (int64_t)kOpsMaxSeq || c->q_start < -(int64_t)kOpsMaxSeq)
        return FA_ERR_UNSUPPORTED;
    return FA_OK;
}

void fill_score(const fa_score_config& c, const ScoreScale& sc, ScoreParams* p) {
    p->batch = static_cast<int>(c.batch);
    p->heads = static_cast<int>(c.heads);
    p->kv_heads = static_cast<int>(c.kv_heads);
    p->group = static_cast<int>(c.heads / c.kv_heads);
    p->sq = static_cast<int>(c.seq_len_q);
    p->sk = static_cast<int>(c.seq_len_k);
    p->d = static_cast<int>(c.d_head);
    p->causal = c.causal ? 1 : 0;
    p->q_start = static_cast<int>(c.q_start);
    p->slopes = c.slopes;
    p->q_doc = c.q_doc;
    p->k_doc = c.k_doc;
    p->prefix = c.causal ? c.prefix : nullptr;
    p->scale = sc.scale;
    p->scale_log2e = sc.scale_log2e;
    p->cap_in = sc.cap_in;
    p->cap_log2e = sc.cap_log2e;
}

// Tables of the documents: ranges of the tiles, and the order of the blocks (of q_rows queries and k_rows keys; 0:
// that side's is not needed).  Order where the workgroups of a side are more than run at once.
struct DocPlan {
    bool q_order, k_order;
    size_t q_blocks, k_blocks, bytes;
};
DocPlan plan_docs(const fa_score_config& c, size_t q_rows, size_t q_slices, size_t k_rows, size_t k_slices, int num_cus) {
    DocPlan r{};
    if (!c.q_doc) return r;
    const size_t qt = c.batch * doc_tiles(c.seq_len_q), kt = c.batch * doc_tiles(c.seq_len_k);
    r.q_blocks = q_rows ? c.batch * ((c.seq_len_q + q_rows - 1) / q_rows) : 0;
    r.k_blocks = k_rows ? c.batch * ((c.seq_len_k + k_rows - 1) / k_rows) : 0;
    const size_t fits = 2 * static_cast<size_t>(num_cus);
    r.q_order = r.q_blocks <= kOrderBlocks && kt <= kOrderTiles && r.q_blocks * q_slices > fits;
    r.k_order = r.k_blocks <= kOrderBlocks && qt <= kOrderTiles && r.k_blocks * k_slices > fits;
    r.bytes = sizeof(int32_t) * (2 * (qt + kt) + r.q_blocks + r.k_blocks);
    return r;
}
int launch_docs(int dev, OpsModule module, hipStream_t stream, const DocPlan& plan, size_t q_rows, size_t k_rows,
                ScoreParams* p, int32_t* ws) {
    const size_t qt = p->batch * doc_tiles(p->sq), kt = p->batch * doc_tiles(p->sk);
    p->q_rng = ws;
    p->k_rng = ws + 2 * qt;
    int rc = ops_launch(dev, module, "fa_score_doc_ranges", (qt + kt + 3) / 4, 256, p, stream);
    int32_t* const q_order = ws + 2 * (qt + kt);
    if (rc != FA_OK || (!plan.q_order && !plan.k_order)) return rc;
    p->q_order = plan.q_order ? q_order : nullptr;
    p->k_order = plan.k_order ? q_order + plan.q_blocks : nullptr;
    p->q_rows = static_cast<int>(q_rows);
    p->k_rows = static_cast<int>(k_rows);
    return ops_launch(dev, module, "fa_score_doc_order", 2, 1024, p, stream);
}

int check_cache(const fa_kv_cache* c, OpsLayout* k, OpsLayout* v, size_t* capacity) {
    if (!c || !valid_dtype(c->dtype)) return FA_ERR_INVALID_ARG;
    if (c->batch == 0 || c->kv_heads == 0 || c->d_head == 0) return FA_OK;
    if (c->d_head > kOpsMaxD || c->batch > kOpsMaxSeq || c->kv_heads > kOpsMaxSeq) return FA_ERR_UNSUPPORTED;
    if (!c->lens) return FA_ERR_INVALID_ARG;
    size_t rows = c->capacity, blocks = c->batch;
    if (c->block_table) {
        if (c->page_size == 0 || (c->page_size & (c->page_size - 1)) != 0) return FA_ERR_INVALID_ARG;
        if (c->page_size > kOpsMaxSeq || c->pages_per_seq > kOpsMaxSeq || c->n_pages > kOpsMaxSeq)
            return FA_ERR_UNSUPPORTED;
        *capacity = c->page_size * c->pages_per_seq;
        rows = c->page_size;
        blocks = c->n_pages;
    } else {
        *capacity = rows;
    }
    if (*capacity > kOpsMaxSeq) return FA_ERR_UNSUPPORTED;
    int rc = resolve_layout(c->k_strides, blocks, rows, c->kv_heads, c->d_head, elem_size(c->dtype), true, k);
    if (rc == FA_OK) rc = resolve_layout(c->v_strides, blocks, rows, c->kv_heads, c->d_head, elem_size(c->dtype), true, v);
    if (rc == FA_OK && *capacity > 0 && (!c->k || !c->v)) rc = FA_ERR_INVALID_ARG;
    return rc;
}

int page_shift(const fa_kv_cache& c) {
    int s = 0;
    while (c.block_table && (size_t(1) << s) < c.page_size) ++s;
    return s;
}

int check_rotary(const fa_rotary_config* c) {
    if (!c || !valid_dtype(c->dtype)) return FA_ERR_INVALID_ARG;
    if (c->d_head > kOpsMaxD) return FA_ERR_UNSUPPORTED;
    if (c->rot_dim < 2 || c->rot_dim % 2 != 0 || c->rot_dim > c->d_head) return FA_ERR_INVALID_ARG;
    return FA_OK;
}

int add_rotary_tensor(RotParams* p, const void* src, void* dst, const OpsLayout& in, const OpsLayout& out, size_t heads,
                      bool rotate, bool cache, bool* wide) {
    RotTensor& t = p->t[p->nt++];
    t.src = src;
    t.dst = dst;
    t.in = in.st;
    t.out = out.st;
    t.heads = static_cast<int>(heads);
    t.rotate = rotate ? 1 : 0;
    t.cache = cache ? 1 : 0;
    *wide = *wide && in.aligned16 && out.aligned16 && aligned16(src) && aligned16(dst);
    return FA_OK;
}

int launch_rotary(int dev, hipStream_t stream, int dtype, RotParams* p, bool wide) {
    const int w = static_cast<int>(16 / elem_size(dtype));
    const int run = p->interleaved ? p->rot : p->rot / 2;   // columns that a unit's runs divide
    wide = wide && run % w == 0 && (p->d - p->rot) % w == 0;
    p->cols = wide ? run / w + (p->d - p->rot) / w : p->rot / 2 + p->d - p->rot;
    const size_t tokens = static_cast<size_t>(p->batch) * p->seq;
    int heads = 1;
    for (int i = 0; i < p->nt; ++i) heads = std::max(heads, p->t[i].heads);
    // threads that share a token's heads: eight heads each where there are tokens enough to fill the GPU
    size_t ht = std::max(1, heads / 8);
    const size_t fill = static_cast<size_t>(g_dev[dev].num_cus) * 2048;
    while (ht < static_cast<size_t>(heads) && tokens * p->cols * ht < fill) ht *= 2;
    p->hthreads = static_cast<int>(std::min<size_t>(ht, heads));
    const size_t grid = (tokens * p->cols * p->hthreads + 255) / 256;
    if (grid > kOpsMaxGrid) return FA_ERR_UNSUPPORTED;
    char name[64];
    std::snprintf(name, sizeof(name), "fa_rotary_%s_%d", dtype_name(dtype), wide ? 1 : 0);
    return ops_launch(dev, kRotaryModule, name, grid, 256, p, stream);
}

}  // namespace

namespace {

// The largest distance between a query and a key, and how much that of the rows that fill up a block passes it.
constexpr int kWindowPast = 4096;
int64_t score_farthest(const fa_score_config& c) {
    const int64_t first = c.q_start, last = first + static_cast<int64_t>(c.seq_len_q) - 1;
    return std::max(std::abs(last), std::abs(first - (static_cast<int64_t>(c.seq_len_k) - 1)));
}

int score_forward(void* stream_, const fa_score_config* c, const fa_window* window, const void* q, const void* k,
                  const void* v, void* out, float* lse) {
    int rc = check_score(c);
    if (rc != FA_OK) return rc;
    if (c->batch == 0 || c->heads == 0 || c->seq_len_q == 0 || c->d_head == 0) return FA_OK;
    const size_t es = elem_size(c->dtype), d = c->d_head;
    ScoreScale sc;
    OpsLayout lq, lk, lv, lo;
    if ((rc = resolve_scale(c->softmax_scale, c->softcap, d, &sc)) != FA_OK ||
        (rc = resolve_layout(c->q, c->batch, c->seq_len_q, c->heads, d, es, false, &lq)) != FA_OK ||
        (rc = resolve_layout(c->k, c->batch, c->seq_len_k, c->kv_heads, d, es, false, &lk)) != FA_OK ||
        (rc = resolve_layout(c->v, c->batch, c->seq_len_k, c->kv_heads, d, es, false, &lv)) != FA_OK ||
        (rc = resolve_layout(c->out, c->batch, c->seq_len_q, c->heads, d, es, true, &lo)) != FA_OK)
        return rc;
    int size, sinks;
    if ((rc = resolve_window(window, c->q_doc, score_farthest(*c), kWindowPast, &size, &sinks)) != FA_OK) return rc;
    if (!q || !out || (c->seq_len_k > 0 && (!k || !v))) return FA_ERR_INVALID_ARG;
    const int D = ops_pad_d(d);
    if (c->batch * c->heads > kOpsMaxGrid || (c->seq_len_q + 31) / 32 * c->batch * c->heads > kOpsMaxGrid)
        return FA_ERR_UNSUPPORTED;
    int dev;
    const OpsModule module = of_type(size ? kScoreWindowModule : kScoreModule, c->dtype);
    if ((rc = ops_begin(&dev, module)) != FA_OK) return rc;
    const hipStream_t stream = static_cast<hipStream_t>(stream_);
    const bool vec = vec_ok(q, lq, d) && vec_ok(k, lk, d) && vec_ok(v, lv, d) && ovec_ok(out, lo, es) &&
                     cap_ok(c->dtype, c->softcap);

    const bool both_sides = !c->causal || c->prefix;
    const size_t keys = window_keys(c->seq_len_k, size, sinks, c->seq_len_q, both_sides);
    if (score_takes_rows(*c, keys, window_keys(c->seq_len_k, size, sinks, 32, both_sides), g_dev[dev].num_cus)) {
        RowsParams p{};
        p.q = q, p.k = k, p.v = v, p.out = out, p.lse = lse;
        p.slopes = c->slopes, p.q_doc = c->q_doc, p.k_doc = c->k_doc, p.prefix = c->causal ? c->prefix : nullptr;
        p.qs = lq.st, p.ks = lk.st, p.vs = lv.st, p.os = lo.st;
        p.batch = static_cast<int>(c->batch), p.heads = static_cast<int>(c->heads);
        p.kv_heads = static_cast<int>(c->kv_heads), p.group = static_cast<int>(c->heads / c->kv_heads);
        p.n = static_cast<int>(c->seq_len_q), p.sk = static_cast<int>(c->seq_len_k), p.d = static_cast<int>(d);
        p.causal = c->causal ? 1 : 0, p.q_start = static_cast<int>(c->q_start);
        p.scale_log2e = sc.scale_log2e, p.cap_in = sc.cap_in, p.cap_log2e = sc.cap_log2e;
        p.window = size, p.sinks = sinks;
        return run_rows(dev, stream, c->dtype, D, vec, &p, keys);
    }
    ScoreParams p{};
    fill_score(*c, sc, &p);
    p.window = size, p.sinks = sinks;
    p.q = q, p.k = k, p.v = v, p.out = out, p.lse = lse;
    p.qs = lq.st, p.ks = lk.st, p.vs = lv.st, p.os = lo.st;
    const ScoreTiles tiles = score_tiles(*c, D, vec, c->seq_len_q, c->batch * c->heads, g_dev[dev].num_cus);
    p.nqb = static_cast<int>((c->seq_len_q + tiles.rows - 1) / tiles.rows);
    OpsWorkspace ws;
    if (c->q_doc) {
        const DocPlan docs = plan_docs(*c, tiles.rows, c->heads, 0, 0, g_dev[dev].num_cus);
        if ((rc = ws.get(dev, stream, docs.bytes)) != FA_OK) return rc;
        rc = launch_docs(dev, module, stream, docs, tiles.rows, 0, &p, static_cast<int32_t*>(ws.ptr));
    }
    if (rc == FA_OK) {
        char name[64];
        std::snprintf(name, sizeof(name), "fa_score_forward_%s_d%d_t%d%s%s", dtype_name(c->dtype), D, tiles.mt,
                      tiles.tag, score_tag(*c, vec, size > 0));
        rc = ops_launch(dev, module, name, c->batch * c->heads * p.nqb, 256, &p, stream);
    }
    return ws.done(stream, rc);
}

int score_backward(void* stream_, const fa_score_config* c, const fa_window* window, const void* q, const void* k,
                   const void* v, const void* out, const float* lse, const void* dout, void* dq, void* dk, void* dv) {
    int rc = check_score(c);
    if (rc != FA_OK) return rc;
    if (c->batch == 0 || c->heads == 0 || c->d_head == 0) return FA_OK;
    if (c->seq_len_q == 0 && c->seq_len_k == 0) return FA_OK;
    const size_t es = elem_size(c->dtype), d = c->d_head, sq = c->seq_len_q, sk = c->seq_len_k;
    ScoreScale sc;
    OpsLayout lq, lk, lv, lo, ldo, ldq, ldk, ldv;
    if ((rc = resolve_scale(c->softmax_scale, c->softcap, d, &sc)) != FA_OK ||
        (rc = resolve_layout(c->q, c->batch, sq, c->heads, d, es, false, &lq)) != FA_OK ||
        (rc = resolve_layout(c->k, c->batch, sk, c->kv_heads, d, es, false, &lk)) != FA_OK ||
        (rc = resolve_layout(c->v, c->batch, sk, c->kv_heads, d, es, false, &lv)) != FA_OK ||
        (rc = resolve_layout(c->out, c->batch, sq, c->heads, d, es, true, &lo)) != FA_OK ||
        (rc = resolve_layout(c->dout, c->batch, sq, c->heads, d, es, false, &ldo)) != FA_OK ||
        (rc = resolve_layout(c->dq, c->batch, sq, c->heads, d, es, true, &ldq)) != FA_OK ||
        (rc = resolve_layout(c->dk, c->batch, sk, c->kv_heads, d, es, true, &ldk)) != FA_OK ||
        (rc = resolve_layout(c->dv, c->batch, sk, c->kv_heads, d, es, true, &ldv)) != FA_OK)
        return rc;
    int size, sinks;
    if ((rc = resolve_window(window, c->q_doc, score_farthest(*c), kWindowPast, &size, &sinks)) != FA_OK) return rc;
    if (sq > 0 && (!q || !out || !lse || !dout)) return FA_ERR_INVALID_ARG;
    if (sk > 0 && (!k || !v)) return FA_ERR_INVALID_ARG;
    const int D = ops_pad_d(d);
    const size_t rows = c->batch * c->heads * sq;
    if (c->batch * c->heads > kOpsMaxGrid || (sq + 31) / 32 * c->batch * c->heads > kOpsMaxGrid ||
        (sk + 31) / 32 * c->batch * c->heads > kOpsMaxGrid)
        return FA_ERR_UNSUPPORTED;
    int dev;
    const OpsModule module = of_type(size ? kScoreWindowModule : kScoreModule, c->dtype);
    if ((rc = ops_begin(&dev, module)) != FA_OK) return rc;
    const hipStream_t stream = static_cast<hipStream_t>(stream_);
    ScoreParams p{};
    fill_score(*c, sc, &p);
    p.window = size, p.sinks = sinks;
    p.q = q, p.k = k, p.v = v, p.out_in = out, p.dout = dout, p.lse_in = lse;
    p.dq = dq, p.dk = dk, p.dv = dv;
    p.qs = lq.st, p.ks = lk.st, p.vs = lv.st, p.os = lo.st, p.dos = ldo.st;
    p.dqs = ldq.st, p.dks = ldk.st, p.dvs = ldv.st;
    const bool vec = vec_ok(q, lq, d) && vec_ok(k, lk, d) && vec_ok(v, lv, d) && vec_ok(out, lo, d) &&
                     vec_ok(dout, ldo, d) && ovec_ok(dq, ldq, es) && ovec_ok(dk, ldk, es) && ovec_ok(dv, ldv, es) &&
                     cap_ok(c->dtype, c->softcap);
    OpsWorkspace ws;
    const DkvPlan dkv = plan_dkv(*c, D, vec, size, g_dev[dev].num_cus);
    ScoreTiles tiles = score_tiles(*c, D, vec, sq, c->batch * c->heads, g_dev[dev].num_cus);
    if (D == 128 && tiles.mt == 2) tiles = {1, 1, 64, ""};   // two tiles' Q, dO and sums leave one wave a SIMD
    const DocPlan docs = plan_docs(*c, tiles.rows, c->heads, dkv.tiles.rows, c->kv_heads * dkv.splits, g_dev[dev].num_cus);
    // partial sums first: they are read and written 16 bytes at a time
    const FarPlan far = dk || dv ? plan_far(*c, D, dkv, size, sinks) : FarPlan{};
    const size_t floats = dk || dv ? dkv.floats : 0;
    if ((rc = ws.get(dev, stream, (floats + far.floats + 2 * rows) * sizeof(float) + docs.bytes + 16)) != FA_OK) return rc;
    p.part = static_cast<float*>(ws.ptr);
    p.far_part = p.part + floats;
    p.lse2 = p.far_part + far.floats;
    p.delta = p.lse2 + rows;
    char name[64];
    if (c->q_doc)
        rc = launch_docs(dev, module, stream, docs, tiles.rows, dkv.tiles.rows, &p,
                         reinterpret_cast<int32_t*>(p.delta + rows));
    const char* mod = score_tag(*c, vec, size > 0);
    // the dQ kernel also forms delta and lse2, and with 16-bit types corrects delta, for the other one
    if (rc == FA_OK && sq > 0) {
        p.nqb = static_cast<int>((sq + tiles.rows - 1) / tiles.rows);
        std::snprintf(name, sizeof(name), "fa_score_dq_%s_d%d_t%d%s%s", dtype_name(c->dtype), D, tiles.mt, tiles.tag, mod);
        rc = ops_launch(dev, module, name, c->batch * c->heads * p.nqb, 256, &p, stream);
    }
    if (rc == FA_OK && (dk || dv)) {
        p.nqb = static_cast<int>(dkv.blocks);
        p.splits = dkv.splits;
        std::snprintf(name, sizeof(name), "fa_score_dkv_%s_d%d_t%d%s%s", dtype_name(c->dtype), D, dkv.tiles.mt,
                      dkv.tiles.tag, mod);
        const size_t slices = c->batch * c->kv_heads, grid = dkv.blocks * slices * dkv.splits;
        p.far_first = static_cast<int>(grid);
        p.far_stages = far.stages, p.far_chunks = far.chunks, p.far_splits = far.splits, p.far_blocks = far.blocks;
        p.far_rows = far.blocks * dkv.tiles.rows;
        rc = ops_launch(dev, module, name, grid + slices * far.splits * far.blocks * far.chunks, 256, &p, stream);
        if (rc == FA_OK && (dkv.splits > 1 || far.blocks)) {
            std::snprintf(name, sizeof(name), "fa_score_dkv_sum_%s_d%d%s", dtype_name(c->dtype), D, vec ? "" : "s");
            const size_t threads = slices * (dkv.splits > 1 ? sk : std::min<size_t>(sk, p.far_rows)) * (D / 4);
            rc = ops_launch(dev, module, name, (threads + 255) / 256, 256, &p, stream);
        }
    }
    return ws.done(stream, rc);
}

int tree_attention(void* stream, const fa_tree_config* c, const fa_window* window, const fa_kv_cache* cache,
                   const void* q, void* out, float* lse) {
    OpsLayout ck, cv, lq, lo;
    size_t capacity = 0;
    int rc = check_cache(cache, &ck, &cv, &capacity);
    if (rc != FA_OK) return rc;
    if (!c) return FA_ERR_INVALID_ARG;
    if (cache->batch == 0 || c->heads == 0 || c->n_tokens == 0 || cache->d_head == 0) return FA_OK;
    if (cache->kv_heads == 0 || c->heads % cache->kv_heads != 0) return FA_ERR_INVALID_ARG;
    if (c->heads > kOpsMaxSeq || c->n_tokens > kTreeMaxTokens) return FA_ERR_UNSUPPORTED;
    const size_t es = elem_size(cache->dtype), d = cache->d_head, n = c->n_tokens;
    ScoreScale sc;
    if ((rc = resolve_scale(c->softmax_scale, c->softcap, d, &sc)) != FA_OK ||
        (rc = resolve_layout(c->q, cache->batch, n, c->heads, d, es, false, &lq)) != FA_OK ||
        (rc = resolve_layout(c->out, cache->batch, n, c->heads, d, es, true, &lo)) != FA_OK)
        return rc;
    int size, sinks;
    if ((rc = resolve_window(window, false, kWindowMaxPos, 0, &size, &sinks)) != FA_OK) return rc;
    if (!q || !out) return FA_ERR_INVALID_ARG;
    if (cache->batch * c->heads > kOpsMaxGrid) return FA_ERR_UNSUPPORTED;
    RowsParams p{};
    p.q = q, p.k = cache->k, p.v = cache->v, p.out = out, p.lse = lse;
    p.slopes = c->slopes, p.lens = cache->lens, p.table = cache->block_table;
    p.pos = c->positions, p.mask = c->mask;
    p.qs = lq.st, p.ks = ck.st, p.vs = cv.st, p.os = lo.st;
    p.batch = static_cast<int>(cache->batch), p.heads = static_cast<int>(c->heads);
    p.kv_heads = static_cast<int>(cache->kv_heads), p.group = static_cast<int>(c->heads / cache->kv_heads);
    p.n = static_cast<int>(n), p.sk = static_cast<int>(capacity), p.d = static_cast<int>(d);
    p.page_shift = page_shift(*cache);
    p.n_pages = static_cast<int>(cache->n_pages), p.pages_per_seq = static_cast<int>(cache->pages_per_seq);
    p.mask_words = static_cast<int>((n + 63) / 64), p.mask_shared = c->mask_shared ? 1 : 0;
    p.window = size, p.sinks = sinks;
    const bool vec = vec_ok(q, lq, d) && vec_ok(cache->k, ck, d) && vec_ok(cache->v, cv, d) && ovec_ok(out, lo, es) &&
                     cap_ok(cache->dtype, c->softcap);
    p.scale_log2e = sc.scale_log2e, p.cap_in = sc.cap_in, p.cap_log2e = sc.cap_log2e;
    int dev;
    if ((rc = ops_begin(&dev, cache_module(cache->dtype, p))) != FA_OK) return rc;
    return run_rows(dev, static_cast<hipStream_t>(stream), cache->dtype, ops_pad_d(d), vec, &p,
                    window_keys(capacity, size, sinks, n, false));
}

// Norms with rotary positions: one tensor of a launch, checked; *wide: whether 16-byte loads and stores do for all so far.
int add_norm_tensor(NormParams* p, bool* wide, size_t batch, size_t seq, size_t d, size_t es, size_t heads,
                    const void* x, const fa_strides& xs, const void* dy, const fa_strides* dys, void* out,
                    const OpsLayout& lo, bool norm, const void* w, bool cache) {
    OpsLayout lx, ldy;
    int rc = resolve_layout(xs, batch, seq, heads, d, es, false, &lx);
    if (rc == FA_OK && dys) rc = resolve_layout(*dys, batch, seq, heads, d, es, false, &ldy);
    if (rc != FA_OK) return rc;
    NormTensor& t = p->t[p->nt++];
    t.x = x, t.dy = dy, t.w = w, t.out = out;
    t.xs = lx.st, t.dys = ldy.st, t.outs = lo.st;
    t.heads = static_cast<int>(heads);
    t.norm = norm ? 1 : 0, t.cache = cache ? 1 : 0;
    *wide = *wide && lx.aligned16 && ldy.aligned16 && lo.aligned16 && aligned16(x) && aligned16(dy) && aligned16(out);
    return FA_OK;
}
bool same_strides(const OpsStrides& a, const OpsStrides& b) { return a.b == b.b && a.s == b.s && a.h == b.h; }

void fill_norm(const fa_rotary_config& c, const fa_head_norm& norm, size_t batch, size_t seq, const int32_t* positions,
               NormParams* p) {
    p->batch = static_cast<int>(batch);
    p->seq = static_cast<int>(seq);
    p->d = static_cast<int>(c.d_head);
    p->rot = static_cast<int>(c.rot_dim);
    p->interleaved = c.interleaved ? 1 : 0;
    p->pos = positions;
    p->gain = c.gain;
    p->eps = norm.eps;
    std::memcpy(p->turns, c.turns, sizeof(p->turns));
}
int check_norm(const fa_rotary_config* c, const fa_head_norm* n) {
    const int rc = check_rotary(c);
    if (rc != FA_OK) return rc;
    return n && n->eps > 0.0f && std::isfinite(n->eps) ? FA_OK : FA_ERR_INVALID_ARG;
}

// The kernel's kind, lanes of a row and tokens of a workgroup.
int plan_norm(int dev, int dtype, bool wide, NormParams* p, const char** kind, size_t* grid) {
    const int w = static_cast<int>(16 / elem_size(dtype));
    const int run = p->interleaved ? p->rot : p->rot / 2;
    wide = wide && run % w == 0 && (p->d - p->rot) % w == 0;
    p->units = wide ? run / w + (p->d - p->rot) / w : p->rot / 2 + p->d - p->rot;
    auto power = [](int n) {
        int l = 1;
        while (l < 64 && l < n) l *= 2;
        return l;
    };
    p->lanes = power(p->units);
    // three units a lane where that leaves fewer lanes idle (20 units: 24 places instead of 32; 2 x 1000 tokens of 16 + 16
    // heads of 80 columns, 40 of them rotary, f32)
    const bool three = wide && (p->interleaved || dtype == FA_DTYPE_F32) && p->units > 2 && 3 * power((p->units + 2) / 3) < p->lanes;
    if (three) p->lanes = power((p->units + 2) / 3);
    const bool full = wide && !three && p->rot == p->d && p->units == p->lanes;
    *kind = !wide ? "0" : full ? (p->interleaved ? "fi" : "f") : three ? (p->interleaved ? "3i" : "3") : p->interleaved ? "1i" : "1";
    const size_t slots = kNormThreads / p->lanes, all = static_cast<size_t>(p->batch) * p->seq;
    *grid = 0;
    for (int i = 0; i < p->nt; ++i) {
        NormTensor& t = p->t[i];
        // some four rows a slot, so that the next is on its way while one is worked on, where that leaves two workgroups a
        // CU, all tensors together; a row for each slot where it leaves one
        size_t tokens = 1;
        const size_t cus = static_cast<size_t>(g_dev[dev].num_cus);
        while (tokens < kNormTokens && tokens * t.heads < 4 * slots &&
               all * p->nt / (2 * tokens) >= (tokens * t.heads < slots ? 1 : 2) * cus)
            tokens *= 2;
        t.tokens = static_cast<int>(tokens);
        const size_t blocks = (all + tokens - 1) / tokens;
        if (blocks > kOpsMaxGrid) return FA_ERR_UNSUPPORTED;
        t.blocks = static_cast<int>(blocks);
        *grid += blocks;
    }
    return *grid > kOpsMaxGrid ? FA_ERR_UNSUPPORTED : FA_OK;
}
int launch_norm(int dev, hipStream_t stream, int dtype, NormParams* p, bool wide) {
    size_t grid;
    const char* kind;
    const int rc = plan_norm(dev, dtype, wide, p, &kind, &grid);
    if (rc != FA_OK) return rc;
    char name[64];
    std::snprintf(name, sizeof(name), "fa_norm_%s_%s", dtype_name(dtype), kind);
    return ops_launch(dev, kNormModule, name, grid, kNormThreads, p, stream);
}

// A cache in 4 bits: rows of a block of memory, and of a sequence.
int check_cache4(const fa_kv_cache4* c, size_t* block_rows, size_t* capacity) {
    if (!c || !valid_dtype(c->dtype)) return FA_ERR_INVALID_ARG;
    if (c->batch == 0 || c->kv_heads == 0 || c->d_head == 0) return FA_OK;
    if (c->dtype == FA_DTYPE_F32 || c->d_head > kOpsMaxD || c->d_head % 32 != 0 || c->batch > kOpsMaxSeq ||
        c->kv_heads > kOpsMaxSeq)
        return FA_ERR_UNSUPPORTED;
    if (!c->lens) return FA_ERR_INVALID_ARG;
    if (c->block_table) {
        if (c->page_size < 8 || (c->page_size & (c->page_size - 1)) != 0) return FA_ERR_INVALID_ARG;
        if (c->page_size > kOpsMaxSeq || c->pages_per_seq > kOpsMaxSeq || c->n_pages > kOpsMaxSeq)
            return FA_ERR_UNSUPPORTED;
        *block_rows = c->page_size;
        *capacity = c->page_size * c->pages_per_seq;
    } else {
        if (c->capacity % 8 != 0) return FA_ERR_INVALID_ARG;
        *block_rows = *capacity = c->capacity;
    }
    if (*capacity > kOpsMaxSeq) return FA_ERR_UNSUPPORTED;
    // rows of all heads are numbered in 32 bits (2^32 of 64 columns have 172 GB)
    const size_t heads = (c->block_table ? c->n_pages : c->batch) * c->kv_heads;
    if (*block_rows > 0 && heads >= (size_t(1) << 32) / *block_rows) return FA_ERR_UNSUPPORTED;
    if (*capacity > 0 && (!c->k || !c->v || !c->k_scale || !c->v_scale)) return FA_ERR_INVALID_ARG;
    // the kernels load words of it, 16 bytes at a time
    if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_scale) || !aligned16(c->v_scale)) return FA_ERR_INVALID_ARG;
    return FA_OK;
}
int page_shift4(const fa_kv_cache4& c) {
    int s = 0;
    while (c.block_table && (size_t(1) << s) < c.page_size) ++s;
    return s;
}
void fill_cache4(const fa_kv_cache4& c, size_t block_rows, size_t capacity, Cache4Params* p) {
    p->k4 = c.k, p->v4 = c.v, p->kscale = c.k_scale, p->vscale = c.v_scale;
    p->lens = c.lens, p->table = c.block_table;
    p->batch = static_cast<int>(c.batch), p->kv_heads = static_cast<int>(c.kv_heads), p->d = static_cast<int>(c.d_head);
    p->capacity = static_cast<int>(capacity), p->block_rows = static_cast<int>(block_rows);
    p->page_shift = page_shift4(c);
    p->n_pages = static_cast<int>(c.n_pages), p->pages_per_seq = static_cast<int>(c.pages_per_seq);
}
OpsModule cache4_module(int dtype, int window) {
    return static_cast<OpsModule>((window ? kCache4WindowModule : kCache4Module) + (dtype == FA_DTYPE_BF16 ? 0 : 1));
}

// Plan of attention over a cache in 4 bits.
RowsPlan plan_rows4(size_t d, bool plain, size_t batch, size_t kv_heads, size_t rows, size_t keys, int num_cus) {
    RowsPlan r{};
    // Two tiles a wave share what a code costs to become a number, but there are half as many workgroups: from more than
    // four steps of 128 keys a resident one on (d128, 8 sequences of up to 8000 keys, 256 rows 134 us with two, 156 with
    // one; 4 of 3000, 200 rows 26 and 24; four tiles, or two of 256 columns, leave one wave a SIMD: 252 us)
    const size_t cus = static_cast<size_t>(num_cus), steps = batch * keys * kv_heads * ((rows + 31) / 32) / (32 * kRows4Waves);
    r.mt = (d == 64 || d == 128) && rows > 16 && steps > 4 * 2 * cus ? 2 : 1;
    r.threads = 64 * kRows4Waves;
    r.rows = 16 * r.mt;
    r.step = 32 * kRows4Waves;
    // workgroups a CU that the registers leave room for
    const size_t resident = cus * (d > 128 ? 1 : r.mt > 1 || !plain ? 2 : d > 64 ? 3 : 4);
    share_keys(&r, batch, kv_heads, rows, keys, resident, 4 * r.step, ops_pad_d(d));
    return r;
}

}  // namespace

extern "C" {

int fa_score_forward(void* stream, const fa_score_config* c, const void* q, const void* k, const void* v, void* out,
                     float* lse) try {
    return score_forward(stream, c, nullptr, q, k, v, out, lse);
} catch (...) {   // no memory for the tables of modules, kernels and workspaces
    return FA_ERR_ALLOC;
}

int fa_window_forward(void* stream, const fa_score_config* c, const fa_window* window, const void* q, const void* k,
                      const void* v, void* out, float* lse) try {
    return score_forward(stream, c, window, q, k, v, out, lse);
} catch (...) {   // no memory for the tables of modules, kernels and workspaces
    return FA_ERR_ALLOC;
}

int fa_score_backward(void* stream, const fa_score_config* c, const void* q, const void* k, const void* v,
                      const void* out, const float* lse, const void* dout, void* dq, void* dk, void* dv) try {
    return score_backward(stream, c, nullptr, q, k, v, out, lse, dout, dq, dk, dv);
} catch (...) {   // no memory for the tables of modules, kernels and workspaces
    return FA_ERR_ALLOC;
}

int fa_window_backward(void* stream, const fa_score_config* c, const fa_window* window, const void* q, const void* k,
                       const void* v, const void* out, const float* lse, const void* dout, void* dq, void* dk,
                       void* dv) try {
    return score_backward(stream, c, window, q, k, v, out, lse, dout, dq, dk, dv);
} catch (...) {   // no memory for the tables of modules, kernels and workspaces
    return FA_ERR_ALLOC;
}

int fa_rotary_init(fa_rotary_config* cfg, int dtype, size_t d_head, size_t rot_dim, int interleaved, double base,
                   int scaling, double factor, double original_len) {
    if (!cfg) return FA_ERR_INVALID_ARG;
    std::memset(cfg, 0, sizeof(*cfg));
    cfg->dtype = dtype;
    cfg->interleaved = interleaved ? 1 : 0;
    cfg->d_head = d_head;
    cfg->rot_dim = rot_dim;
    cfg->gain = 1.0f;
    const int rc = check_rotary(cfg);
    if (rc != FA_OK) return rc;
    if (!(base > 1.0) || !std::isfinite(base)) return FA_ERR_INVALID_ARG;
    if (scaling < FA_ROTARY_NONE || scaling > FA_ROTARY_YARN) return FA_ERR_INVALID_ARG;
    if (scaling != FA_ROTARY_NONE && (!(factor >= 1.0) || !std::isfinite(factor))) return FA_ERR_INVALID_ARG;
    if (scaling == FA_ROTARY_NTK && rot_dim == 2) return FA_ERR_INVALID_ARG;   // its exponent has no value
    if (scaling == FA_ROTARY_YARN && (!(original_len > 0.0) || !std::isfinite(original_len))) return FA_ERR_INVALID_ARG;
    const double two_pi = 6.283185307179586476925, rot = static_cast<double>(rot_dim);
    if (scaling == FA_ROTARY_NTK) base *= std::pow(factor, rot / (rot - 2.0));
    double lo = 0.0, hi = 0.0;
    if (scaling == FA_ROTARY_YARN) {
        // pair index at which a pair makes that many turns over the trained length
        auto index = [&](double turns) { return rot * std::log(original_len / (turns * two_pi)) / (2.0 * std::log(base)); };
        lo = std::max(std::floor(index(32.0)), 0.0);
        hi = std::min(std::ceil(index(1.0)), rot - 1.0);
        cfg->gain = static_cast<float>(0.1 * std::log(factor) + 1.0);
    }
    for (size_t c = 0; c < rot_dim / 2; ++c) {
        double f = std::pow(base, -2.0 * static_cast<double>(c) / rot) / two_pi;
        if (scaling == FA_ROTARY_LINEAR) f /= factor;
        if (scaling == FA_ROTARY_YARN) {
            const double ramp =
                std::min(1.0, std::max(0.0, (static_cast<double>(c) - lo) / std::max(hi - lo, 0.001)));
            f = f / factor * ramp + f * (1.0 - ramp);
        }
        cfg->turns[c] = f;
    }
    return FA_OK;
}

int fa_rotary(void* stream, const fa_rotary_config* cfg, size_t batch, size_t seq_len, const int32_t* positions,
              int inverse, const fa_rotary_tensor* ql, const void* q, void* q_out, const fa_rotary_tensor* kl,
              const void* k, void* k_out) try {
    int rc = check_rotary(cfg);
    if (rc != FA_OK) return rc;
    if (!ql) return FA_ERR_INVALID_ARG;
    if (batch == 0 || seq_len == 0) return FA_OK;
    if (batch > kOpsMaxSeq || seq_len > kOpsMaxSeq || batch * seq_len > kOpsMaxTokens) return FA_ERR_UNSUPPORTED;
    if (!positions) return FA_ERR_INVALID_ARG;
    RotParams p{};
    bool wide = true;
    for (int n = 0; n < (kl ? 2 : 1); ++n) {
        const fa_rotary_tensor* t = n ? kl : ql;
        const void* src = n ? k : q;
        void* dst = n ? k_out : q_out;
        if (t->heads == 0) continue;
        if (t->heads > kOpsMaxSeq) return FA_ERR_UNSUPPORTED;
        OpsLayout in, out;
        if ((rc = resolve_layout(t->in, batch, seq_len, t->heads, cfg->d_head, elem_size(cfg->dtype), false, &in)) !=
                FA_OK ||
            (rc = resolve_layout(t->out, batch, seq_len, t->heads, cfg->d_head, elem_size(cfg->dtype), true, &out)) !=
                FA_OK)
            return rc;
        if (!src || !dst) return FA_ERR_INVALID_ARG;
        // in place the layouts have to agree: a thread reads what it writes
        if (src == dst && (in.st.b != out.st.b || in.st.s != out.st.s || in.st.h != out.st.h)) return FA_ERR_INVALID_ARG;
        add_rotary_tensor(&p, src, dst, in, out, t->heads, true, false, &wide);
    }
    if (p.nt == 0) return FA_OK;
    p.batch = static_cast<int>(batch);
    p.seq = static_cast<int>(seq_len);
    p.d = static_cast<int>(cfg->d_head);
    p.rot = static_cast<int>(cfg->rot_dim);
    p.interleaved = cfg->interleaved ? 1 : 0;
    p.pos = positions;
    p.gain = cfg->gain;
    p.sign = inverse ? -1.0f : 1.0f;
    std::memcpy(p.turns, cfg->turns, sizeof(p.turns));
    int dev;
    if ((rc = ops_begin(&dev, kRotaryModule)) != FA_OK) return rc;
    return launch_rotary(dev, static_cast<hipStream_t>(stream), cfg->dtype, &p, wide);
} catch (...) {   // no memory for the tables of modules, kernels and workspaces
    return FA_ERR_ALLOC;
}

int fa_norm_rotary(void* stream, const fa_rotary_config* cfg, const fa_head_norm* norm, size_t batch, size_t seq_len,
                   const int32_t* positions, const fa_rotary_tensor* ql, const void* q, void* q_out,
                   const fa_rotary_tensor* kl, const void* k, void* k_out) try {
    int rc = check_norm(cfg, norm);
    if (rc != FA_OK) return rc;
    if (!ql) return FA_ERR_INVALID_ARG;
    if (batch == 0 || seq_len == 0) return FA_OK;
    if (batch > kOpsMaxSeq || seq_len > kOpsMaxSeq || batch * seq_len > kOpsMaxTokens) return FA_ERR_UNSUPPORTED;
    if (!positions) return FA_ERR_INVALID_ARG;
    NormParams p{};
    bool wide = true;
    const size_t d = cfg->d_head, es = elem_size(cfg->dtype);
    for (int n = 0; n < (kl ? 2 : 1); ++n) {
        const fa_rotary_tensor* t = n ? kl : ql;
        const void* src = n ? k : q;
        void* dst = n ? k_out : q_out;
        if (t->heads == 0) continue;
        if (t->heads > kOpsMaxSeq) return FA_ERR_UNSUPPORTED;
        OpsLayout out;
        if ((rc = resolve_layout(t->out, batch, seq_len, t->heads, d, es, true, &out)) != FA_OK) return rc;
        if (!src || !dst) return FA_ERR_INVALID_ARG;
        if ((rc = add_norm_tensor(&p, &wide, batch, seq_len, d, es, t->heads, src, t->in, nullptr, nullptr, dst, out, true,
                                  n ? norm->k_weight : norm->q_weight, false)) != FA_OK)
            return rc;
        // in place the layouts have to agree: a lane reads what it writes
        if (src == dst && !same_strides(p.t[p.nt - 1].xs, out.st)) return FA_ERR_INVALID_ARG;
    }
    if (p.nt == 0) return FA_OK;
    fill_norm(*cfg, *norm, batch, seq_len, positions, &p);
    int dev;
    if ((rc = ops_begin(&dev, kNormModule)) != FA_OK) return rc;
    return launch_norm(dev, static_cast<hipStream_t>(stream), cfg->dtype, &p, wide);
} catch (...) {   // no memory for the tables of modules, kernels and workspaces
    return FA_ERR_ALLOC;
}

int fa_norm_rotary_backward(void* stream_, const fa_rotary_config* cfg, const fa_head_norm* norm, size_t batch,
                            size_t seq_len, const int32_t* positions, const fa_norm_grad* qg, const void* q,
                            const void* dq_out, void* dq, float* dq_weight, const fa_norm_grad* kg, const void* k,
                            const void* dk_out, void* dk, float* dk_weight) try {
    int rc = check_norm(cfg, norm);
    if (rc != FA_OK) return rc;
    if (!qg) return FA_ERR_INVALID_ARG;
    if (batch > kOpsMaxSeq || seq_len > kOpsMaxSeq || (seq_len > 0 && batch > kOpsMaxTokens / seq_len))
        return FA_ERR_UNSUPPORTED;
    const bool any = batch > 0 && seq_len > 0;
    if (any && !positions) return FA_ERR_INVALID_ARG;
    NormParams p{};
    bool wide = true;
    const size_t d = cfg->d_head, es = elem_size(cfg->dtype);
    bool weights = false;
    for (int n = 0; n < (kg ? 2 : 1); ++n) {
        const fa_norm_grad* t = n ? kg : qg;
        const void *x = n ? k : q, *dy = n ? dk_out : dq_out;
        void* dx = n ? dk : dq;
        float* dw = n ? dk_weight : dq_weight;
        if (t->heads > kOpsMaxSeq) return FA_ERR_UNSUPPORTED;
        if (!dx && !dw) continue;
        if (!any || t->heads == 0) {   // the sums of no rows: zeros
            p.t[p.nt++].dw = dw;
            weights = weights || dw;
            continue;
        }
        OpsLayout out;
        if ((rc = resolve_layout(t->dx, batch, seq_len, t->heads, d, es, true, &out)) != FA_OK) return rc;
        if (!x || !dy) return FA_ERR_INVALID_ARG;
        if ((rc = add_norm_tensor(&p, &wide, batch, seq_len, d, es, t->heads, x, t->x, dy, &t->dout, dx, out, true,
                                  n ? norm->k_weight : norm->q_weight, false)) != FA_OK)
            return rc;
        NormTensor& added = p.t[p.nt - 1];
        if ((dx && dx == x && !same_strides(added.xs, out.st)) || (dx && dx == dy && !same_strides(added.dys, out.st)))
            return FA_ERR_INVALID_ARG;
        added.dw = dw;
        weights = weights || dw;
    }
    if (p.nt == 0) return FA_OK;
    fill_norm(*cfg, *norm, batch, seq_len, positions, &p);
    int dev;
    if ((rc = ops_begin(&dev, kNormModule)) != FA_OK) return rc;
    const hipStream_t stream = static_cast<hipStream_t>(stream_);
    // tensors without rows are left out of the first launch
    NormParams rows = p;
    rows.nt = 0;
    int from[3];
    for (int i = 0; i < p.nt; ++i)
        if (p.t[i].heads > 0) {
            from[rows.nt] = i;
            rows.t[rows.nt++] = p.t[i];
        }
    OpsWorkspace ws;
    if (rows.nt > 0) {
        size_t grid;
        const char* kind;
        if ((rc = plan_norm(dev, cfg->dtype, wide, &rows, &kind, &grid)) != FA_OK) return rc;
        if (weights) {
            if ((rc = ws.get(dev, stream, grid * d * sizeof(float))) != FA_OK) return rc;
            float* part = static_cast<float*>(ws.ptr);
            for (int i = 0; i < rows.nt; ++i) {
                rows.t[i].part = rows.t[i].dw ? part : nullptr;
                part += rows.t[i].blocks * d;
                p.t[from[i]] = rows.t[i];
            }
        }
        char name[64];
        std::snprintf(name, sizeof(name), "fa_norm_back_%s_%s", dtype_name(cfg->dtype), kind);
        rc = ops_launch(dev, kNormModule, name, grid, kNormThreads, &rows, stream);
    }
    if (rc == FA_OK && weights) rc = ops_launch(dev, kNormModule, "fa_norm_weights", p.nt * ((d + kNormColumns - 1) / kNormColumns), 1024, &p,
                                              stream);
    return ws.done(stream, rc);
} catch (...) {   // no memory for the tables of modules, kernels and workspaces
    return FA_ERR_ALLOC;
}

int fa_norm_cache_append(void* stream, const fa_kv_cache* cache, const fa_append_config* cfg, const fa_head_norm* norm,
                         const void* k, const void* v, const int32_t* positions, const void* q, void* q_out) try {
    OpsLayout ck, cv;
    size_t capacity = 0;
    int rc = check_cache(cache, &ck, &cv, &capacity);
    if (rc != FA_OK) return rc;
    if (!cfg) return FA_ERR_INVALID_ARG;
    const fa_rotary_config* rot = cfg->rotary;
    if ((rc = check_norm(rot, norm)) != FA_OK) return rc;
    if (rot->dtype != cache->dtype || rot->d_head != cache->d_head) return FA_ERR_INVALID_ARG;
    if (cache->batch == 0 || cache->kv_heads == 0 || cache->d_head == 0 || cfg->n_tokens == 0) return FA_OK;
    const size_t es = elem_size(cache->dtype), d = cache->d_head, n = cfg->n_tokens;
    if (n > kOpsMaxSeq || cache->batch * n > kOpsMaxTokens) return FA_ERR_UNSUPPORTED;
    if (!k || !v || !positions) return FA_ERR_INVALID_ARG;
    NormParams p{};
    bool wide = true;
    // checked also where there is no room for a row
    if ((rc = add_norm_tensor(&p, &wide, cache->batch, n, d, es, cache->kv_heads, k, cfg->k, nullptr, nullptr, cache->k,
                              ck, true, norm->k_weight, true)) != FA_OK ||
        (rc = add_norm_tensor(&p, &wide, cache->batch, n, d, es, cache->kv_heads, v, cfg->v, nullptr, nullptr, cache->v,
                              cv, false, nullptr, true)) != FA_OK)
        return rc;
    if (capacity == 0) {
        p.nt = 0;
        wide = true;
    }
    if (cfg->q_layout && cfg->q_layout->heads > 0) {
        const fa_rotary_tensor* t = cfg->q_layout;
        OpsLayout out;
        if (t->heads > kOpsMaxSeq) return FA_ERR_UNSUPPORTED;
        if ((rc = resolve_layout(t->out, cache->batch, n, t->heads, d, es, true, &out)) != FA_OK) return rc;
        if (!q || !q_out) return FA_ERR_INVALID_ARG;
        if ((rc = add_norm_tensor(&p, &wide, cache->batch, n, d, es, t->heads, q, t->in, nullptr, nullptr, q_out, out,
                                  true, norm->q_weight, false)) != FA_OK)
            return rc;
        if (q == q_out && !same_strides(p.t[p.nt - 1].xs, out.st)) return FA_ERR_INVALID_ARG;
    }
    if (p.nt == 0) return FA_OK;
    fill_norm(*rot, *norm, cache->batch, n, positions, &p);
    p.lens = cache->lens;
    p.table = cache->block_table;
    p.capacity = static_cast<int>(capacity);
    p.page_shift = page_shift(*cache);
    p.n_pages = static_cast<int>(cache->n_pages);
    p.pages_per_seq = static_cast<int>(cache->pages_per_seq);
    int dev;
    if ((rc = ops_begin(&dev, kNormModule)) != FA_OK) return rc;
    return launch_norm(dev, static_cast<hipStream_t>(stream), cache->dtype, &p, wide);
} catch (...) {   // no memory for the tables of modules, kernels and workspaces
    return FA_ERR_ALLOC;
}

int fa_cache_append(void* stream, const fa_kv_cache* cache, const fa_append_config* cfg, const void* k, const void* v,
                    const int32_t* positions, const void* q, void* q_out) try {
    OpsLayout ck, cv, lk, lv;
    size_t capacity = 0;
    int rc = check_cache(cache, &ck, &cv, &capacity);
    if (rc != FA_OK) return rc;
    if (!cfg) return FA_ERR_INVALID_ARG;
    const fa_rotary_config* rot = cfg->rotary;
    if (rot && (rc = check_rotary(rot)) != FA_OK) return rc;
    if (rot && (rot->dtype != cache->dtype || rot->d_head != cache->d_head)) return FA_ERR_INVALID_ARG;
    if (cfg->q_layout && !rot) return FA_ERR_INVALID_ARG;
    if (cache->batch == 0 || cache->kv_heads == 0 || cache->d_head == 0 || cfg->n_tokens == 0) return FA_OK;
    const size_t es = elem_size(cache->dtype), d = cache->d_head, n = cfg->n_tokens;
    if (n > kOpsMaxSeq || cache->batch * n > kOpsMaxTokens) return FA_ERR_UNSUPPORTED;
    if ((rc = resolve_layout(cfg->k, cache->batch, n, cache->kv_heads, d, es, false, &lk)) != FA_OK ||
        (rc = resolve_layout(cfg->v, cache->batch, n, cache->kv_heads, d, es, false, &lv)) != FA_OK)
        return rc;
    if (!k || !v || (rot && !positions)) return FA_ERR_INVALID_ARG;
    RotParams p{};
    bool wide = true;
    if (capacity > 0) {
        add_rotary_tensor(&p, k, cache->k, lk, ck, cache->kv_heads, rot != nullptr, true, &wide);
        add_rotary_tensor(&p, v, cache->v, lv, cv, cache->kv_heads, false, true, &wide);
    }
    if (cfg->q_layout && cfg->q_layout->heads > 0) {
        const fa_rotary_tensor* t = cfg->q_layout;
        OpsLayout in, out;
        if (t->heads > kOpsMaxSeq) return FA_ERR_UNSUPPORTED;
        if ((rc = resolve_layout(t->in, cache->batch, n, t->heads, d, es, false, &in)) != FA_OK ||
            (rc = resolve_layout(t->out, cache->batch, n, t->heads, d, es, true, &out)) != FA_OK)
            return rc;
        if (!q || !q_out) return FA_ERR_INVALID_ARG;
        if (q == q_out && (in.st.b != out.st.b || in.st.s != out.st.s || in.st.h != out.st.h)) return FA_ERR_INVALID_ARG;
        add_rotary_tensor(&p, q, q_out, in, out, t->heads, true, false, &wide);
    }
    if (p.nt == 0) return FA_OK;
    p.batch = static_cast<int>(cache->batch);
    p.seq = static_cast<int>(n);
    p.d = static_cast<int>(d);
    p.pos = positions;
    p.lens = cache->lens;
    p.table = cache->block_table;
    p.capacity = static_cast<int>(capacity);
    p.page_shift = page_shift(*cache);
    p.n_pages = static_cast<int>(cache->n_pages);
    p.pages_per_seq = static_cast<int>(cache->pages_per_seq);
    p.sign = 1.0f;
    if (rot) {
        p.rot = static_cast<int>(rot->rot_dim);
        p.interleaved = rot->interleaved ? 1 : 0;
        p.gain = rot->gain;
        std::memcpy(p.turns, rot->turns, sizeof(p.turns));
    }
    int dev;
    if ((rc = ops_begin(&dev, kRotaryModule)) != FA_OK) return rc;
    return launch_rotary(dev, static_cast<hipStream_t>(stream), cache->dtype, &p, wide);
} catch (...) {   // no memory for the tables of modules, kernels and workspaces
    return FA_ERR_ALLOC;
}

int fa_tree_attention(void* stream, const fa_tree_config* c, const fa_kv_cache* cache, const void* q, void* out,
                      float* lse) try {
    return tree_attention(stream, c, nullptr, cache, q, out, lse);
} catch (...) {   // no memory for the tables of modules, kernels and workspaces
    return FA_ERR_ALLOC;
}

int fa_window_tree_attention(void* stream, const fa_tree_config* c, const fa_window* window, const fa_kv_cache* cache,
                             const void* q, void* out, float* lse) try {
    return tree_attention(stream, c, window, cache, q, out, lse);
} catch (...) {   // no memory for the tables of modules, kernels and workspaces
    return FA_ERR_ALLOC;
}

int fa_cache4_append(void* stream, const fa_kv_cache4* cache, const fa_append_config* cfg, const void* k,
                     const void* v) try {
    size_t block_rows = 0, capacity = 0;
    int rc = check_cache4(cache, &block_rows, &capacity);
    if (rc != FA_OK) return rc;
    if (!cfg) return FA_ERR_INVALID_ARG;
    if (cfg->rotary || cfg->q_layout) return FA_ERR_UNSUPPORTED;   // rows come as they are to be kept
    if (cache->batch == 0 || cache->kv_heads == 0 || cache->d_head == 0 || cfg->n_tokens == 0) return FA_OK;
    const size_t d = cache->d_head, n = cfg->n_tokens;
    if (n > kOpsMaxSeq || cache->batch * n > kOpsMaxTokens) return FA_ERR_UNSUPPORTED;
    OpsLayout lk, lv;
    if ((rc = resolve_layout(cfg->k, cache->batch, n, cache->kv_heads, d, 2, false, &lk)) != FA_OK ||
        (rc = resolve_layout(cfg->v, cache->batch, n, cache->kv_heads, d, 2, false, &lv)) != FA_OK)
        return rc;
    if (!k || !v) return FA_ERR_INVALID_ARG;
    if (capacity == 0) return FA_OK;
    Cache4Params p{};
    fill_cache4(*cache, block_rows, capacity, &p);
    p.k = k, p.v = v, p.ks = lk.st, p.vs = lv.st;
    p.n = static_cast<int>(n);
    p.vec = vec_ok(k, lk, d) && vec_ok(v, lv, d);
    const size_t runs = (n + 7) / 8 + 1, per = 256 / d;   // n rows touch that many runs of 8 at most
    const size_t heads = 2 * cache->batch * cache->kv_heads;
    int dev;
    const OpsModule module = cache4_module(cache->dtype, 0);
    if (heads > kOpsMaxGrid / ((runs + per - 1) / per)) return FA_ERR_UNSUPPORTED;
    if ((rc = ops_begin(&dev, module)) != FA_OK) return rc;
    // pieces enough a workgroup that all run at once, eight a CU: a last round of few costs as much as a full one (4 x 2048
    // rows of 8 heads of 128 columns, 64 workgroups of 2112 in a second round: 20 us)
    const size_t resident = 8 * static_cast<size_t>(g_dev[dev].num_cus), pieces = heads * ((runs + per - 1) / per);
    const size_t loops = std::min<size_t>(16, (pieces + resident - 1) / resident);
    const size_t parts = (runs + loops * per - 1) / (loops * per);
    p.nparts = static_cast<int>(parts);
    p.loops = static_cast<int>(loops);
    return ops_launch(dev, module, cache->dtype == FA_DTYPE_BF16 ? "fa_cache4_append_bf16" : "fa_cache4_append_f16",
                      heads * parts, 256, &p, static_cast<hipStream_t>(stream));
} catch (...) {   // no memory for the tables of modules, kernels and workspaces
    return FA_ERR_ALLOC;
}

int fa_cache4_read(void* stream, const fa_kv_cache4* cache, const fa_read_config* cfg, const int32_t* rows, void* k_out,
                   void* v_out) try {
    size_t block_rows = 0, capacity = 0;
    int rc = check_cache4(cache, &block_rows, &capacity);
    if (rc != FA_OK) return rc;
    if (!cfg) return FA_ERR_INVALID_ARG;
    if (cache->batch == 0 || cache->kv_heads == 0 || cache->d_head == 0 || cfg->n_rows == 0) return FA_OK;
    const size_t d = cache->d_head, n = cfg->n_rows;
    if (n > kOpsMaxSeq || cache->batch * n > kOpsMaxTokens) return FA_ERR_UNSUPPORTED;
    OpsLayout lk, lv;
    if ((rc = resolve_layout(cfg->k, cache->batch, n, cache->kv_heads, d, 2, true, &lk)) != FA_OK ||
        (rc = resolve_layout(cfg->v, cache->batch, n, cache->kv_heads, d, 2, true, &lv)) != FA_OK)
        return rc;
    if (!rows) return FA_ERR_INVALID_ARG;
    if (!k_out && !v_out) return FA_OK;
    const size_t heads = 2 * cache->batch * cache->kv_heads, per = 256 / (d / 8) * kCache4ReadRows, parts = (n + per - 1) / per;
    if (heads > kOpsMaxGrid / parts) return FA_ERR_UNSUPPORTED;
    Cache4Params p{};
    fill_cache4(*cache, block_rows, capacity, &p);
    p.ko = k_out, p.vo = v_out, p.ks = lk.st, p.vs = lv.st, p.rows = rows;
    p.n = static_cast<int>(n);
    p.nparts = static_cast<int>(parts);
    p.vec = vec_ok(k_out, lk, d) && vec_ok(v_out, lv, d);
    int dev;
    const OpsModule module = cache4_module(cache->dtype, 0);
    if ((rc = ops_begin(&dev, module)) != FA_OK) return rc;
    return ops_launch(dev, module, cache->dtype == FA_DTYPE_BF16 ? "fa_cache4_read_bf16" : "fa_cache4_read_f16",
                      heads * parts, 256, &p, static_cast<hipStream_t>(stream));
} catch (...) {   // no memory for the tables of modules, kernels and workspaces
    return FA_ERR_ALLOC;
}

int fa_cache4_attention(void* stream_, const fa_tree_config* c, const fa_window* window, const fa_kv_cache4* cache,
                        const void* q, void* out, float* lse) try {
    size_t block_rows = 0, capacity = 0;
    int rc = check_cache4(cache, &block_rows, &capacity);
    if (rc != FA_OK) return rc;
    if (!c) return FA_ERR_INVALID_ARG;
    if (cache->batch == 0 || c->heads == 0 || c->n_tokens == 0 || cache->d_head == 0) return FA_OK;
    if (cache->kv_heads == 0 || c->heads % cache->kv_heads != 0) return FA_ERR_INVALID_ARG;
    if (c->heads > kOpsMaxSeq || c->n_tokens > kTreeMaxTokens) return FA_ERR_UNSUPPORTED;
    const size_t d = cache->d_head, n = c->n_tokens;
    ScoreScale sc;
    OpsLayout lq, lo;
    if ((rc = resolve_scale(c->softmax_scale, c->softcap, d, &sc)) != FA_OK ||
        (rc = resolve_layout(c->q, cache->batch, n, c->heads, d, 2, false, &lq)) != FA_OK ||
        (rc = resolve_layout(c->out, cache->batch, n, c->heads, d, 2, true, &lo)) != FA_OK)
        return rc;
    int size, sinks;
    if ((rc = resolve_window(window, false, kWindowMaxPos, 0, &size, &sinks)) != FA_OK) return rc;
    if (!q || !out) return FA_ERR_INVALID_ARG;
    if (cache->batch * c->heads > kOpsMaxGrid) return FA_ERR_UNSUPPORTED;
    RowsParams p{};
    p.q = q, p.k = cache->k, p.v = cache->v, p.k_scale = cache->k_scale, p.v_scale = cache->v_scale;
    p.out = out, p.lse = lse;
    p.slopes = c->slopes, p.lens = cache->lens, p.table = cache->block_table;
    p.pos = c->positions, p.mask = c->mask;
    p.qs = lq.st, p.os = lo.st;
    p.batch = static_cast<int>(cache->batch), p.heads = static_cast<int>(c->heads);
    p.kv_heads = static_cast<int>(cache->kv_heads), p.group = static_cast<int>(c->heads / cache->kv_heads);
    p.n = static_cast<int>(n), p.sk = static_cast<int>(capacity), p.d = static_cast<int>(d);
    p.page_shift = page_shift4(*cache);
    p.n_pages = static_cast<int>(cache->n_pages), p.pages_per_seq = static_cast<int>(cache->pages_per_seq);
    p.mask_words = static_cast<int>((n + 63) / 64), p.mask_shared = c->mask_shared ? 1 : 0;
    p.window = size, p.sinks = sinks;
    p.scale_log2e = sc.scale_log2e, p.cap_in = sc.cap_in, p.cap_log2e = sc.cap_log2e;
    p.block4 = static_cast<int>(block_rows);
    p.vec4 = vec_ok(q, lq, d) && ovec_ok(out, lo, 2);
    int dev;
    const OpsModule module = cache4_module(cache->dtype, size), joins = cache_module(cache->dtype, p);
    if ((rc = ops_begin(&dev, module)) != FA_OK || (rc = ops_module(dev, joins)) != FA_OK) return rc;
    const hipStream_t stream = static_cast<hipStream_t>(stream_);
    const size_t rows = n * static_cast<size_t>(p.group);
    const char* kind = cache->block_table && cache->page_size < 32                           ? "p"
                       : c->softcap > 0.0f || c->slopes || (d != 64 && d != 128 && d != 256) ? "m"
                                                                                              : "";
    const RowsPlan plan = plan_rows4(d, !*kind, cache->batch, cache->kv_heads, rows,
                                     window_keys(capacity, size, sinks, n, false), g_dev[dev].num_cus);
    char name[64];
    std::snprintf(name, sizeof(name), "fa_rows4_%s_c%d_t%d%s", dtype_name(cache->dtype), static_cast<int>(d / 32), plan.mt, kind);
    return launch_rows(dev, stream, cache->dtype, module, name, plan, ops_pad_d(d), p.vec4, &p);
} catch (...) {   // no memory for the tables of modules, kernels and workspaces
    return FA_ERR_ALLOC;
}

}  // extern "C"
