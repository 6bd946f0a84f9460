"""Calls of several threads on one stream: the kernels of a call are queued together.

The host library's own source runs against a stand-in for the HIP runtime
(tests/callers/stub_hip.h) that records the launches, so this needs no GPU.
A call of several kernels hands partial sums from one to the next in the
stream's workspace, which the next call on the stream uses too.
"""
from __future__ import annotations

import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "flash-attention-cpu_amd", "csrc")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
MODULES = ["fa_kernels", "fa_rotary"] + [f"{a}_{b}" for a in ("fa_score", "fa_cache") for b in ("f32", "bf16", "f16")]


def compile_with_stub(tmp_path, source):
    """A program of the host library, the stand-in and `source`; returns (program, environment)."""
    src, exe = tmp_path / "main.cpp", tmp_path / "main"
    src.write_text('#include "stub_hip.h"\n#include "fa_host.cpp"\n' + source)
    subprocess.run([os.path.join(ROCM, "llvm", "bin", "clang++"), "-std=c++17", "-O1", "-w", "-D__HIP_PLATFORM_AMD__",
                    "-I", os.path.join(ROCM, "include"), "-I", CSRC, "-I", os.path.join(ROOT, "tests", "callers"),
                    str(src), "-lpthread", "-ldl", "-o", str(exe)], check=True)
    for m in MODULES:
        (tmp_path / f"{m}.hsaco").write_bytes(b"")
    return str(exe), dict(os.environ, FA_HIP_MODULE=str(tmp_path / "fa_kernels.hsaco"))


DRIVER = r"""
static char mem[64] __attribute__((aligned(64)));

// One call of each kind that queues several kernels.
static int one(int kind, hipStream_t stream) {
    void* p = mem;
    if (kind == 0) {   // documents, heads of a group shared out: ranges, order, dQ, dK / dV, sum
        fa_score_config c{};
        c.dtype = FA_DTYPE_BF16, c.causal = 1, c.batch = 4, c.heads = 64, c.kv_heads = 8;
        c.seq_len_q = c.seq_len_k = 600, c.d_head = 64;
        c.q_doc = c.k_doc = static_cast<const int32_t*>(p);
        return fa_score_backward(stream, &c, p, p, p, p, static_cast<float*>(p), p, p, p, p);
    }
    if (kind == 1) {   // keys split over runs, then the merge
        fa_kv_cache k{};
        k.dtype = FA_DTYPE_BF16, k.batch = 2, k.kv_heads = 2, k.d_head = 64, k.k = p, k.v = p;
        k.lens = static_cast<const int32_t*>(p), k.capacity = 5000;
        fa_tree_config c{};
        c.heads = 8, c.n_tokens = 4;
        return fa_tree_attention(stream, &c, &k, p, p, nullptr);
    }
    const float* f = static_cast<const float*>(p);
    if (kind == 2) return fa_device_ex(2, stream, f, f, f, 1, 4, 1, 20000, 128, nullptr, nullptr, static_cast<float*>(p));
    return fa_device_ex_noalloc(2, stream, f, f, f, 1, 4, 1, 20000, 128, nullptr, nullptr, static_cast<float*>(p));
}

// argv: kinds of the threads' calls.  Prints the launches' names, a call a line; fails where one call's lie apart.
int main(int argc, char** argv) {
    stub::yields = 4;
    if (fa_init() != FA_OK) return 2;
    const hipStream_t stream = reinterpret_cast<hipStream_t>(&mem);
    std::vector<std::thread> threads;
    int failed = 0;
    for (int t = 1; t < argc; ++t)
        threads.emplace_back([&, t] {
            for (int i = 0; i < 200; ++i) {
                stub::call = t * 1000 + i;
                if (one(std::atoi(argv[t]), stream) != FA_OK) failed = 1;
                if (i % 50 == 49 && fa_release_stream_workspace(stream) != FA_OK) failed = 1;
            }
        });
    for (auto& t : threads) t.join();
    if (failed) return 3;
    std::unordered_map<int, int> ended;
    int apart = 0, last = -1;
    for (const auto& l : stub::launches) {
        if (l.call != last) {
            if (last >= 0) ended[last] = 1;
            if (ended.count(l.call)) ++apart;
            last = l.call;
        }
    }
    std::printf("%zu launches of %d calls, apart %d\n", stub::launches.size(), 200 * (argc - 1), apart);
    return apart ? 1 : 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    return compile_with_stub(tmp_path_factory.mktemp("threads"), DRIVER)


@pytest.mark.parametrize("kinds,per", (((0, 0), (5, 5)), ((1, 1, 1), (2, 2, 2)), ((0, 1, 2), (5, 2, 2)), ((2, 2), (2, 2)),
                                       ((3, 3), (2, 2))))
def test_kernels_of_a_call_are_queued_together(program, kinds, per):
    exe, env = program
    r = subprocess.run([exe, *map(str, kinds)], capture_output=True, text=True, env=env, timeout=120)
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr)
    assert r.stdout.startswith(f"{200 * sum(per)} launches of {200 * len(kinds)} calls, apart 0"), r.stdout


SIZES = r"""
int main() {
    static char mem[64] __attribute__((aligned(64)));
    float* const f = reinterpret_cast<float*>(mem);
    char text[256];
    int i = 0;
    for (size_t sk : {3000, 20000, 100000, 1000000}) {   // each on a stream of its own, twice
        if (fa_describe_launch(2, 1, 16, 1, sk, 128, 0, nullptr, text, sizeof(text)) != FA_OK) return 2;
        ++i;
        for (int n = 0; n < 2; ++n)
            if (fa_device_ex(2, reinterpret_cast<hipStream_t>(mem + i), f, f, f, 1, 16, 1, sk, 128, nullptr, nullptr, f) !=
                FA_OK)
                return 2;
        std::printf("%zu %s\n", stub::allocations.back(), std::strstr(text, "workspace=") + 10);
    }
    std::printf("%zu allocations\n", stub::allocations.size());
    return 0;
}
"""


def test_workspaces_are_whole_units_and_one_more_than_needed(tmp_path):
    """Units of 2 MiB, in which free memory is reported."""
    exe, env = compile_with_stub(tmp_path, SIZES)
    out = subprocess.run([exe], capture_output=True, text=True, env=env, check=True, timeout=60).stdout.splitlines()
    unit = 2 << 20
    for line in out[:-1]:
        size, need = (int(x) for x in line.split()[:2])
        assert size % unit == 0 and need + unit <= size < need + 2 * unit, line
    assert out[-1] == "4 allocations"


RELEASE = r"""
int main() {
    static char mem[64] __attribute__((aligned(64)));
    float* const f = reinterpret_cast<float*>(mem);
    const hipStream_t s = reinterpret_cast<hipStream_t>(mem);
    if (fa_init() != FA_OK || fa_release_stream_workspace(s) != FA_OK) return 2;
    std::printf("%d\n", stub::synchronized);
    if (fa_device_ex(2, s, f, f, f, 1, 16, 1, 20000, 128, nullptr, nullptr, f) != FA_OK) return 2;
    for (int i = 0; i < 2; ++i)
        if (fa_release_stream_workspace(s) != FA_OK) return 2;
    std::printf("%d\n", stub::synchronized);
    return 0;
}
"""


def test_a_stream_without_a_workspace_is_left_alone(tmp_path):
    """Releasing the workspace of a stream that has none does not wait for the stream (which may be capturing)."""
    exe, env = compile_with_stub(tmp_path, RELEASE)
    out = subprocess.run([exe], capture_output=True, text=True, env=env, check=True, timeout=60).stdout.split()
    assert out == ["0", "1"]
