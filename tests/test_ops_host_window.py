"""Windows: what the host refuses or settles without a GPU."""
from __future__ import annotations

import ctypes
import os
import subprocess

import pytest

import flash_attention_amd as fa
from test_host_threads import compile_with_stub
from test_ops_host import INVALID, NO_DEVICE, PTR, ROOT, UNSUPPORTED, backward, cache, needs_no_gpu, score, status


def calls(window, **kw):
    """Status of each entry point with that window; kw: of the score config."""
    c = fa.score_config(fa.DTYPE_BF16, 2, 4, 2, kw.pop("sq", 5), kw.pop("sk", 7), 64, **kw)
    return (status(fa.score_attention_device, c, PTR, PTR, PTR, PTR, window=window),
            status(fa.score_attention_backward_device, c, *([PTR] * 9), window=window))


def tree(window, **kw):
    return status(fa.tree_attention_device, fa.tree_config(4, 5, **kw), cache(), PTR, PTR, window=window)


@pytest.mark.parametrize("size,sinks", ((0, 0), (-1, 0), (4, -1), (-(1 << 62), 5)))
def test_refused_windows(size, sinks):
    assert set(calls(fa.window(size, sinks))) == {INVALID}
    assert tree(fa.window(size, sinks)) == INVALID


def test_sinks_among_documents_are_refused():
    assert set(calls(fa.window(3, 1), q_doc_ptr=PTR, k_doc_ptr=PTR)) == {UNSUPPORTED}


def test_far_positions_are_refused():
    assert set(calls(fa.window(3, 1), q_start=(1 << 30) + 8)) == {UNSUPPORTED}
    assert set(calls(fa.window(3), sk=1 << 30, sq=1 << 30, q_start=1 << 29)) == {UNSUPPORTED}


@needs_no_gpu
def test_how_far_positions_may_be():
    """The largest distance, here of 5 queries from q_start to key 0, is 2^30 - 4096, as the header says."""
    last = (1 << 30) - 4096
    assert set(calls(fa.window(3, 1), q_start=last - 4)) == {NO_DEVICE}
    assert set(calls(fa.window(3, 1), q_start=last - 3)) == {UNSUPPORTED}
    assert set(calls(fa.window(last + 1), q_start=last - 3)) == {UNSUPPORTED}   # the query at last + 1
    assert set(calls(fa.window(last + 2), q_start=last - 3)) == {NO_DEVICE}     # hides nothing


@needs_no_gpu
@pytest.mark.parametrize("size,sinks", ((1, 0), (1, 1 << 62), (1 << 62, 1 << 62), (5, 100)))
def test_accepted_windows_reach_the_device(size, sinks):
    assert set(calls(fa.window(size, sinks))) == {NO_DEVICE}
    assert tree(fa.window(size, sinks)) == NO_DEVICE
    assert set(calls(fa.window(3), q_doc_ptr=PTR, k_doc_ptr=PTR)) == {NO_DEVICE}


def test_what_the_plain_calls_refuse_is_refused():
    w = fa.window(4)
    assert score(dtype=3) == INVALID and backward(kv_heads=3) == INVALID
    assert set(calls(w, softcap=-1.0)) == {INVALID}
    assert set(calls(w, q_start=1 << 31)) == {UNSUPPORTED}
    assert tree(w, softcap=-2.0) == INVALID
    lib = fa.lib()
    assert lib.fa_window_forward(None, None, w, PTR, PTR, PTR, PTR, None) == INVALID
    assert lib.fa_window_backward(None, None, w, *([PTR] * 9)) == INVALID
    assert lib.fa_window_tree_attention(None, None, w, cache(), PTR, PTR, None) == INVALID


def test_no_window_is_the_plain_call():
    lib = fa.lib()
    c = fa.score_config(fa.DTYPE_BF16, 2, 4, 2, 0, 7, 64)
    assert lib.fa_window_forward(None, c, None, None, None, None, None, None) == fa.FA_OK


def test_struct_matches_the_header(tmp_path):
    src, exe = tmp_path / "size.c", tmp_path / "size"
    src.write_text('#include <stdio.h>\n#include "fa_hip.h"\nint main(void) {'
                   'printf("%zu %zu %zu", sizeof(fa_window), offsetof(fa_window, size), offsetof(fa_window, sinks)); }')
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(fa.Window), fa.Window.size.offset, fa.Window.sinks.offset]

KERNELS = r"""
// stdin, a call a line: dtype heads kv_heads sq sk q_start d causal size (0: no window) sinks; stdout: the first kernel
int main() {
    static char mem[64] __attribute__((aligned(64)));
    void* p = mem;
    fa_score_config c{};
    c.batch = 1;
    fa_window w;
    while (std::scanf("%d %zu %zu %zu %zu %ld %zu %d %ld %ld", &c.dtype, &c.heads, &c.kv_heads, &c.seq_len_q, &c.seq_len_k,
                      &c.q_start, &c.d_head, &c.causal, &w.size, &w.sinks) == 10) {
        stub::launches.clear();
        if (fa_window_forward(nullptr, &c, w.size ? &w : nullptr, p, p, p, p, nullptr) != FA_OK) return 1;
        std::printf("%s\n", stub::launches[0].name.c_str());
    }
    return 0;
}
"""
F32, BF16 = fa.DTYPE_F32, fa.DTYPE_BF16


def test_walks_that_a_window_leaves_short_do_not_split_the_keys(tmp_path):
    """The kernel that splits the keys takes every row through all of a call's keys; a window leaves each a few."""
    exe, env = compile_with_stub(tmp_path, KERNELS)
    for m in ("fa_score", "fa_cache"):
        for t in ("f32", "bf16", "f16"):
            (tmp_path / f"{m}_w_{t}.hsaco").write_bytes(b"")
    calls = {
        "score": [(dt, h, h, n, n, 0, d, causal, size, 4) for dt in (F32, BF16) for causal in (0, 1)
                  for h, n, d, size in ((1, 4096, 64, 100), (1, 4096, 128, 100), (2, 2048, 128, 200), (1, 2500, 64, 100),
                                        (1, 4000, 256, 100))]
                 + [(BF16, 1, 1, 1100, 1100, 0, 256, 1, 300, 4), (F32, 1, 1, 4096, 4096, 0, 128, 1, 2000, 0),
                    (BF16, 8, 8, 512, 8192, 7680, 128, 1, 1700, 4)],
        "rows": [(dt, *x) for dt in (F32, BF16) for x in
                 ((8, 8, 512, 8192, 7680, 128, 1, 3000, 4), (1, 1, 128, 8192, 8064, 128, 1, 1900, 4),
                  (1, 1, 64, 8192, 8128, 128, 1, 100, 4), (1, 1, 1100, 1100, 0, 256, 1, 900, 0),
                  (1, 1, 4096, 4096, 0, 128, 1, 0, 0), (1, 1, 4096, 4096, 0, 128, 0, 3900, 0), (1, 1, 1900, 1900, 0, 256, 1, 0, 0),
                  (2, 2, 2048, 2048, 0, 64, 1, 0, 0))]
                + [(F32, 1, 1, 1100, 1100, 0, 256, 1, 300, 4), (F32, 8, 8, 512, 8192, 7680, 128, 1, 1700, 4)],
    }
    text = "".join(" ".join(str(int(x)) for x in c) + "\n" for cs in calls.values() for c in cs)
    got = subprocess.run([exe], input=text, capture_output=True, text=True, env=env, check=True, timeout=60).stdout.split()
    want = [(name, c) for name, cs in calls.items() for c in cs]
    assert len(got) == len(want)
    wrong = [(c, g) for (name, c), g in zip(want, got) if not g.startswith(f"fa_{name}_")]
    assert not wrong, wrong
