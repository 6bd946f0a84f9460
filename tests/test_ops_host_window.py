"""Windows: what the host refuses or settles without a GPU."""
from __future__ import annotations

import ctypes
import os
import subprocess

import pytest

import flash_attention_amd as fa
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
