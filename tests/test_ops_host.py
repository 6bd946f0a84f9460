"""Score attention, rotary, cache: what the host refuses or settles without a GPU.

Every refusal comes before any device access, so each is seen here, on a
machine without one; a call that passes all checks ends in FA_ERR_NO_DEVICE.
"""
from __future__ import annotations

import ctypes
import math
import os
import subprocess

import pytest

import flash_attention_amd as fa

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PTR = 1 << 20   # an address that is never read
needs_no_gpu = pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="the accepted calls would run")


def status(f, *args, **kw):
    try:
        f(*args, **kw)
    except fa.FaError as e:
        return e.status
    return fa.FA_OK


def score(q=PTR, k=PTR, v=PTR, out=PTR, batch=2, heads=4, kv_heads=2, sq=5, sk=7, d=64, dtype=fa.DTYPE_BF16, **kw):
    c = fa.score_config(dtype, batch, heads, kv_heads, sq, sk, d, **kw)
    return status(fa.score_attention_device, c, q, k, v, out)


def backward(p=(PTR,) * 9, batch=2, heads=4, kv_heads=2, sq=5, sk=7, d=64, **kw):
    c = fa.score_config(fa.DTYPE_F16, batch, heads, kv_heads, sq, sk, d, **kw)
    return status(fa.score_attention_backward_device, c, *p)


INVALID, UNSUPPORTED, NO_DEVICE = fa.FA_ERR_INVALID_ARG, fa.FA_ERR_UNSUPPORTED, fa.FA_ERR_NO_DEVICE


@needs_no_gpu
def test_accepted_calls_reach_the_device():
    assert score() == NO_DEVICE
    assert backward() == NO_DEVICE
    assert score(k=0, v=0, sk=0) == NO_DEVICE
    assert backward(p=(PTR,) * 6 + (0, 0, 0)) == NO_DEVICE
    assert tree() == NO_DEVICE
    assert append() == NO_DEVICE
    assert rotary() == NO_DEVICE


@pytest.mark.parametrize("want,kw", (
    (INVALID, {"dtype": 3}), (INVALID, {"dtype": -1}),
    (INVALID, {"kv_heads": 0}), (INVALID, {"kv_heads": 3}), (INVALID, {"kv_heads": 8}),
    (INVALID, {"q": 0}), (INVALID, {"k": 0}), (INVALID, {"v": 0}), (INVALID, {"out": 0}),
    (INVALID, {"softcap": -1.0}), (INVALID, {"softcap": math.nan}), (INVALID, {"softcap": math.inf}),
    (INVALID, {"q_doc_ptr": PTR}), (INVALID, {"k_doc_ptr": PTR}),
    (UNSUPPORTED, {"d": 257}), (UNSUPPORTED, {"sk": (1 << 30) + 1}), (UNSUPPORTED, {"q_start": -(1 << 31)}),
    (INVALID, {"strides": {"q": (0, 63, 0)}}), (INVALID, {"strides": {"k": (0, 0, 64)}}),
    (INVALID, {"strides": {"v": (-1, 64, 64)}}), (UNSUPPORTED, {"strides": {"v": (0, 1 << 22, 64)}}),
    # outputs may not overlap: batches, heads or tokens on top of each other
    (INVALID, {"strides": {"out": (0, 64, 320)}}), (INVALID, {"strides": {"out": (1280, 64, 64)}}),
    (INVALID, {"strides": {"out": (1280, 65, 64)}}),
))
def test_score_refusals(want, kw):
    assert score(**kw) == want


@needs_no_gpu
@pytest.mark.parametrize("strides", ({"q": (0, 64, 320)}, {"k": (64, 256, 0)}, {"out": (1280, 256, 64)},
                                     {"out": (2000, 264, 66)}, {"out": (100, 10000, 2000)}))
def test_layouts_that_are_allowed(strides):
    """Inputs may share memory between batches or heads; outputs in any order of dimensions."""
    assert score(strides=strides) == NO_DEVICE


@pytest.mark.parametrize("i", range(6))
def test_backward_needs_its_inputs(i):
    p = [PTR] * 9
    p[i] = 0
    assert backward(p=p) == INVALID


@pytest.mark.parametrize("name", ("dq", "dk", "dv"))
def test_gradients_may_not_overlap(name):
    assert backward(strides={name: (0, 64, 448)}) == INVALID


def test_zero_sizes_queue_nothing():
    assert score(batch=0, q=0, out=0) == fa.FA_OK
    assert score(heads=0, kv_heads=0, q=0, out=0) == fa.FA_OK
    assert score(sq=0, q=0, out=0) == fa.FA_OK
    assert score(d=0, q=0, out=0) == fa.FA_OK
    assert backward(sq=0, sk=0, p=(0,) * 9) == fa.FA_OK


def test_unknown_strides_and_missing_configs():
    with pytest.raises(ValueError):
        fa.score_config(0, 1, 1, 1, 1, 1, 8, strides={"o": (1, 1, 1)})
    lib = fa.lib()
    assert lib.fa_score_forward(None, None, PTR, PTR, PTR, PTR, None) == INVALID
    assert lib.fa_score_backward(None, None, *([PTR] * 9)) == INVALID
    assert lib.fa_rotary(None, None, 1, 1, PTR, 0, fa.rotary_tensor(1), PTR, PTR, None, None, None) == INVALID
    assert lib.fa_tree_attention(None, None, cache(), PTR, PTR, None) == INVALID
    assert lib.fa_tree_attention(None, fa.tree_config(4, 4), None, PTR, PTR, None) == INVALID
    assert lib.fa_cache_append(None, cache(), None, PTR, PTR, None, None, None) == INVALID
    assert lib.fa_cache_append(None, None, fa.append_config(1), PTR, PTR, None, None, None) == INVALID


# ---- rotary ---------------------------------------------------------------
def rotary(d=64, rot=64, batch=2, seq=3, pos=PTR, q=PTR, qo=PTR + 4096, layout=None, dtype=fa.DTYPE_F32, k_layout=None,
           k=0, ko=0):
    c = fa.rotary_config(dtype, d, rot)
    return status(fa.rotary_device, c, batch, seq, pos, layout or fa.rotary_tensor(2), q, qo, k_layout, k, ko)


@pytest.mark.parametrize("want,args,kw", (
    (INVALID, (3, 64), {}), (UNSUPPORTED, (0, 258), {}), (INVALID, (0, 64, 0), {}), (INVALID, (0, 64, 3), {}),
    (INVALID, (0, 64, 66), {}), (INVALID, (0, 64), {"base": 1.0}), (INVALID, (0, 64), {"base": math.nan}),
    (INVALID, (0, 64), {"scaling": 4}), (INVALID, (0, 64), {"scaling": fa.ROTARY_LINEAR, "factor": 0.5}),
    (INVALID, (0, 64, 2), {"scaling": fa.ROTARY_NTK, "factor": 2.0}),
    (INVALID, (0, 64), {"scaling": fa.ROTARY_YARN, "factor": 2.0}),
    (INVALID, (0, 64), {"scaling": fa.ROTARY_YARN, "factor": math.inf, "original_len": 10.0}),
))
def test_rotary_config_refusals(want, args, kw):
    assert status(fa.rotary_config, *args, **kw) == want


def test_rotary_refusals():
    assert rotary(pos=0) == INVALID and rotary(q=0) == INVALID and rotary(qo=0) == INVALID
    assert rotary(k_layout=fa.rotary_tensor(2)) == INVALID   # a second tensor without memory
    assert rotary(layout=fa.rotary_tensor(2, None, (0, 64, 192))) == INVALID   # outputs on top of each other
    # in place with two layouts: a row would be read after it was written
    assert rotary(qo=PTR, layout=fa.rotary_tensor(2, None, (384, 128, 64))) == INVALID
    assert rotary(batch=0, q=0, qo=0) == fa.FA_OK and rotary(seq=0, q=0, qo=0) == fa.FA_OK


def test_rotary_turns():
    c = fa.rotary_config(fa.DTYPE_F32, 64, 32, base=10000.0)
    assert [c.turns[i] for i in range(16)] == pytest.approx(
        [10000.0 ** (-2.0 * i / 32) / (2 * math.pi) for i in range(16)], rel=1e-14)
    c = fa.rotary_config(fa.DTYPE_F32, 64, 32, scaling=fa.ROTARY_LINEAR, factor=4.0)
    assert c.turns[3] == pytest.approx(10000.0 ** (-6.0 / 32) / (8 * math.pi), rel=1e-14) and c.gain == 1.0
    c = fa.rotary_config(fa.DTYPE_F32, 64, 32, scaling=fa.ROTARY_NTK, factor=4.0)
    # the slowest pair is interpolated by the whole factor, the fastest not at all
    assert c.turns[0] == pytest.approx(1 / (2 * math.pi), rel=1e-14)
    assert c.turns[15] == pytest.approx(10000.0 ** (-30.0 / 32) / (8 * math.pi), rel=1e-13)
    c = fa.rotary_config(fa.DTYPE_F32, 128, 128, scaling=fa.ROTARY_YARN, factor=8.0, original_len=4096)
    assert c.gain == pytest.approx(0.1 * math.log(8) + 1, rel=1e-7)
    assert c.turns[0] == pytest.approx(1 / (2 * math.pi)) and c.turns[63] == pytest.approx(
        10000.0 ** (-126.0 / 128) / (16 * math.pi))


# ---- cache ------------------------------------------------------------------
def cache(batch=2, kv_heads=2, d=64, k=PTR, v=PTR, lens=PTR, dtype=fa.DTYPE_BF16, **kw):
    kw = kw or {"capacity": 32}
    return fa.kv_cache(dtype, batch, kv_heads, d, k, v, lens, **kw)


PAGES = {"block_table_ptr": PTR, "page_size": 16, "n_pages": 8, "pages_per_seq": 3}


def tree(heads=4, n=5, q=PTR, out=PTR, c=None, **kw):
    return status(fa.tree_attention_device, fa.tree_config(heads, n, **kw), c or cache(), q, out)


def append(n=5, k=PTR, v=PTR, pos=0, q=0, qo=0, c=None, **kw):
    return status(fa.cache_append_device, c or cache(), fa.append_config(n, **kw), k, v, pos, q, qo)


@pytest.mark.parametrize("want,c", (
    (INVALID, {"dtype": 9}), (UNSUPPORTED, {"d": 300}), (INVALID, {"lens": 0}), (INVALID, {"k": 0}),
    (INVALID, {"v": 0}), (INVALID, dict(PAGES, page_size=0)), (INVALID, dict(PAGES, page_size=24)),
    (UNSUPPORTED, {"capacity": (1 << 30) + 1}), (UNSUPPORTED, dict(PAGES, pages_per_seq=1 << 27)),
    (INVALID, {"capacity": 32, "k_strides": (0, 64, 2048)}), (INVALID, dict(PAGES, v_strides=(64, 64, 1024))),
))
def test_cache_refusals(want, c):
    assert tree(c=cache(**c)) == want
    assert append(c=cache(**c)) == want


def test_tree_refusals():
    assert tree(heads=3) == INVALID and tree(n=257) == UNSUPPORTED
    assert tree(q=0) == INVALID and tree(out=0) == INVALID
    assert tree(softcap=-2.0) == INVALID
    assert tree(out_strides=(0, 64, 320)) == INVALID
    assert tree(n=0, q=0, out=0) == fa.FA_OK and tree(heads=0, q=0, out=0) == fa.FA_OK
    assert tree(c=cache(batch=0, lens=0)) == fa.FA_OK


def test_append_refusals():
    rot = fa.rotary_config(fa.DTYPE_BF16, 64, 64)
    assert append(k=0) == INVALID and append(v=0) == INVALID
    assert append(rotary=rot) == INVALID   # no positions
    assert append(rotary=fa.rotary_config(fa.DTYPE_F16, 64, 64), pos=PTR) == INVALID
    assert append(rotary=fa.rotary_config(fa.DTYPE_BF16, 128, 64), pos=PTR) == INVALID
    assert append(q_layout=fa.rotary_tensor(4), q=PTR, qo=PTR) == INVALID   # queries without rotary
    assert append(rotary=rot, pos=PTR, q_layout=fa.rotary_tensor(4)) == INVALID   # queries without memory
    assert append(n=0, k=0, v=0) == fa.FA_OK


def test_structs_match_the_header(tmp_path):
    """Sizes and member offsets of the ctypes structures against the C compiler's."""
    pairs = {"fa_strides": fa.Strides, "fa_score_config": fa.ScoreConfig, "fa_rotary_config": fa.RotaryConfig,
             "fa_rotary_tensor": fa.RotaryTensor, "fa_kv_cache": fa.KvCache, "fa_append_config": fa.AppendConfig,
             "fa_tree_config": fa.TreeConfig}
    rename = {("fa_rotary_tensor", "src"): "in", ("fa_rotary_tensor", "dst"): "out"}
    lines = ['#include <stdio.h>', '#include "fa_hip.h"', "int main(void) {"]
    want = []
    for name, cls in pairs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for field, *_ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {rename.get((name, field), field)}));')
            want.append(getattr(cls, field).offset)
    lines += ["return 0; }"]
    src, exe = tmp_path / "offsets.c", tmp_path / "offsets"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == want


def test_sizes_whose_products_pass_64_bits():
    big = 1 << 30
    assert rotary(batch=big, seq=big) == UNSUPPORTED
    assert rotary(layout=fa.rotary_tensor(big), batch=2, seq=big) == UNSUPPORTED
    assert score(batch=big, heads=big, kv_heads=1, sq=big) == UNSUPPORTED
    assert tree(c=cache(batch=big, kv_heads=2, capacity=big)) == UNSUPPORTED
    # heads 2^44 apart, 2^30 of them, inside a batch stride that they pass
    assert score(heads=big, kv_heads=1, out=PTR, strides={"out": (1 << 44, 64, 1 << 44)}) in (INVALID, UNSUPPORTED)
