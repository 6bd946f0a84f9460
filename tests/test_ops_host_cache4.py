"""The cache in 4 bits: what the host refuses or settles without a GPU."""
from __future__ import annotations

import ctypes
import os
import subprocess

import pytest

import flash_attention_amd as fa
from test_ops_host import INVALID, NO_DEVICE, PTR, ROOT, UNSUPPORTED, needs_no_gpu, status

PAGES = {"block_table_ptr": PTR, "page_size": 16, "n_pages": 8, "pages_per_seq": 3}


def cache(batch=2, kv_heads=2, d=64, k=PTR, ks=PTR, v=PTR, vs=PTR, lens=PTR, dtype=fa.DTYPE_BF16, **kw):
    return fa.kv_cache4(dtype, batch, kv_heads, d, k, ks, v, vs, lens, **(kw or {"capacity": 32}))


def attention(heads=4, n=5, q=PTR, out=PTR, c=None, window=None, **kw):
    return status(fa.cache4_attention_device, fa.tree_config(heads, n, **kw), c or cache(), q, out, window=window)


def append(n=5, k=PTR, v=PTR, c=None, **kw):
    return status(fa.cache4_append_device, c or cache(), fa.append_config(n, **kw), k, v)


def read(n=5, rows=PTR, k=PTR, v=PTR, c=None, **kw):
    return status(fa.cache4_read_device, c or cache(), fa.read_config(n, **kw), rows, k, v)


@pytest.mark.parametrize("want,c", (
    (INVALID, {"dtype": 9}), (UNSUPPORTED, {"dtype": fa.DTYPE_F32}), (UNSUPPORTED, {"d": 288}), (UNSUPPORTED, {"d": 80}),
    (INVALID, {"lens": 0}), (INVALID, {"k": 0}), (INVALID, {"v": 0}), (INVALID, {"ks": 0}), (INVALID, {"vs": 0}),
    (INVALID, {"k": PTR + 4}), (INVALID, {"v": PTR + 8}), (INVALID, {"ks": PTR + 2}), (INVALID, {"vs": PTR + 2}),
    (INVALID, {"capacity": 33}), (UNSUPPORTED, {"capacity": 1 << 31}),
    (INVALID, dict(PAGES, page_size=0)), (INVALID, dict(PAGES, page_size=4)), (INVALID, dict(PAGES, page_size=24)),
    (UNSUPPORTED, dict(PAGES, pages_per_seq=1 << 27)),
))
def test_cache_refusals(want, c):
    assert attention(c=cache(**c)) == want and append(c=cache(**c)) == want and read(c=cache(**c)) == want


def test_refusals():
    assert attention(heads=3) == INVALID and attention(n=257) == UNSUPPORTED
    assert attention(q=0) == INVALID and attention(out=0) == INVALID and attention(softcap=-2.0) == INVALID
    assert attention(out_strides=(0, 64, 320)) == INVALID and attention(window=fa.window(0)) == INVALID
    assert append(k=0) == INVALID and append(v=0) == INVALID
    rot = fa.rotary_config(fa.DTYPE_BF16, 64, 64)
    assert append(rotary=rot) == UNSUPPORTED and append(q_layout=fa.rotary_tensor(4)) == UNSUPPORTED
    assert append(k_strides=(0, 63, 0)) == INVALID and append(n=(1 << 30) + 1) == UNSUPPORTED
    assert read(rows=0) == INVALID and read(k_strides=(0, 64, 320)) == INVALID
    big = 1 << 30
    assert append(c=cache(batch=big), n=8) == UNSUPPORTED and read(c=cache(batch=big), n=8) == UNSUPPORTED
    assert append(c=cache(batch=1 << 20, kv_heads=1 << 20), n=8) == UNSUPPORTED
    assert attention(c=cache(batch=big, kv_heads=2)) == UNSUPPORTED
    assert attention(c=cache(**dict(PAGES, page_size=1 << 20, pages_per_seq=1, n_pages=1 << 11))) == UNSUPPORTED   # 2^32 rows
    lib = fa.lib()
    assert lib.fa_cache4_append(None, cache(), None, PTR, PTR) == INVALID
    assert lib.fa_cache4_append(None, None, fa.append_config(1), PTR, PTR) == INVALID
    assert lib.fa_cache4_read(None, cache(), None, PTR, PTR, PTR) == INVALID
    assert lib.fa_cache4_attention(None, None, None, cache(), PTR, PTR, None) == INVALID
    assert lib.fa_cache4_attention(None, fa.tree_config(4, 4), None, None, PTR, PTR, None) == INVALID


def test_nothing_to_do():
    assert attention(n=0, q=0, out=0) == fa.FA_OK and attention(heads=0, q=0, out=0) == fa.FA_OK
    assert attention(c=cache(batch=0, lens=0)) == fa.FA_OK
    assert append(n=0, k=0, v=0) == fa.FA_OK and append(c=cache(capacity=0, k=0, ks=0, v=0, vs=0)) == fa.FA_OK
    assert read(n=0, rows=0) == fa.FA_OK and read(k=0, v=0) == fa.FA_OK


@needs_no_gpu
def test_accepted_calls_reach_the_device():
    assert attention() == NO_DEVICE and attention(c=cache(**PAGES), window=fa.window(5, 2)) == NO_DEVICE
    assert append() == NO_DEVICE and append(c=cache(**PAGES)) == NO_DEVICE
    assert read() == NO_DEVICE and read(k=0) == NO_DEVICE and read(v=0) == NO_DEVICE
    assert attention(c=cache(capacity=0, k=0, ks=0, v=0, vs=0)) == NO_DEVICE


def test_shapes_of_the_buffers():
    s = fa.cache4_shapes(3, 2, 16, 96)
    assert s == {"k": (3, 2, 16, 12), "k_scale": (3, 2, 16, 3, 2), "v": (3, 2, 2, 96), "v_scale": (3, 2, 2, 3, 2, 8)}


def test_structs_match_the_header(tmp_path):
    lines, want = ['#include <stdio.h>', '#include "fa_hip.h"', "int main(void) {"], []
    for name, cls in (("fa_kv_cache4", fa.KvCache4), ("fa_read_config", fa.ReadConfig)):
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for field, *_ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
    lines += ["return 0; }"]
    src, exe = tmp_path / "offsets.c", tmp_path / "offsets"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == want
