"""Norms of queries and keys: what the host refuses or settles without a GPU."""
from __future__ import annotations

import ctypes
import math
import os
import subprocess

import pytest

import flash_attention_amd as fa
from test_ops_host import INVALID, NO_DEVICE, PAGES, PTR, ROOT, UNSUPPORTED, cache, needs_no_gpu, status

FAR = PTR + (1 << 16)


def config(dtype=fa.DTYPE_F32, d=64, rot=64):
    return fa.rotary_config(dtype, d, rot)


def forward(batch=2, seq=3, pos=PTR, q=PTR, qo=FAR, layout=None, k_layout=None, k=0, ko=0, eps=1e-6, w=PTR, cfg=None):
    return status(fa.norm_rotary_device, cfg or config(), fa.head_norm(w, w, eps), batch, seq, pos,
                  layout or fa.rotary_tensor(2), q, qo, k_layout, k, ko)


def backward(batch=2, seq=3, pos=PTR, x=PTR, dy=FAR, dx=2 * FAR, dw=PTR, grad=None, kg=None, eps=1e-6, cfg=None):
    return status(fa.norm_rotary_backward_device, cfg or config(), fa.head_norm(0, 0, eps), batch, seq, pos,
                  grad or fa.norm_grad(2), x, dy, dx, dw, kg)


def append(n=5, k=PTR, v=PTR, pos=PTR, q=0, qo=0, c=None, eps=1e-6, rot=True, **kw):
    if rot is True:
        rot = config(fa.DTYPE_BF16)
    return status(fa.cache_append_device, c or cache(), fa.append_config(n, rotary=rot or None, **kw), k, v, pos, q, qo,
                  norm=fa.head_norm(0, 0, eps))


def test_refusals():
    assert forward(pos=0) == INVALID and forward(q=0) == INVALID and forward(qo=0) == INVALID
    assert forward(k_layout=fa.rotary_tensor(2)) == INVALID
    assert forward(layout=fa.rotary_tensor(2, None, (0, 64, 192))) == INVALID
    assert forward(qo=PTR, layout=fa.rotary_tensor(2, None, (384, 128, 64))) == INVALID
    assert backward(pos=0) == INVALID and backward(x=0) == INVALID and backward(dy=0) == INVALID
    assert backward(grad=fa.norm_grad(2, None, None, (0, 64, 192))) == INVALID
    assert backward(dx=PTR, grad=fa.norm_grad(2, (384, 128, 64))) == INVALID   # in place with two layouts
    assert backward(dx=FAR, grad=fa.norm_grad(2, None, (384, 128, 64))) == INVALID
    assert backward(kg=fa.norm_grad(2), dx=0) in (INVALID, NO_DEVICE)
    big = 1 << 30
    assert forward(batch=big, seq=big) == UNSUPPORTED and backward(batch=big, seq=big) == UNSUPPORTED
    assert forward(batch=2, seq=big, layout=fa.rotary_tensor(big)) == UNSUPPORTED
    lib = fa.lib()
    n = fa.head_norm()
    assert lib.fa_norm_rotary(None, None, n, 1, 1, PTR, fa.rotary_tensor(1), PTR, PTR, None, None, None) == INVALID
    assert lib.fa_norm_rotary(None, config(), None, 1, 1, PTR, fa.rotary_tensor(1), PTR, PTR, None, None, None) == INVALID
    assert lib.fa_norm_rotary(None, config(), n, 1, 1, PTR, None, PTR, PTR, None, None, None) == INVALID
    assert lib.fa_norm_rotary_backward(None, config(), n, 1, 1, PTR, None, *([PTR] * 4), None, *([PTR] * 4)) == INVALID


@pytest.mark.parametrize("eps", (0.0, -1.0, math.nan, math.inf))
def test_eps(eps):
    assert forward(eps=eps) == INVALID and backward(eps=eps) == INVALID and append(eps=eps) == INVALID


def test_append_refusals():
    assert append(rot=False) == INVALID   # norms come before a rotation
    assert append(k=0) == INVALID and append(v=0) == INVALID and append(pos=0) == INVALID
    assert append(rot=config(fa.DTYPE_F16)) == INVALID and append(rot=config(fa.DTYPE_BF16, 128)) == INVALID
    assert append(q_layout=fa.rotary_tensor(4)) == INVALID
    assert append(c=cache(**dict(PAGES, page_size=24))) == INVALID and append(c=cache(lens=0)) == INVALID
    assert append(n=0, k=0, v=0) == fa.FA_OK and append(c=cache(batch=0, lens=0)) == fa.FA_OK


def test_nothing_to_do():
    assert forward(batch=0, q=0, qo=0) == fa.FA_OK and forward(seq=0, q=0, qo=0) == fa.FA_OK
    assert forward(layout=fa.rotary_tensor(0), q=0, qo=0) == fa.FA_OK
    assert backward(dx=0, dw=0) == fa.FA_OK


@needs_no_gpu
def test_accepted_calls_reach_the_device():
    assert forward() == NO_DEVICE and forward(w=0) == NO_DEVICE and forward(qo=PTR) == NO_DEVICE
    assert backward() == NO_DEVICE and backward(dx=0) == NO_DEVICE and backward(dw=0) == NO_DEVICE
    assert backward(dx=PTR) == NO_DEVICE and backward(dx=FAR) == NO_DEVICE
    assert backward(seq=0, pos=0, x=0, dy=0) == NO_DEVICE   # the weights' gradients are zeros
    assert append() == NO_DEVICE and append(q=PTR, qo=FAR, q_layout=fa.rotary_tensor(4)) == NO_DEVICE


def test_structs_match_the_header(tmp_path):
    lines, want = ['#include <stdio.h>', '#include "fa_hip.h"', "int main(void) {"], []
    for name, cls in (("fa_head_norm", fa.HeadNorm), ("fa_norm_grad", fa.NormGrad)):
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
