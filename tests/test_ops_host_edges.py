"""What the host refuses, or lets pass, at the ends of the arguments' ranges.  No GPU needed."""
from __future__ import annotations

import pytest

import flash_attention_amd as fa
from test_ops_host import NO_DEVICE, UNSUPPORTED, append, backward, cache, needs_no_gpu, rotary, score, tree


@pytest.mark.parametrize("cap,scale", ((1e-39, None), (3e38, None), (1e-38, 100.0), (1e30, 1e-15)))
def test_caps_beyond_the_range_of_f32_are_refused(cap, scale):
    """cap * log2(e), or 2 log2(e) scale / cap, is no normal number."""
    for call in (score, backward, tree):
        assert call(softcap=cap, softmax_scale=scale) == UNSUPPORTED


@needs_no_gpu
@pytest.mark.parametrize("cap", (1e-37, 1e-3, 512.0, 513.0, 1e6, 1e30, 1e37))
def test_caps_of_any_size_are_accepted(cap):
    for call in (score, backward, tree):
        assert call(softcap=cap) == NO_DEVICE
    assert score(softcap=cap, dtype=fa.DTYPE_F32) == NO_DEVICE


FAR = 1 << 23   # more than rows may lie apart


@needs_no_gpu
def test_strides_of_single_entries_are_not_looked_at():
    """One token cut out of a tensor whose tokens lie far apart, one batch, one head."""
    for name in ("q", "out"):
        assert score(sq=1, strides={name: (256, FAR, 64)}) == NO_DEVICE
        assert backward(sq=1, strides={"d" + name: (256, FAR, 64)}) == NO_DEVICE
    for name in ("k", "v"):
        assert score(sk=1, strides={name: (256, FAR, 64)}) == NO_DEVICE
    assert score(batch=1, strides={"q": (1 << 60, 64, 320), "out": (1 << 60, 64, 320)}) == NO_DEVICE
    assert score(heads=1, kv_heads=1, strides={"q": (320, 64, 1 << 60), "k": (448, 64, 1 << 60)}) == NO_DEVICE
    assert tree(n=1, q_strides=(256, FAR, 64), out_strides=(256, FAR, 64)) == NO_DEVICE
    assert append(n=1, k_strides=(128, FAR, 64), v_strides=(128, FAR, 64)) == NO_DEVICE
    assert tree(c=cache(capacity=1, k_strides=(128, FAR, 64), v_strides=(128, FAR, 64))) == NO_DEVICE
    assert rotary(seq=1, layout=fa.rotary_tensor(2, (128, FAR, 64), (128, FAR, 64))) == NO_DEVICE


def test_rows_too_far_apart_are_refused():
    assert score(strides={"q": (FAR * 8, FAR, 64)}) == UNSUPPORTED
    assert tree(q_strides=(FAR * 8, FAR, 64)) == UNSUPPORTED
    assert append(k_strides=(FAR * 8, FAR, 64)) == UNSUPPORTED
    assert score(strides={"q": (1 << 45, 64, 320)}) == UNSUPPORTED
