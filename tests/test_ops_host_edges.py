"""What the host refuses, or lets pass, at the ends of the arguments' ranges.  No GPU needed."""
from __future__ import annotations

import math

import pytest

import flash_attention_amd as fa
from test_ops_host import NO_DEVICE, UNSUPPORTED, backward, needs_no_gpu, score, tree


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
