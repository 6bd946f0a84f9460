"""Score attention on the GPU where its definition allows more than training usually asks for: any sign of
the slopes, gradients of any size, caps of any size, many small calls in one.

Bounds: tests/ops_reference.py.
"""
from __future__ import annotations

import pytest
import torch

from test_gpu_score import Call, check_batch, doc_ids

pytestmark = pytest.mark.gpu


def with_slopes(c, slopes, q_start=0):
    """The call with other slopes than the usual powers of two."""
    c.slopes = torch.tensor(slopes)
    c.keep[3].copy_(c.slopes)
    sq, sk = c.q.shape[2], c.k.shape[2]
    dist = (torch.arange(sq)[:, None] + q_start - torch.arange(sk)[None, :]).abs().double()
    c.bias = [-s.double() * dist for s in c.slopes]
    return c


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("sq,sk,causal", ((150, 150, True), (150, 190, False), (1, 70, False), (64, 33, True)))
@pytest.mark.parametrize("d,cap", ((64, 0.0), (128, 20.0), (256, 0.0), (36, 0.0)))
def test_negative_slopes(dtype, sq, sk, causal, d, cap):
    """Far keys weigh more; the rows that fill up the last tile of queries weigh nothing all the same."""
    c = Call(dtype, 2, 4, 2, sq, sk, d, causal=causal, alibi=True, cap=cap, q_start=3, seed=1)
    with_slopes(c, [-0.3, 0.0, -2.0, 0.25], 3).run_and_check()


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
def test_negative_slopes_with_documents_and_many_blocks(dtype):
    ids = doc_ids(8, 500, ([100, 300], [450, 20]), pad=9)
    c = Call(dtype, 8, 16, 4, 500, 500, 64, causal=True, alibi=True, q_doc=ids, k_doc=ids, seed=2)
    with_slopes(c, [-0.1 * (i % 5) for i in range(16)])
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    check_batch(c, 6)
