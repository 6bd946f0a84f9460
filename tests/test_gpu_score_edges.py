"""Score attention on the GPU where its definition allows more than training usually asks for: any sign of
the slopes, gradients of any size, caps of any size, many small calls in one.

Bounds: tests/ops_reference.py.
"""
from __future__ import annotations

import threading

import pytest
import torch

from test_gpu_rotary_tree import Tree
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


def test_threads_that_share_a_stream():
    """Calls of several kernels from three threads on one stream: each gets what it gets alone."""
    ids = [doc_ids(4, 600, x) for x in (([200, 400], [500, 90]), ([64, 300], [7, 580]))]
    train = [Call("bf16", 4, 64, 8, 600, 600, 64, causal=True, q_doc=x, k_doc=x, seed=s) for s, x in zip((3, 4), ids)]
    tree = Tree("bf16", [3000, 1700], 8, 2, 4, 64, seed=5)

    def step(c):
        if c is tree:
            c.run()
        else:
            c.forward()
            c.backward()

    def results(c):
        return [c.out, c.lse] if c is tree else [*c.outs.values(), c.lse]

    cases = train + [tree]
    for c in cases:
        step(c)
    torch.cuda.synchronize()
    alone = [[x.clone() for x in results(c)] for c in cases]
    for c in cases:
        for x in results(c):
            x.fill_(7.0)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=lambda c=c: [step(c) for _ in range(20)]) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for c, want in zip(cases, alone):
        for x, y in zip(results(c), want):
            assert torch.equal(x, y)
