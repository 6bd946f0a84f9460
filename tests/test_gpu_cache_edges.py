"""Attention over a cache on the GPU: bad pages under every kernel, shared masks, layouts of Q and O.

Bounds: tests/ops_reference.py.
"""
from __future__ import annotations

import pytest
import torch

from test_gpu_rotary_tree import Tree

pytestmark = pytest.mark.gpu


def spoil(c, where):
    """Page numbers outside of the pool at (sequence, page) places; returns which rows they hide."""
    table = c.table.clone()
    hidden = [torch.zeros(c.capacity, dtype=torch.bool) for _ in c.lens]
    for n, (b, page) in enumerate(where):
        table[b, page] = (-1, c.cache.n_pages, 10 ** 6, -2 ** 31)[n % 4]
        hidden[b][page * c.page:(page + 1) * c.page] = True
    c.keep[3].copy_(table)
    return hidden


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("page,d", ((1, 64), (2, 36), (8, 64), (8, 36), (16, 36), (8, 200), (16, 64), (32, 128),
                                    (64, 256)))
@pytest.mark.parametrize("n", (4, 48))
def test_bad_pages_of_any_alignment(dtype, page, d, n):
    """Bad pages in some stages of the keys and under some waves' rows of them; drafted rows among them."""
    c = Tree(dtype, [700, 150, 333], 4, 2, n, d, page=page, seed=page)
    last = [(x + n - 1) // page for x in c.lens]
    hidden = spoil(c, [(0, 0), (0, 70 // page), (0, 300 // page), (0, 511 // page), (0, last[0]), (1, 100 // page),
                       (2, 64 // page), (2, 200 // page)])
    for _ in range(2):
        c.out.fill_(7.0)
        c.run()
        c.check(hidden)
