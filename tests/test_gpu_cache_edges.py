"""Attention over a cache on the GPU: bad pages under every kernel, shared masks, layouts of Q and O.

Bounds: tests/ops_reference.py.
"""
from __future__ import annotations

import pytest
import torch

import flash_attention_amd as fa
from ops_reference import attend, check
from test_gpu_rotary_tree import Tree
from test_gpu_score import filled, make, strides, to_gpu

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


def share_mask(c, **kw):
    """All sequences with the first one's mask, given once."""
    c.see[:] = c.see[0]
    c.cfg = fa.tree_config(c.h, c.n, mask_ptr=c.bits.data_ptr(), mask_shared=True, softcap=c.cap, softmax_scale=c.scale,
                           slopes_ptr=0 if c.slopes is None else c.keep[2].data_ptr(), **kw)
    return c


@pytest.mark.parametrize("dtype,d", (("f32", 64), ("bf16", 64), ("f16", 128), ("bf16", 36)))
@pytest.mark.parametrize("n", (1, 5, 65, 130))
@pytest.mark.parametrize("page", (0, 16))
def test_one_mask_for_all_sequences(dtype, d, n, page):
    """Lengths that put the drafted rows everywhere within a stage of 64 keys, masks of one word and of several."""
    c = share_mask(Tree(dtype, [500, 0, 63, 1, 31, 190, 640], 4, 2, n, d, page=page, mask="any", seed=n))
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("n,d", ((6, 64), (70, 64), (70, 36)))
def test_one_mask_and_an_infinite_drafted_value(dtype, n, d):
    """Only the tokens that see the row get its infinities, in every sequence."""
    c = share_mask(Tree(dtype, [50, 200, 127], 2, 1, n, d, mask="any", seed=7))
    at = n // 2
    hit = c.see[0, :, at].clone()
    for i, x in enumerate(c.lens):
        p, r = c.place(i, torch.tensor([x + at]))
        c.gv[int(p), int(r)] = float("inf")
    c.run()
    torch.cuda.synchronize()
    rows = hit.nonzero().flatten().tolist()
    assert rows and len(rows) < n
    assert torch.isinf(c.out[:, :, rows]).all()
    for i, x in enumerate(c.lens):   # the row as zeros: those that do not see it notice nothing
        c.v[i][:, x + at] = 0.0
        see = torch.cat((torch.ones(n, x, dtype=torch.bool), c.see[0]), dim=1)
        rest = [j for j in range(n) if j not in rows]
        for j in range(c.h):
            value, bound = attend(c.q[i, j], c.k[i][0], c.v[i][0], see, c.scale, dtype=c.t)["out"]
            check("rest", c.out[i, j, rest], value[rest], bound[rest])


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("n,d,pad", ((1, 128, 0), (7, 64, 0), (7, 64, 8), (40, 128, 0), (40, 64, 3), (5, 36, 0)))
def test_tokens_before_heads(dtype, n, d, pad):
    """Q and O as [batch, tokens, heads, d], with columns between the rows; O's surroundings stay as they were."""
    c = Tree(dtype, [700, 129, -1], 8, 2, n, d, page=32, seed=n)
    q = make(torch.Generator().manual_seed(1), c.t, 3, 8, n, d, layout="bshd", pad=pad)
    q.copy_(c.q)
    c.gq, c.out = to_gpu(q), filled(q)
    c.cfg = fa.tree_config(8, n, mask_ptr=c.bits.data_ptr(), q_strides=strides(c.gq), out_strides=strides(c.out))
    c.run()
    c.check()
    if pad:
        whole = torch.empty(0, dtype=c.t, device="cuda").set_(c.out.untyped_storage()).view(-1, d + pad)
        assert (whole[:, d:] == 7.0).all()


def test_a_token_of_a_tensor_whose_tokens_lie_far_apart():
    """The strides of single entries are not looked at: the last token of [tokens, batch, heads, d]."""
    c = Tree("bf16", [300, 40], 4, 2, 1, 64, seed=3)
    far = 1 << 23
    st = (c.gq.stride(0), far, c.gq.stride(1))
    c.cfg = fa.tree_config(4, 1, q_strides=st, out_strides=st)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("n,d,page", ((1, 128, 0), (7, 64, 16), (64, 128, 16), (9, 36, 8)))
def test_same_bits_every_time(dtype, n, d, page):
    c = Tree(dtype, [3000, 70, 1500], 8, 2, n, d, page=page, seed=4)
    c.run()
    torch.cuda.synchronize()
    out, lse = c.out.clone(), c.lse.clone()
    for _ in range(3):
        c.out.fill_(7.0)
        c.lse.fill_(7.0)
        c.run()
        torch.cuda.synchronize()
        assert torch.equal(c.out, out) and torch.equal(c.lse, lse)
