"""Sliding windows with sinks on the GPU: score attention, forward and backward, and attention over a cache."""
from __future__ import annotations

import math

import pytest
import torch

import flash_attention_amd as fa
from ops_reference import attend, check
from test_gpu_rotary_tree import Tree
from test_gpu_score import Call, doc_ids

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


class Window(Call):
    def __init__(self, dtype, b, h, hk, sq, sk, d, size, sinks, q_start=0, **kw):
        super().__init__(dtype, b, h, hk, sq, sk, d, q_start=q_start, **kw)
        i, j = torch.arange(sq)[:, None] + q_start, torch.arange(sk)[None, :]
        near = ((i - j).abs() < size) | (j < sinks)
        self.see = [x & near for x in self.see]
        self.window = fa.window(size, sinks)

    def forward(self, lse=True):
        fa.score_attention_device(self.cfg, *(self.gpu[n].data_ptr() for n in ("q", "k", "v")),
                                  self.outs["out"].data_ptr(), self.lse.data_ptr() if lse else 0, stream(),
                                  window=self.window)

    def backward(self, dq=True, dk=True, dv=True):
        o = self.outs
        fa.score_attention_backward_device(
            self.cfg, *(self.gpu[n].data_ptr() for n in ("q", "k", "v")), o["out"].data_ptr(), self.lse.data_ptr(),
            self.gpu["dout"].data_ptr(), *(o[n].data_ptr() if w else 0 for n, w in (("dq", dq), ("dk", dk), ("dv", dv))),
            stream(), window=self.window)


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("size,sinks", ((1, 0), (1, 3), (17, 0), (64, 64), (100, 5), (299, 1), (300, 0), (5000, 7)))
@pytest.mark.parametrize("causal", (True, False))
def test_window(dtype, size, sinks, causal):
    Window(dtype, 1, 4, 2, 300, 300, 64, size, sinks, causal=causal, seed=size + sinks).run_and_check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("d", (8, 40, 128, 200, 256))
def test_head_widths(dtype, d):
    Window(dtype, 1, 2, 1, 400, 400, d, 70, 9, causal=True, seed=d).run_and_check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("mods", ({"cap": 5.0}, {"alibi": True}, {"cap": 9.0, "alibi": True}, {"prefix": [120, 7]},
                                  {"layout": "bshd", "pad": 8}, {"layout": "bshd", "pad": 3}))
def test_with_other_changes_of_scores(dtype, mods):
    Window(dtype, 2, 4, 2, 260, 260, 64, 50, 4, causal=True, seed=2, **mods).run_and_check()


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
def test_documents(dtype):
    ids = doc_ids(2, 330, [[100, 17, 200], [300]], pad=6)
    Window(dtype, 2, 4, 4, 330, 330, 64, 40, 0, causal=True, q_doc=ids, k_doc=ids, seed=3).run_and_check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("sq", (1, 2, 13, 70, 150))
@pytest.mark.parametrize("causal", (True, False))
def test_chunks_of_queries(dtype, sq, causal):
    """A few queries at the end of, within or past the keys, on the kernels that split the keys and on the others."""
    for start, size, sinks in ((900 - sq, 200, 6), (400, 33, 0), (1000, 150, 4), (1200, 100, 0), (-50, 60, 2)):
        Window(dtype, 2, 4, 2, sq, 900, 64, size, sinks, q_start=start, causal=causal, seed=sq).run_and_check()


@pytest.mark.parametrize("dtype", ("bf16", "f32"))
def test_rows_that_see_nothing(dtype):
    c = Window(dtype, 1, 2, 2, 200, 100, 64, 20, 0, causal=True, seed=4)   # queries far past the last key
    assert not c.see[0][130].any()
    c.run_and_check()
    assert (c.outs["out"][0, :, 130:] == 0).all() and (c.lse[0, :, 130:] == -math.inf).all()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("heads,d,n,size,sinks", ((2, 64, 3000, 90, 70), (16, 64, 2100, 200, 3), (8, 128, 1500, 64, 130)))
def test_long(dtype, heads, d, n, size, sinks):
    """More stages than are looked at together, sinks beyond one block of keys."""
    Window(dtype, 1, heads, heads // 2, n, n, d, size, sinks, causal=True, seed=n).run_and_check()


@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("sinks", (0, 70))
@pytest.mark.parametrize("dtype,n,d,size", (("f32", 2100, 64, 700), ("bf16", 2100, 64, 1500), ("f16", 2100, 128, 1500),
                                            ("f32", 1100, 256, 330), ("bf16", 1100, 256, 550)))
def test_split_keys_of_many_rows(dtype, n, d, size, sinks, causal):
    """Few heads, keys cut into runs that all blocks of rows walk: whole runs are hidden from some."""
    Window(dtype, 1, 1, 1, n, n, d, size, sinks, causal=causal, seed=n + sinks).run_and_check(grads=False)


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("mods", ({"alibi": True, "cap": 9.0}, {"prefix": [1900]}, {"layout": "bshd", "pad": 3}))
def test_split_keys_of_many_rows_and_other_changes(dtype, mods):
    Window(dtype, 1, 2, 1, 900, 2600, 64, 2000, 5, q_start=1500, causal=True, seed=14, **mods).run_and_check(grads=False)


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("sinks", (60, 200, 512, 100000))
@pytest.mark.parametrize("causal", (True, False))
def test_many_sinks(dtype, sinks, causal):
    """From a few blocks of keys to all of them; as many queries as keys, and fewer."""
    Window(dtype, 1, 4, 2, 512, 512, 64, 40, sinks, causal=causal, seed=sinks).run_and_check()
    Window(dtype, 1, 16, 2, 70, 512, 64, 40, sinks, q_start=400, causal=causal, seed=sinks).run_and_check()


def by_row(see, q, k, v, scale, bias, dout=None):
    """attend of each row with the keys that it sees alone: bounds of sums over those."""
    rows = [attend(q[i:i + 1], k[see[i]], v[see[i]], torch.ones(1, int(see[i].sum()), dtype=torch.bool), scale,
                   bias=bias[i:i + 1, see[i]], dout=None if dout is None else dout[i:i + 1]) for i in range(q.shape[0])]
    return {n: tuple(torch.cat([r[n][i] for r in rows]) for i in (0, 1))
            for n in (("out", "lse") if dout is None else ("out", "lse", "dq"))}


@pytest.mark.parametrize("sq", (4, 600))
@pytest.mark.parametrize("sinks", (4, 70))
def test_sinks_far_below_the_other_scores(sq, sinks):
    """A bias by distance leaves sinks thousands below: what weighs is as exact as without them."""
    c = Window("f32", 1, 8, 8, sq, 6000, 64, 100, sinks, q_start=6000 - sq, causal=True, alibi=True, seed=sq)
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    rows = torch.arange(0, sq, 37 if sq > 4 else 1)
    for h in range(8):
        e = by_row(c.see[0][rows], c.q[0, h, rows], c.k[0, h], c.v[0, h], c.scale, c.bias[h][rows], c.dout[0, h, rows])
        for n, (x, bound) in e.items():
            check(n, (c.lse if n == "lse" else c.outs[n])[0, h, rows.cuda()], x, bound)
    # The weights of sinks reach down to 0.  One below f32's smallest normal number, 2^-126, may count as 0, and so may its
    # product with what it weighs: sq terms of a sum, each off by 2^-126 (1 + its factor).  Of dV that is |dO|, of dK
    # |dP - delta| |q| scale, where |dP| and |delta| are at most |dO| times the longest row of V.
    full, tiny = c.expect(), 2.0 ** -126
    long_v = c.v.norm(dim=-1).max().double()
    for n, factor in (("dv", c.dout.double().abs().amax()),
                      ("dk", 2 * c.dout.double().norm(dim=-1).max() * long_v * c.q.double().abs().amax())):
        check(n, c.outs[n], full[n][0], full[n][1] + sq * tiny * (1 + factor))


@pytest.mark.parametrize("value", (math.nan, math.inf))
@pytest.mark.parametrize("sq,start", ((400, 0), (3, 397)))
def test_what_lies_outside_does_not_reach_a_row(value, sq, start):
    """Infinite and NaN keys and values at 100: seen by queries 100 .. 149 alone."""
    c = Window("bf16", 1, 2, 1, sq, 400, 64, 50, 4, q_start=start, causal=True, seed=5)
    c.gpu["k"][0, 0, 100] = value
    c.gpu["v"][0, 0, 100] = value
    c.gpu["v"][0, 0, 90, 3] = value
    c.forward()
    torch.cuda.synchronize()
    c.k[0, 0, 100], c.v[0, 0, 100], c.v[0, 0, 90, 3] = 0, 0, 0
    out, lse = c.expect(False)["out"], c.expect(False)["lse"]
    rows = torch.arange(sq) + start
    clean = (rows < 90) | (rows >= 150)
    check("out", c.outs["out"][:, :, clean], out[0][:, :, clean], out[1][:, :, clean])
    check("lse", c.lse[:, :, clean], lse[0][:, :, clean], lse[1][:, :, clean])
    if start == 0:
        assert not torch.isfinite(c.outs["out"][0, :, 90:140, 3]).any()
        c.backward()
        torch.cuda.synchronize()
        dq = c.expect()["dq"]
        check("dq", c.outs["dq"][:, :, clean], dq[0][:, :, clean], dq[1][:, :, clean])


def test_a_window_that_hides_nothing_is_none():
    c = Window("bf16", 1, 4, 2, 300, 300, 64, 300, 2, causal=True, seed=6)
    c.forward()
    c.backward()
    d = Call("bf16", 1, 4, 2, 300, 300, 64, causal=True, seed=6)
    d.forward()
    d.backward()
    torch.cuda.synchronize()
    assert all(torch.equal(c.outs[n], d.outs[n]) for n in c.outs) and torch.equal(c.lse, d.lse)


@pytest.mark.parametrize("wanted", ((True, False, False), (False, True, False), (False, False, True)))
def test_single_gradients(wanted):
    c = Window("bf16", 1, 4, 2, 500, 500, 64, 80, 70, causal=True, seed=7)
    c.forward()
    c.backward(*wanted)
    torch.cuda.synchronize()
    e = c.expect()
    for n, w in zip(("dq", "dk", "dv"), wanted):
        if w:
            check(n, c.outs[n], *e[n])
        else:
            assert (c.outs[n] == 7).all()


def test_gradients_against_differences():
    """The directional derivative of sum(o dout) by central differences of the kernel's own forward pass, f32."""
    c = Window("f32", 1, 2, 1, 90, 90, 64, 20, 3, causal=True, seed=8)
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    g = torch.Generator().manual_seed(9)
    eps = 2.0 ** -7
    for n in ("q", "k", "v"):
        way = torch.randn(c.gpu[n].shape, generator=g).cuda()
        base, values = c.gpu[n].clone(), []
        for s in (eps, -eps):
            c.gpu[n].copy_(base + s * way)
            c.forward()
            torch.cuda.synchronize()
            values.append((c.outs["out"].double() * c.gpu["dout"].double()).sum().item())
        c.gpu[n].copy_(base)
        want = (c.outs["d" + n].double() * way.double()).sum().item()
        got = (values[0] - values[1]) / (2 * eps)
        # third derivatives: eps^2 / 6 of sums of some 11520 terms of order 1 (2^-14 / 6 * 11520 = 0.12); rounding:
        # 2^-24 * 11520 * 4 / (2 eps) = 0.18
        assert abs(got - want) < 0.6


def test_the_same_bits_every_time():
    c = Window("f16", 2, 8, 2, 700, 700, 64, 100, 20, causal=True, seed=10)
    seen = []
    for _ in range(3):
        c.forward()
        c.backward()
        torch.cuda.synchronize()
        seen.append([c.outs[n].clone() for n in sorted(c.outs)] + [c.lse.clone()])
    assert all(torch.equal(a, b) for other in seen[1:] for a, b in zip(seen[0], other))


# ---------------------------------------------------------------------------
# Over a cache
# ---------------------------------------------------------------------------
class WindowTree(Tree):
    def __init__(self, dtype, lens, h, hk, n, d, size, sinks, **kw):
        super().__init__(dtype, lens, h, hk, n, d, **kw)
        self.size, self.sinks = size, sinks
        self.window = fa.window(size, sinks)

    def seen(self, i):
        """[n, lens + n] what the tokens of sequence i see."""
        x = self.lens[i]
        see = torch.cat((torch.ones(self.n, x, dtype=torch.bool), self.see[i]), dim=1)
        pos = self.pos[i].long().clamp_min(x)
        at = torch.cat((torch.arange(x), pos))
        return see & ((pos[:, None] - at[None, :] < self.size) | (torch.arange(x + self.n) < self.sinks)[None, :])

    def run(self):
        fa.tree_attention_device(self.cfg, self.cache, self.gq.data_ptr(), self.out.data_ptr(), self.lse.data_ptr(),
                                 stream(), window=self.window)

    def check(self):
        torch.cuda.synchronize()
        for i, x in enumerate(self.lens):
            if x < 0:
                assert (self.out[i] == 0).all() and (self.lse[i] == -math.inf).all()
                continue
            see = self.seen(i)
            kpos = torch.cat((torch.arange(x), self.pos[i].long()))
            dist = (self.pos[i].long()[:, None] - kpos[None, :]).abs().double()
            for j in range(self.h):
                r = attend(self.q[i, j], self.k[i][j * self.hk // self.h], self.v[i][j * self.hk // self.h], see,
                           self.scale, self.cap, None if self.slopes is None else -self.slopes[j].double() * dist, self.t)
                check(f"out {i} {j}", self.out[i, j], *r["out"])
                check(f"lse {i} {j}", self.lse[i, j], *r["lse"])


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("n", (1, 5, 33, 130))
@pytest.mark.parametrize("page", (0, 4, 16))
@pytest.mark.parametrize("size,sinks", ((1, 0), (40, 3), (128, 0), (200, 100), (5000, 4)))
def test_cache(dtype, n, page, size, sinks):
    c = WindowTree(dtype, [500, 0, 63, 1, 901, -1, 200], 4, 2, n, 64, size, sinks, page=page, mask="chain", seed=n)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("mask", ("tree", "any", "none"))
@pytest.mark.parametrize("mods", ({}, {"positions": True}, {"alibi": True, "positions": True, "cap": 9.0}))
@pytest.mark.parametrize("size", (3, 30, 130))
def test_cache_masks_and_scores(dtype, mask, mods, size):
    c = WindowTree(dtype, [300, 40, -1, 0], 4, 2, 24, 64, size, 4, mask=mask, seed=3, **mods)
    c.run()
    c.check()


@pytest.mark.parametrize("d", (36, 128, 256))
@pytest.mark.parametrize("n,h", ((1, 8), (7, 4), (40, 8)))
def test_long_cache(d, n, h):
    """Keys split over many workgroups, with and without rows left out before the window."""
    c = WindowTree("bf16", [9000, 10, 2500, 1100], h, 1, n, d, 1000, 70, page=64, seed=4)
    c.run()
    c.check()


def test_positions_before_the_filled_rows_count_as_their_end():
    c = WindowTree("f32", [400, 70], 4, 2, 6, 64, 50, 2, positions=True, seed=5)
    c.pos[:, 2] = 3
    c.keep[1].copy_(c.pos)
    c.run()
    c.check()


def test_pages_out_of_reach_may_be_gone():
    """The table's entries before the window (without the sinks' page) are bad, their rows NaN."""
    c = WindowTree("bf16", [2000, 700], 8, 2, 2, 128, 100, 5, page=16, seed=6)
    table = c.table.clone()
    table[0, 1:(2000 - 99) // 16], table[1, 1:(700 - 99) // 16] = -1, 10 ** 6
    c.keep[3].copy_(table)
    c.run()
    c.check()


@pytest.mark.parametrize("n,h,d", ((1, 8, 64), (40, 8, 64), (3, 8, 36)))
@pytest.mark.parametrize("sinks", (4, 70))
def test_sinks_far_below_in_a_cache(n, h, d, sinks):
    c = WindowTree("f32", [6000, 300, 90], h, 8, n, d, 100, sinks, alibi=True, seed=12)
    c.run()
    torch.cuda.synchronize()
    for i, x in enumerate(c.lens):
        pos = c.pos[i].double()
        dist = (pos[:, None] - torch.cat((torch.arange(x), pos))[None, :]).abs()
        for j in range(h):
            for name, (value, bound) in by_row(c.seen(i), c.q[i, j], c.k[i][j], c.v[i][j], c.scale,
                                               -c.slopes[j].double() * dist).items():
                check(f"{name} {i} {j}", (c.lse if name == "lse" else c.out)[i, j], value, bound)


@pytest.mark.parametrize("size", (1, 5, 30, 64, 65, 97))
@pytest.mark.parametrize("length", (449, 480, 512, 513))
def test_ends_of_the_window(size, length):
    """Last keys and first ones anywhere in a block of 64, with sinks walked after them."""
    for dtype, d, n in (("f32", 64, 20), ("bf16", 256, 20), ("bf16", 64, 3)):
        c = WindowTree(dtype, [length], 2, 1, n, d, size, 3, seed=13)
        c.run()
        c.check()


def test_lengths_beyond_the_capacity():
    """Tokens stand so far behind that their window reaches no row but the sinks."""
    c = WindowTree("bf16", [300], 2, 1, 4, 64, 100, 3, spare=0, seed=11)
    for length in (10 ** 9, 2 ** 31 - 1):
        c.keep[0].fill_(length)
        c.run()
        torch.cuda.synchronize()
        see = torch.zeros(4, 304, dtype=torch.bool)
        see[:, :3] = True
        for j in range(2):
            r = attend(c.q[0, j], c.k[0][0], c.v[0][0], see, c.scale, dtype=c.t)
            check("out", c.out[0, j], *r["out"])
            check("lse", c.lse[0, j], *r["lse"])


@pytest.mark.parametrize("page", (0, 16))
def test_rows_out_of_reach_do_not_count(page):
    """Infinite and NaN rows next to the window and to the sinks."""
    c = WindowTree("bf16", [700], 4, 2, 3, 64, 100, 5, page=page, seed=7)
    for row in (5, 6, 63, 600, 599):
        p, r = c.place(0, torch.tensor([row]))
        c.gk[int(p), int(r)], c.gv[int(p), int(r)] = math.nan, math.inf
        c.k[0][:, row], c.v[0][:, row] = 0, 0
    assert not c.seen(0)[:, [5, 6, 63, 600, 599]].any()
    c.run()
    c.check()


def test_captured_and_replayed():
    c = WindowTree("bf16", [9000, 4000], 8, 2, 1, 128, 2000, 4, seed=8)
    w = Window("bf16", 1, 4, 2, 600, 600, 64, 100, 70, causal=True, seed=8)

    def passes():
        c.run()
        w.forward()
        w.backward()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        passes()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            passes()
        for _ in range(3):
            c.out.fill_(7.0)
            for x in w.outs.values():
                x.fill_(7.0)
            graph.replay()
            side.synchronize()
            c.check()
            for n, (x, e) in w.expect().items():
                check(n, w.lse if n == "lse" else w.outs[n], x, e)
            passes()
            side.synchronize()
