"""Rotary positions, cache append and attention of drafted trees on the GPU, against float64."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import flash_attention_amd as fa
from ops_reference import EPS32, attend, check, unit
from test_gpu_score import DT, filled, make, strides, to_gpu

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


def frequencies(rot, base=10000.0, scaling=fa.ROTARY_NONE, factor=1.0, length=0.0):
    """Angle a position of each pair, and the gain."""
    c = torch.arange(rot // 2, dtype=torch.float64)
    if scaling == fa.ROTARY_NTK:
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2.0 * c / rot)
    if scaling == fa.ROTARY_LINEAR:
        return f / factor, 1.0
    if scaling != fa.ROTARY_YARN:
        return f, 1.0
    at = [rot * math.log(length / (2 * math.pi * turns)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
    lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
    ramp = ((c - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1


def rotate(x, pos, f, gain, interleaved, inverse=False):
    """x: [b, h, s, d] float64."""
    rot = 2 * f.shape[0]
    angle = pos.double()[:, None, :, None] * f * (-1 if inverse else 1)
    c, s = torch.cos(angle) * gain, torch.sin(angle) * gain
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, a * s + b * c
    return y


def rotary_bound(x, y, pos, gain, dtype):
    """Two products, a sum and sines within a few 2^-24; the angle's fraction of a turn is
    rounded once to f32 after its reduction in 64 bits: 2 pi (2^-25 + |pos| 2^-53)."""
    angle = 2 * math.pi * (2.0 ** -25 + pos.double().abs().max().item() * 2.0 ** -53)
    pair = x.abs().amax(dim=-1, keepdim=True) * 2 * gain
    e = (8 * EPS32 + angle) * pair
    return e + unit(dtype) * (y.abs() + e) + (2.0 ** -25 if dtype == torch.float16 else 0.0)


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("d,rot", ((64, 64), (128, 64), (80, 40), (256, 256), (50, 18), (2, 2), (7, 6)))
@pytest.mark.parametrize("inverse", (False, True))
def test_rotary(dtype, interleaved, d, rot, inverse):
    t, code = DT[dtype]
    g = torch.Generator().manual_seed(d + rot)
    for layout in ("bhsd", "bshd"):
        q, k = make(g, t, 2, 6, 37, d, 1.0, layout), make(g, t, 2, 3, 37, d, 1.0, layout, pad=8)
        pos = torch.randint(0, 300000, (2, 37), generator=g, dtype=torch.int32)
        cfg = fa.rotary_config(code, d, rot, interleaved=interleaved)
        f, gain = frequencies(rot)
        dq, dk, dp = to_gpu(q), to_gpu(k), pos.cuda()
        qo, ko = torch.full_like(dq, 7.0), filled(k)
        fa.rotary_device(cfg, 2, 37, dp.data_ptr(), fa.rotary_tensor(6, strides(dq), strides(qo)), dq.data_ptr(),
                         qo.data_ptr(), fa.rotary_tensor(3, strides(dk), strides(ko)), dk.data_ptr(), ko.data_ptr(),
                         stream(), inverse=inverse)
        torch.cuda.synchronize()
        for got, x in ((qo, q.double()), (ko, k.double())):
            y = rotate(x, pos, f, gain, interleaved, inverse)
            check("rotary", got, y, rotary_bound(x, y, pos, gain, t))
            assert torch.equal(got.cpu()[..., rot:], x[..., rot:].to(t))


@pytest.mark.parametrize("scaling", (fa.ROTARY_LINEAR, fa.ROTARY_NTK, fa.ROTARY_YARN))
@pytest.mark.parametrize("tokens,heads", ((1, 1), (1, 32), (700, 5)))
def test_rotary_scaling_and_in_place(scaling, tokens, heads):
    g = torch.Generator().manual_seed(scaling)
    x = torch.randn(1, heads, tokens, 128, generator=g)
    pos = torch.randint(0, 1000000, (1, tokens), generator=g, dtype=torch.int32)
    cfg = fa.rotary_config(fa.DTYPE_F32, 128, 128, base=500000.0, scaling=scaling, factor=16.0, original_len=8192)
    f, gain = frequencies(128, 500000.0, scaling, 16.0, 8192)
    y = rotate(x.double(), pos, f, gain, False)
    dx, dp = x.cuda(), pos.cuda()
    fa.rotary_device(cfg, 1, tokens, dp.data_ptr(), fa.rotary_tensor(heads), dx.data_ptr(), dx.data_ptr(),
                     stream=stream())
    torch.cuda.synchronize()
    check("in place", dx, y, rotary_bound(x.double(), y, pos, gain, torch.float32))


def test_rotary_gradient_is_the_inverse():
    """<rotate(x), w> = <x, rotate_inverse(w)> with the scaled gain."""
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(2, 4, 50, 64, generator=g).cuda(), torch.randn(2, 4, 50, 64, generator=g).cuda()
    pos = torch.arange(50, dtype=torch.int32, device="cuda").repeat(2, 1).contiguous()
    cfg = fa.rotary_config(fa.DTYPE_F32, 64, 64, scaling=fa.ROTARY_YARN, factor=4.0, original_len=512)
    t = fa.rotary_tensor(4)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    fa.rotary_device(cfg, 2, 50, pos.data_ptr(), t, x.data_ptr(), y.data_ptr(), stream=stream())
    fa.rotary_device(cfg, 2, 50, pos.data_ptr(), t, w.data_ptr(), dx.data_ptr(), stream=stream(), inverse=True)
    a, b = (y.double() * w.double()).sum().item(), (x.double() * dx.double()).sum().item()
    n = x.numel()
    # every product is within 16 2^-24 of |x||w|, and errors of 25600 terms add up at most linearly
    assert abs(a - b) <= 32 * EPS32 * 2 * (x.double().abs() * w.double().abs()).sum().item()


# ---------------------------------------------------------------------------
# Cache and trees
# ---------------------------------------------------------------------------
class Tree:
    """A cache with rows for lens[b] filled tokens and n drafted ones, contiguous or in shuffled pages."""

    def __init__(self, dtype, lens, h, hk, n, d, page=0, mask="tree", cap=0.0, alibi=False, positions=False, spare=5,
                 layout="bshd", scale=None, seed=0):
        self.t, code = DT[dtype]
        g = torch.Generator().manual_seed(seed)
        b = len(lens)
        self.lens, self.n, self.h, self.hk, self.d, self.cap, self.page = lens, n, h, hk, d, cap, page
        self.scale = scale or 1.0 / math.sqrt(d)
        rows = max(max(lens), 0) + n + spare
        if page:
            per = -(-rows // page)
            self.table = torch.randperm(b * per + 3, generator=g)[:b * per].reshape(b, per).to(torch.int32)
            shape = (b * per + 3, page, hk, d)
            self.capacity = per * page
        else:
            self.table = None
            shape = (b, rows, hk, d)
            self.capacity = rows
        if layout == "bhsd":
            shape = (shape[0], shape[2], shape[1], shape[3])
        # whatever is not a row of a sequence is NaN
        self.kc = torch.full(shape, math.nan, dtype=self.t)
        self.vc = torch.full(shape, math.nan, dtype=self.t)
        if layout == "bhsd":
            self.kc, self.vc = self.kc.transpose(1, 2), self.vc.transpose(1, 2)
        self.q = torch.randn(b, h, n, d, generator=g).to(self.t)
        self.k = [torch.randn(hk, max(x, 0) + n, d, generator=g).to(self.t) for x in lens]
        self.v = [torch.randn(hk, max(x, 0) + n, d, generator=g).to(self.t) for x in lens]
        for i, x in enumerate(lens):
            if x >= 0:
                p, r = self.place(i, torch.arange(x + n))
                self.kc[p, r], self.vc[p, r] = self.k[i].transpose(0, 1), self.v[i].transpose(0, 1)
        # a random tree (or any pairs, or nothing); None: a chain
        words = -(-n // 64)
        self.see = torch.zeros(b, n, n, dtype=torch.bool)
        for i in range(b):
            for j in range(n):
                if mask == "tree":
                    if j:
                        self.see[i, j] = self.see[i, int(torch.randint(max(0, j - 4), j, (1,), generator=g))]
                    self.see[i, j, j] = True
                elif mask == "chain":
                    self.see[i, j, :j + 1] = True
                elif mask == "any":
                    self.see[i, j] = torch.rand(n, generator=g) < 0.5
        bits = np.zeros((b, n, words * 64), dtype=np.uint64)
        bits[:, :, :n] = self.see.numpy()
        packed = (bits.reshape(b, n, words, 64) << np.arange(64, dtype=np.uint64)).sum(axis=-1, dtype=np.uint64)
        self.bits = torch.from_numpy(packed.view(np.int64)).cuda()
        self.pos = torch.tensor([[max(x, 0) + int(self.see[i, j].sum()) - 1 if positions else max(x, 0) + j
                                  for j in range(n)] for i, x in enumerate(lens)], dtype=torch.int32)
        self.slopes = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)]) if alibi else None
        self.keep = [torch.tensor(lens, dtype=torch.int32).cuda(), self.pos.cuda(),
                     None if self.slopes is None else self.slopes.cuda(),
                     None if self.table is None else self.table.cuda()]
        self.gk, self.gv, self.gq = to_gpu(self.kc), to_gpu(self.vc), self.q.cuda()
        self.out = torch.full_like(self.gq, 7.0)
        self.lse = torch.full((b, h, n), 7.0, device="cuda")
        st = (self.gk.stride(0), self.gk.stride(1), self.gk.stride(2))
        self.cache = fa.kv_cache(code, b, hk, d, self.gk.data_ptr(), self.gv.data_ptr(), self.keep[0].data_ptr(),
                                 k_strides=st, v_strides=st, capacity=0 if page else rows,
                                 block_table_ptr=self.keep[3].data_ptr() if page else 0, page_size=page,
                                 n_pages=shape[0] if page else 0, pages_per_seq=self.table.shape[1] if page else 0)
        self.cfg = fa.tree_config(h, n, mask_ptr=0 if mask == "chain" else self.bits.data_ptr(), softcap=cap,
                                  softmax_scale=scale,
                                  slopes_ptr=self.keep[2].data_ptr() if alibi else 0,
                                  positions_ptr=self.keep[1].data_ptr() if positions else 0)

    def place(self, i, rows):
        if self.page:
            return self.table[i].long()[rows // self.page], rows % self.page
        return torch.full_like(rows, i), rows

    def run(self):
        fa.tree_attention_device(self.cfg, self.cache, self.gq.data_ptr(), self.out.data_ptr(), self.lse.data_ptr(),
                                 stream())

    def check(self, hidden=None):
        torch.cuda.synchronize()
        for i, x in enumerate(self.lens):
            if x < 0:
                assert (self.out[i] == 0).all() and (self.lse[i] == -math.inf).all()
                continue
            see = torch.cat((torch.ones(self.n, x, dtype=torch.bool), self.see[i]), dim=1)
            if hidden is not None:
                see = see & ~hidden[i][None, :x + self.n]
            kpos = torch.cat((torch.arange(x), self.pos[i].long()))
            dist = (self.pos[i].long()[:, None] - kpos[None, :]).abs().double()
            for j in range(self.h):
                r = attend(self.q[i, j], self.k[i][j * self.hk // self.h], self.v[i][j * self.hk // self.h], see,
                           self.scale, self.cap, None if self.slopes is None else -self.slopes[j].double() * dist, self.t)
                check(f"out {i} {j}", self.out[i, j], *r["out"])
                check(f"lse {i} {j}", self.lse[i, j], *r["lse"])


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("n", (1, 5, 16, 33, 64, 130))
@pytest.mark.parametrize("page", (0, 16))
def test_tree(dtype, n, page):
    c = Tree(dtype, [500, 0, 63, 1, 200], 4, 2, n, 64, page=page, seed=n)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("d", (8, 36, 80, 128, 192, 256))
def test_tree_head_widths(dtype, d):
    c = Tree(dtype, [700, 129], 8, 2, 7, d, page=32, seed=d)
    c.run()
    c.check()


@pytest.mark.parametrize("page", (1, 2, 8, 64, 256))
def test_tree_pages(page):
    """Pages that end inside a block of keys, or hold several blocks."""
    c = Tree("bf16", [333, 256, 31], 4, 1, 9, 64, page=page, layout="bhsd", seed=page)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("mask", ("chain", "any", "none"))
@pytest.mark.parametrize("mods", ({}, {"cap": 5.0}, {"alibi": True}, {"alibi": True, "positions": True, "cap": 9.0}))
def test_tree_masks_and_scores(dtype, mask, mods):
    c = Tree(dtype, [300, 40, -1, 0], 4, 2, 12, 64, mask=mask, seed=3, **mods)
    c.run()
    c.check()


def test_tree_long_cache():
    """Keys split over many workgroups; one sequence much longer than the others."""
    c = Tree("bf16", [9000, 10, 2500], 8, 1, 3, 128, page=128, alibi=True, seed=4)
    c.run()
    c.check()


def test_tree_capacity_ends_inside_the_draft():
    """Rows at or past the capacity are not seen."""
    c = Tree("bf16", [100], 2, 1, 8, 64, spare=0, seed=5)
    c.cache.capacity = 105
    c.see[:, :, 5:] = False
    c.run()
    c.check()


def test_bad_pages_hold_no_keys():
    c = Tree("bf16", [200, 150], 4, 2, 4, 64, page=16, seed=6)
    bad = c.table.clone()
    bad[0, 3], bad[0, 5], bad[1, 0] = -1, 10 ** 6, c.cache.n_pages
    c.keep[3].copy_(bad)
    hidden = [torch.zeros(300, dtype=torch.bool) for _ in range(2)]
    hidden[0][48:64] = hidden[0][80:96] = True
    hidden[1][:16] = True
    c.run()
    c.check(hidden)


def test_lengths_beyond_the_capacity():
    """A length that the cache cannot hold: all of its rows are seen, no drafted ones."""
    c = Tree("bf16", [90], 2, 1, 4, 64, spare=0, seed=7)
    c.keep[0].fill_(10 ** 9)
    c.k[0], c.v[0] = c.k[0][:, :94], c.v[0][:, :94]
    c.see[:] = True
    c.run()
    c.check()


@pytest.mark.parametrize("value", (math.nan, math.inf))
def test_siblings_do_not_see_each_others_infinities(value):
    c = Tree("bf16", [50], 2, 1, 6, 64, mask="tree", seed=8)
    rows = c.see[0, :, 4].clone()
    p, r = c.place(0, torch.tensor([54]))
    c.gv[int(p), int(r)] = value
    c.run()
    c.v[0][:, 54] = 0.0
    torch.cuda.synchronize()
    out, hit = c.out.clone(), rows.nonzero().flatten().tolist()
    assert hit and not torch.isfinite(out[0, :, hit]).any()
    rest = [i for i in range(6) if i not in hit]
    see = torch.cat((torch.ones(6, 50, dtype=torch.bool), c.see[0]), dim=1)
    for j in range(2):
        x, e = attend(c.q[0, j], c.k[0][0], c.v[0][0], see, c.scale, dtype=c.t)["out"]
        check("rest", out[0, j, rest], x[rest], e[rest])


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("page", (0, 8))
@pytest.mark.parametrize("rot", (0, 32, 64))
def test_append(dtype, page, rot):
    """Rotated keys and values go behind each sequence's rows and nowhere else."""
    c = Tree(dtype, [20, 0, -1, 7], 4, 2, 5, 64, page=page, seed=9)
    t, code = DT[dtype]
    g = torch.Generator().manual_seed(10)
    k, v = torch.randn(4, 2, 5, 64, generator=g).to(t), torch.randn(4, 2, 5, 64, generator=g).to(t)
    q = torch.randn(4, 4, 5, 64, generator=g).to(t)
    gk, gv, gq = k.cuda(), v.cuda(), q.cuda()
    qo = torch.full_like(gq, 7.0)
    pos = c.keep[1]
    cfg = fa.append_config(5, rotary=fa.rotary_config(code, 64, rot) if rot else None,
                           q_layout=fa.rotary_tensor(4) if rot else None)
    before = (c.gk.clone(), c.gv.clone())
    fa.cache_append_device(c.cache, cfg, gk.data_ptr(), gv.data_ptr(), pos.data_ptr(), gq.data_ptr(), qo.data_ptr(),
                           stream())
    torch.cuda.synchronize()
    f, gain = frequencies(rot) if rot else (torch.zeros(0, dtype=torch.float64), 1.0)
    for i, x in enumerate(c.lens):
        if x < 0:
            continue
        p, r = c.place(i, torch.arange(x, x + 5))
        want = rotate(k[i:i + 1].double(), c.pos[i:i + 1], f, gain, False)
        bound = rotary_bound(k[i:i + 1].double(), want, c.pos, gain, t)
        check("k", c.gk.cpu()[p, r].transpose(0, 1)[None], want, bound)
        assert torch.equal(c.gv.cpu()[p, r].transpose(0, 1), v[i])
        for now, was in ((c.gk, before[0]), (c.gv, before[1])):
            was[p.cuda(), r.cuda()] = now[p.cuda(), r.cuda()]
    for now, was in ((c.gk, before[0]), (c.gv, before[1])):
        assert torch.equal(torch.isnan(now), torch.isnan(was))
        assert torch.equal(now.nan_to_num(0), was.nan_to_num(0))
    if rot:
        want = rotate(q.double(), c.pos, f, gain, False)
        check("q", qo, want, rotary_bound(q.double(), want, c.pos, gain, t))
    else:
        assert (qo == 7.0).all()


def test_append_stops_at_the_capacity_and_skips_bad_pages():
    c = Tree("bf16", [6, 20], 2, 1, 4, 64, page=8, spare=0, seed=11)
    k = torch.ones(2, 1, 4, 64, dtype=torch.bfloat16, device="cuda")
    c.keep[0].copy_(torch.tensor([22, 20], dtype=torch.int32))   # 24 rows a sequence
    table = c.table.clone()
    table[1, 2] = 99
    c.keep[3].copy_(table)
    before = c.gk.clone()
    fa.cache_append_device(c.cache, fa.append_config(4), k.data_ptr(), k.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    p, r = c.place(0, torch.arange(22, 24))
    assert (c.gk.cpu()[p, r] == 1).all()
    before[p.cuda(), r.cuda()] = 1.0
    assert torch.equal(c.gk.nan_to_num(0), before.nan_to_num(0))


def test_a_step_as_it_is_used():
    """Prefill (score attention), then drafted tokens: rotary + append + tree, against attention in float64 over all rows."""
    t, code = DT["f16"]
    g = torch.Generator().manual_seed(12)
    b, h, hk, s, n, d = 2, 4, 2, 70, 5, 64
    cfg = fa.rotary_config(code, d, d, scaling=fa.ROTARY_YARN, factor=4.0, original_len=64)
    q, k, v = (torch.randn(b, x, s + n, d, generator=g).to(t) for x in (h, hk, hk))
    cap = s + n + 3
    kc, vc = (torch.zeros(b, hk, cap, d, dtype=t, device="cuda") for _ in range(2))
    pos = torch.arange(s + n, dtype=torch.int32)[None].repeat(b, 1)
    lens = torch.zeros(b, dtype=torch.int32, device="cuda")
    cache = fa.kv_cache(code, b, hk, d, kc.data_ptr(), vc.data_ptr(), lens.data_ptr(), capacity=cap)
    f, gain = frequencies(d, 10000.0, fa.ROTARY_YARN, 4.0, 64)
    got, qrot = [], torch.empty(b, h, s + n, d, dtype=t)
    for lo, hi in ((0, s), (s, s + n)):   # prompt, then the drafted chain
        m = hi - lo
        gq, gk, gv = (x[:, :, lo:hi].contiguous().cuda() for x in (q, k, v))
        gp = pos[:, lo:hi].contiguous().cuda()
        qo, out = torch.empty_like(gq), torch.empty_like(gq)
        app = fa.append_config(m, rotary=cfg, q_layout=fa.rotary_tensor(h))
        fa.cache_append_device(cache, app, gk.data_ptr(), gv.data_ptr(), gp.data_ptr(), gq.data_ptr(), qo.data_ptr(),
                               stream())
        if lo == 0:   # the prompt attends to itself in the cache it just filled
            c = fa.score_config(code, b, h, hk, s, s, d, causal=True,
                                strides={x: (hk * cap * d, d, cap * d) for x in ("k", "v")})
            fa.score_attention_device(c, qo.data_ptr(), kc.data_ptr(), vc.data_ptr(), out.data_ptr(), 0, stream())
            lens.fill_(s)
        else:
            fa.tree_attention_device(fa.tree_config(h, n), cache, qo.data_ptr(), out.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        got.append(out.cpu())
        qrot[:, :, lo:hi] = qo.cpu()
    kr = rotate(k.double(), pos, f, gain, False)
    check("keys", kc[:, :, :s + n], kr, rotary_bound(k.double(), kr, pos, gain, t))
    see = torch.arange(s + n)[None, :] <= torch.arange(s + n)[:, None]
    for i in range(b):
        for j in range(h):
            x, e = attend(qrot[i, j], kc[i, j // 2, :s + n].cpu(), vc[i, j // 2, :s + n].cpu(), see, d ** -0.5, dtype=t)["out"]
            check("out", torch.cat([y[i, j] for y in got]), x, e)


def test_training_through_rotary_and_attention():
    """Gradients of the unrotated Q and K: rotary, attention, its backward, rotary inverse, against autograd in float64."""
    g = torch.Generator().manual_seed(13)
    b, h, hk, s, d = 1, 2, 1, 60, 32
    q, k, v, do = (torch.randn(b, x, s, d, generator=g) for x in (h, hk, hk, h))
    pos = torch.arange(s, dtype=torch.int32)[None].repeat(b, 1)
    cfg = fa.rotary_config(fa.DTYPE_F32, d, d, interleaved=True)
    tq, tk, gp = fa.rotary_tensor(h), fa.rotary_tensor(hk), pos.cuda()
    gq, gk, gv, gdo = (x.cuda() for x in (q, k, v, do))
    qr, kr, out, dq, dk, dv = (torch.empty_like(x) for x in (gq, gk, gq, gq, gk, gv))
    lse = torch.empty(b, h, s, device="cuda")
    c = fa.score_config(fa.DTYPE_F32, b, h, hk, s, s, d, causal=True, softcap=8.0)
    fa.rotary_device(cfg, b, s, gp.data_ptr(), tq, gq.data_ptr(), qr.data_ptr(), tk, gk.data_ptr(), kr.data_ptr(), stream())
    p = [x.data_ptr() for x in (qr, kr, gv, out, lse)]
    fa.score_attention_device(c, *p, stream())
    fa.score_attention_backward_device(c, *p, gdo.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), stream())
    fa.rotary_device(cfg, b, s, gp.data_ptr(), tq, dq.data_ptr(), dq.data_ptr(), tk, dk.data_ptr(), dk.data_ptr(), stream(),
                     inverse=True)
    torch.cuda.synchronize()
    f, gain = frequencies(d)
    ref = [x.double().requires_grad_() for x in (q, k, v)]
    rq, rk = (rotate(x, pos, f, gain, True) for x in ref[:2])
    z = 8.0 * torch.tanh(rq @ rk.repeat_interleave(2, 1).transpose(2, 3) / math.sqrt(d) / 8.0)
    z = z.masked_fill(torch.arange(s)[None, :] > torch.arange(s)[:, None], -math.inf)
    o = torch.softmax(z, -1) @ ref[2].repeat_interleave(2, 1)
    grads = torch.autograd.grad((o * do.double()).sum(), ref)
    for name, got, want in zip(("dq", "dk", "dv"), (dq, dk, dv), grads):
        # f32 throughout: some 60 products and sums a value, each within 2^-24 of the largest terms
        assert (got.double().cpu() - want).abs().max() <= 1e-5 * max(1.0, want.abs().max().item()), name


def test_tree_graph_replays_and_two_streams():
    """Captured steps on a growing cache; two captured graphs and eager calls do not share partial sums."""
    cases = [Tree("bf16", [600, 900], 8, 2, 4, 128, page=16, spare=40, seed=s) for s in (14, 15)]
    side, graphs = torch.cuda.Stream(), []
    for c in cases:
        with torch.cuda.stream(side):
            c.run()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            c.run()
        graphs.append(graph)
    extra = Tree("bf16", [5000], 8, 2, 4, 128, seed=16)
    other = torch.cuda.Stream()
    for _ in range(3):
        for c in cases:
            c.out.fill_(7.0)
        side.synchronize()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        extra.run()
        torch.cuda.synchronize()
        for c in cases + [extra]:
            c.check()


@pytest.mark.parametrize("n", (63, 64, 65, 128, 256))
def test_chains_longer_than_a_mask_word(n):
    """No mask: token i sees tokens up to i, also past the first 64."""
    c = Tree("bf16", [40, 7], 2, 2, n, 64, mask="chain", seed=n)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("n", (3, 40))
def test_more_sequences_than_lanes(dtype, n):
    """70 and 140 sequences of all lengths, idle ones among them."""
    for b in (70, 140):
        lens = [(37 * i) % 300 if i % 9 else -1 for i in range(b)]
        c = Tree(dtype, lens, 2, 1, n, 64, page=16, seed=b)
        c.run()
        c.check()


@pytest.mark.parametrize("n", (4, 48))
def test_pages_far_into_the_pool(n):
    """Pages whose offsets pass 2^32 elements give what the same pages at the start of a small pool give."""
    c = Tree("bf16", [1500, 700], 4, 2, n, 128, page=256, seed=17)
    g = torch.Generator().manual_seed(18)
    new_k, new_v = (torch.randn(2, 2, n, 128, generator=g).bfloat16().cuda() for _ in range(2))
    cfg = fa.append_config(n)
    fa.cache_append_device(c.cache, cfg, new_k.data_ptr(), new_v.data_ptr(), stream=stream())
    c.run()
    torch.cuda.synchronize()
    want, want_lse = c.out.clone(), c.lse.clone()
    pages = c.gk.shape[0]
    total = 2 ** 32 // (256 * 2 * 128) + pages
    at = total - pages
    far = [torch.empty((total, 256, 2, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for pool, small in zip(far, (c.kc, c.vc)):
        pool[at:].copy_(small)
    assert far[0][at:].storage_offset() >= 2 ** 32
    c.keep[3].add_(at)
    c.cache.k, c.cache.v, c.cache.n_pages = far[0].data_ptr(), far[1].data_ptr(), total
    c.out.fill_(7.0)
    fa.cache_append_device(c.cache, cfg, new_k.data_ptr(), new_v.data_ptr(), stream=stream())
    c.run()
    torch.cuda.synchronize()
    assert torch.equal(c.out, want) and torch.equal(c.lse, want_lse)
    for pool, small in zip(far, (c.gk, c.gv)):
        assert torch.equal(pool[at:].nan_to_num(0), small.nan_to_num(0))
