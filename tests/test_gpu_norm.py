"""Norms of queries and keys with rotary positions on the GPU, against float64.

Bounds: rotations as in test_gpu_rotary_tree (rotary_bound).  A row's sum of squares is within d 2^-24 of
itself, so r within (d / 2 + 4) 2^-24; products and differences each add 2^-24 of their terms.
"""
from __future__ import annotations

import math

import pytest
import torch

import flash_attention_amd as fa
from ops_reference import EPS32, check, unit
from test_gpu_rotary_tree import Tree, frequencies, rotate, rotary_bound
from test_gpu_score import DT, filled, make, strides, to_gpu

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


def normed(x, w, eps):
    x = x.double()
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()


def forward_expect(x, w, eps, pos, f, gain, interleaved, dtype):
    n = normed(x, w, eps)
    y = rotate(n, pos, f, gain, interleaved)
    d = x.shape[-1]
    far = (d / 2 + 6) * EPS32 * n.abs().amax(-1, keepdim=True) * 2 * gain
    e = rotary_bound(n, y, pos, gain, torch.float32) + far
    return y, e + unit(dtype) * (y.abs() + e) + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def backward_expect(x, dy, w, eps, pos, f, gain, interleaved, dtype):
    """(dx, bound), (dw, bound)."""
    x, dy, w = x.double(), dy.double(), w.double()
    d = x.shape[-1]
    rs = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    g = rotate(dy, pos, f, gain, interleaved, True)
    eg = rotary_bound(dy, g, pos, gain, torch.float32)
    far = (d / 2 + 6) * EPS32   # of rs
    m = (w * g * x).mean(-1, keepdim=True) * rs ** 2
    em = rs ** 2 * ((w * x).abs() * eg + (d + 4) * EPS32 * (w * g * x).abs()).mean(-1, keepdim=True) + m.abs() * 2 * far
    dx = rs * (w * g - x * m)
    edx = rs * (w.abs() * eg + x.abs() * em + 4 * EPS32 * ((w * g).abs() + (x * m).abs())) + dx.abs() * far
    edx = edx + unit(dtype) * (dx.abs() + edx) + (2.0 ** -25 if dtype == torch.float16 else 0.0) + 1e-37
    y = x * rs
    n = x.numel() // d
    dw = (g * y).sum((0, 1, 2))
    edw = (y.abs() * eg + (g * y).abs() * (far + (n + 4) * EPS32)).sum((0, 1, 2)) + 1e-37
    return (dx, edx), (dw, edw)


class Norm:
    def __init__(self, dtype, b, h, hk, s, d, rot, interleaved=False, layout="bhsd", pad=0, eps=1e-6, weights=True,
                 far=300000, scaling=fa.ROTARY_NONE, sigma=1.0, seed=0):
        self.t, code = DT[dtype]
        g = torch.Generator().manual_seed(seed)
        self.b, self.s, self.d, self.eps, self.interleaved, self.heads = b, s, d, eps, interleaved, (h, hk)
        self.x = [make(g, self.t, b, n, s, d, sigma, layout, pad) for n in self.heads]
        self.dy = [make(g, self.t, b, n, s, d, 1.0, layout, pad) for n in self.heads]
        self.w = [(1 + 0.3 * torch.randn(d, generator=g)).to(self.t) if weights else torch.ones(d) for _ in range(2)]
        self.pos = torch.randint(0, far, (b, s), generator=g, dtype=torch.int32)
        self.cfg = fa.rotary_config(code, d, rot, interleaved=interleaved, scaling=scaling, factor=4.0, original_len=512)
        self.f, self.gain = frequencies(rot, 10000.0, scaling, 4.0, 512)
        self.gx, self.gdy = [to_gpu(x) for x in self.x], [to_gpu(x) for x in self.dy]
        self.gw, self.gpos = [w.cuda() for w in self.w], self.pos.cuda()
        self.y, self.dx = [filled(x) for x in self.x], [filled(x) for x in self.x]
        self.dw = [torch.full((d,), 7.0, device="cuda") for _ in range(2)]
        self.norm = fa.head_norm(*(w.data_ptr() if weights else 0 for w in self.gw), eps)

    def forward(self):
        t = [fa.rotary_tensor(h, strides(x), strides(y)) for h, x, y in zip(self.heads, self.gx, self.y)]
        fa.norm_rotary_device(self.cfg, self.norm, self.b, self.s, self.gpos.data_ptr(), t[0], self.gx[0].data_ptr(),
                              self.y[0].data_ptr(), t[1], self.gx[1].data_ptr(), self.y[1].data_ptr(), stream())

    def backward(self, dx=True, dw=True):
        t = [fa.norm_grad(h, strides(x), strides(y), strides(z))
             for h, x, y, z in zip(self.heads, self.gx, self.gdy, self.dx)]
        args = []
        for i in range(2):
            args += [t[i], self.gx[i].data_ptr(), self.gdy[i].data_ptr(), self.dx[i].data_ptr() if dx else 0,
                     self.dw[i].data_ptr() if dw else 0]
        fa.norm_rotary_backward_device(self.cfg, self.norm, self.b, self.s, self.gpos.data_ptr(), *args, stream())

    def check_forward(self):
        torch.cuda.synchronize()
        for i in range(2):
            check(f"y{i}", self.y[i], *forward_expect(self.x[i], self.w[i], self.eps, self.pos, self.f, self.gain,
                                                      self.interleaved, self.t))

    def check_backward(self, dx=True, dw=True):
        torch.cuda.synchronize()
        for i in range(2):
            ex, ew = backward_expect(self.x[i], self.dy[i], self.w[i], self.eps, self.pos, self.f, self.gain,
                                     self.interleaved, self.t)
            if dx:
                check(f"dx{i}", self.dx[i], *ex)
            else:
                assert (self.dx[i] == 7).all()
            if dw:
                check(f"dw{i}", self.dw[i], *ew)
            else:
                assert (self.dw[i] == 7).all()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("d,rot", ((64, 64), (128, 128), (128, 64), (80, 40), (256, 256), (256, 16), (50, 18), (2, 2), (7, 6),
                                   (255, 254)))
@pytest.mark.parametrize("layout,pad", (("bhsd", 0), ("bshd", 8), ("bshd", 3)))
def test_forward_and_backward(dtype, interleaved, d, rot, layout, pad):
    c = Norm(dtype, 2, 6, 3, 37, d, rot, interleaved, layout, pad, seed=d + rot)
    c.forward()
    c.check_forward()
    c.backward()
    c.check_backward()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("b,s,h,hk", ((1, 1, 1, 1), (1, 1, 64, 8), (3, 1, 5, 5), (700, 3, 2, 1), (2, 2500, 4, 1), (1, 9000, 1, 1)))
def test_sizes(dtype, b, s, h, hk):
    """One token to many, rows that fill no workgroup, tokens of several sequences in one."""
    c = Norm(dtype, b, h, hk, s, 128, 128, layout="bshd", seed=s)
    c.forward()
    c.check_forward()
    c.backward()
    c.check_backward()


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("kw", ({"weights": False}, {"scaling": fa.ROTARY_YARN}, {"eps": 0.5}, {"sigma": 1e-3},
                                {"sigma": 1e4}, {"far": 1}))
def test_options(dtype, kw):
    c = Norm(dtype, 2, 4, 2, 50, 64, 64, seed=3, **kw)
    c.forward()
    c.check_forward()
    c.backward()
    c.check_backward()


def test_rows_of_zeros():
    """y = 0, dx = w g / sqrt(eps)."""
    c = Norm("f32", 1, 2, 1, 9, 64, 64, seed=4)
    c.x[0][0, 1, 3], c.gx[0][0, 1, 3] = 0, 0
    c.forward()
    c.check_forward()
    c.backward()
    c.check_backward()
    assert (c.y[0][0, 1, 3] == 0).all()


def test_what_is_not_finite_stays_in_its_row():
    c = Norm("bf16", 1, 4, 2, 9, 64, 64, seed=5)
    c.gx[0][0, 1, 3, 5] = math.nan
    c.gdy[1][0, 1, 3, 5] = math.inf
    c.forward()
    c.backward(dw=False)
    torch.cuda.synchronize()
    assert torch.isnan(c.y[0][0, 1, 3]).all() and torch.isnan(c.dx[0][0, 1, 3]).all()
    for i, t in ((0, c.y[0]), (0, c.dx[0]), (1, c.dx[1])):
        rest = torch.isfinite(t).all(-1)
        rest[0, 1, 3] = True
        assert rest.all()


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("d,rot,interleaved", ((64, 64, False), (128, 128, True), (80, 40, False), (50, 18, True), (80, 40, True)))
@pytest.mark.parametrize("big", (1e20, 3e38))
def test_rows_whose_squares_pass_the_range(dtype, d, rot, interleaved, big):
    """Zeros forward and backward, whatever the sums that enter the gradients; other rows as ever."""
    c = Norm(dtype, 1, 3, 2, 9, d, rot, interleaved, "bshd", seed=8)
    for x, gx in zip(c.x, c.gx):
        x[0, 1, 3] = big
        gx.copy_(x)
    c.gdy[0][0, 1, 3] = c.gdy[0][0, 1, 3].abs() * 100
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    for t in c.y + c.dx:
        assert (t[0, 1, 3] == 0).all() and torch.isfinite(t).all()
    for i in range(2):
        c.x[i][0, 1, 3] = 0   # the row's share of the weights' gradients is 0 then too
        (dx, edx), (dw, edw) = backward_expect(c.x[i], c.dy[i], c.w[i], c.eps, c.pos, c.f, c.gain, interleaved, c.t)
        dx[0, 1, 3] = 0
        check("dx", c.dx[i], dx, edx)
        check("dw", c.dw[i], dw, edw)


def test_infinite_rows_are_no_numbers_backward():
    c = Norm("bf16", 1, 2, 1, 5, 64, 64, seed=9)
    c.gx[0][0, 1, 2, 7] = math.inf
    c.backward()
    torch.cuda.synchronize()
    assert torch.isnan(c.dx[0][0, 1, 2]).all()
    keep = torch.ones(1, 2, 5, dtype=torch.bool)
    keep[0, 1, 2] = False
    assert torch.isfinite(c.dx[0][keep.cuda()]).all()


@pytest.mark.parametrize("dx,dw", ((True, False), (False, True)))
def test_single_gradients(dx, dw):
    c = Norm("bf16", 2, 4, 2, 50, 64, 64, seed=6)
    c.backward(dx, dw)
    c.check_backward(dx, dw)


@pytest.mark.parametrize("dtype", ("f32", "f16"))
def test_in_place_and_one_tensor(dtype):
    c = Norm(dtype, 2, 4, 2, 50, 128, 64, seed=7)
    keep = c.y[1].clone()
    x = c.gx[0].clone()
    t = fa.rotary_tensor(4)
    fa.norm_rotary_device(c.cfg, c.norm, 2, 50, c.gpos.data_ptr(), t, x.data_ptr(), x.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    check("in place", x, *forward_expect(c.x[0], c.w[0], c.eps, c.pos, c.f, c.gain, False, c.t))
    assert torch.equal(c.y[1], keep)
    ex, ew = backward_expect(c.x[0], c.dy[0], c.w[0], c.eps, c.pos, c.f, c.gain, False, c.t)
    for target in ("x", "dy"):
        x, dy = c.gx[0].clone(), c.gdy[0].clone()
        to = x if target == "x" else dy
        fa.norm_rotary_backward_device(c.cfg, c.norm, 2, 50, c.gpos.data_ptr(), fa.norm_grad(4), x.data_ptr(), dy.data_ptr(),
                                       to.data_ptr(), c.dw[0].data_ptr(), stream=stream())
        torch.cuda.synchronize()
        check("dx", to, *ex)
        check("dw", c.dw[0], *ew)


def test_no_rows():
    """The weights' gradients of no rows are zeros; nothing else is written."""
    c = Norm("f32", 1, 2, 1, 4, 64, 64, seed=8)
    g = fa.norm_grad(2)
    fa.norm_rotary_backward_device(c.cfg, c.norm, 1, 0, 0, g, 0, 0, c.dx[0].data_ptr(), c.dw[0].data_ptr(), stream=stream())
    torch.cuda.synchronize()
    assert (c.dw[0] == 0).all() and (c.dx[0] == 7).all()
    fa.norm_rotary_backward_device(c.cfg, c.norm, 1, 4, c.gpos.data_ptr(), fa.norm_grad(0), 0, 0, c.dx[0].data_ptr(),
                                   c.dw[0].data_ptr(), g, c.gx[0].data_ptr(), c.gdy[0].data_ptr(), c.dx[0].data_ptr(),
                                   c.dw[1].data_ptr(), stream())
    torch.cuda.synchronize()
    ex, ew = backward_expect(c.x[0], c.dy[0], c.w[1], c.eps, c.pos, c.f, c.gain, False, c.t)
    assert (c.dw[0] == 0).all()
    check("dw", c.dw[1], *ew)
    check("dx", c.dx[0], *ex)


def test_broadcast_inputs():
    """One row read by all heads and batches (strides of 0): each place gets its own result."""
    t, code = DT["f32"]
    g = torch.Generator().manual_seed(9)
    x = torch.randn(7, 64, generator=g)
    pos = torch.randint(0, 100, (2, 7), generator=g, dtype=torch.int32)
    cfg, norm = fa.rotary_config(code, 64, 64), fa.head_norm(eps=1e-5)
    gx, y, gp = x.cuda(), torch.empty(2, 3, 7, 64, device="cuda"), pos.cuda()
    fa.norm_rotary_device(cfg, norm, 2, 7, gp.data_ptr(), fa.rotary_tensor(3, (0, 64, 0)), gx.data_ptr(), y.data_ptr(),
                          stream=stream())
    torch.cuda.synchronize()
    f, gain = frequencies(64)
    check("y", y, *forward_expect(x.expand(2, 3, 7, 64), torch.ones(64), 1e-5, pos, f, gain, False, t))


def test_gradients_against_differences():
    c = Norm("f32", 1, 2, 1, 20, 64, 32, seed=10)
    c.backward()
    torch.cuda.synchronize()
    g = torch.Generator().manual_seed(11)
    eps = 2.0 ** -8

    def loss():
        c.forward()
        torch.cuda.synchronize()
        return sum((y.double() * dy.double()).sum().item() for y, dy in zip(c.y, c.gdy))
    for i in range(2):
        for x, grad in ((c.gx[i], c.dx[i]), (c.gw[i], c.dw[i])):
            way, base, got = torch.randn(x.shape, generator=g).cuda(), x.clone(), []
            for s in (eps, -eps):
                x.copy_(base + s * way)
                got.append(loss())
            x.copy_(base)
            want = (grad.double() * way.double()).sum().item()
            # rounding: 3840 values of order 1 within 2^-20 at worst, over 2 eps: 0.48; curvature: eps^2 of 3840 terms: 0.06
            assert abs((got[0] - got[1]) / (2 * eps) - want) < 0.6


def test_the_same_bits_every_time():
    c = Norm("bf16", 2, 8, 2, 3000, 128, 128, seed=12)
    seen = []
    for _ in range(3):
        c.backward()
        torch.cuda.synchronize()
        seen.append([x.clone() for x in c.dx + c.dw])
    assert all(torch.equal(a, b) for other in seen[1:] for a, b in zip(seen[0], other))


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("page", (0, 8))
@pytest.mark.parametrize("d,rot", ((64, 32), (128, 128), (36, 20)))
def test_append(dtype, page, d, rot):
    """Normed and rotated keys, and values as they are, behind each sequence's rows and nowhere else."""
    c = Tree(dtype, [20, 0, -1, 7], 4, 2, 5, d, page=page, seed=13)
    t, code = DT[dtype]
    g = torch.Generator().manual_seed(14)
    k, v = torch.randn(4, 2, 5, d, generator=g).to(t), torch.randn(4, 2, 5, d, generator=g).to(t)
    q = torch.randn(4, 4, 5, d, generator=g).to(t)
    w = [(1 + 0.3 * torch.randn(d, generator=g)).to(t) for _ in range(2)]
    gk, gv, gq, gw = k.cuda(), v.cuda(), q.cuda(), [x.cuda() for x in w]
    qo = torch.full_like(gq, 7.0)
    cfg = fa.append_config(5, rotary=fa.rotary_config(code, d, rot), q_layout=fa.rotary_tensor(4))
    before = (c.gk.clone(), c.gv.clone())
    fa.cache_append_device(c.cache, cfg, gk.data_ptr(), gv.data_ptr(), c.keep[1].data_ptr(), gq.data_ptr(), qo.data_ptr(),
                           stream(), norm=fa.head_norm(gw[0].data_ptr(), gw[1].data_ptr(), 1e-6))
    torch.cuda.synchronize()
    f, gain = frequencies(rot)
    for i, x in enumerate(c.lens):
        if x < 0:
            continue
        p, r = c.place(i, torch.arange(x, x + 5))
        check("k", c.gk.cpu()[p, r].transpose(0, 1)[None],
              *forward_expect(k[i:i + 1], w[1], 1e-6, c.pos[i:i + 1], f, gain, False, t))
        assert torch.equal(c.gv.cpu()[p, r].transpose(0, 1), v[i])
        for now, was in ((c.gk, before[0]), (c.gv, before[1])):
            was[p.cuda(), r.cuda()] = now[p.cuda(), r.cuda()]
    for now, was in ((c.gk, before[0]), (c.gv, before[1])):
        assert torch.equal(torch.isnan(now), torch.isnan(was))
        assert torch.equal(now.nan_to_num(0), was.nan_to_num(0))
    check("q", qo, *forward_expect(q, w[0], 1e-6, c.pos, f, gain, False, t))


@pytest.mark.parametrize("dtype,page,d,rot,n", (("bf16", 16, 128, 128, 700), ("f16", 0, 80, 40, 333), ("f32", 64, 128, 64, 501),
                                                ("bf16", 0, 64, 64, 1)))
def test_append_of_prompts(dtype, page, d, rot, n):
    """Hundreds of tokens of sequences of unequal length, in place of a first or a later part of a prompt."""
    c = Tree(dtype, [0, 333, -1, 15, 16], 6, 2, n, d, page=page, mask="chain", seed=20)
    t, code = DT[dtype]
    g = torch.Generator().manual_seed(21)
    k, v, q = (torch.randn(5, x, n, d, generator=g).to(t) for x in (2, 2, 6))
    w = [(1 + 0.3 * torch.randn(d, generator=g)).to(t) for _ in range(2)]
    gk, gv, gq, gw = k.cuda(), v.cuda(), q.cuda(), [x.cuda() for x in w]
    cfg = fa.append_config(n, rotary=fa.rotary_config(code, d, rot), q_layout=fa.rotary_tensor(6))
    fa.cache_append_device(c.cache, cfg, gk.data_ptr(), gv.data_ptr(), c.keep[1].data_ptr(), gq.data_ptr(), gq.data_ptr(),
                           stream(), norm=fa.head_norm(gw[0].data_ptr(), gw[1].data_ptr(), 1e-5))
    torch.cuda.synchronize()
    f, gain = frequencies(rot)
    rows, values = c.gk.cpu(), c.gv.cpu()
    for i, x in enumerate(c.lens):
        if x < 0:
            continue
        p, r = c.place(i, torch.arange(x, x + n))
        check(f"k {i}", rows[p, r].transpose(0, 1)[None],
              *forward_expect(k[i:i + 1], w[1], 1e-5, c.pos[i:i + 1], f, gain, False, t))
        assert torch.equal(values[p, r].transpose(0, 1), v[i])
        if x:   # rows that were there stay
            p, r = c.place(i, torch.arange(x))
            assert torch.equal(rows[p, r].transpose(0, 1), c.k[i][:, :x]) and torch.equal(values[p, r].transpose(0, 1), c.v[i][:, :x])
    check("q", gq, *forward_expect(q, w[0], 1e-5, c.pos, f, gain, False, t))


def test_append_stops_at_the_capacity_and_skips_bad_pages():
    c = Tree("bf16", [6, 20], 2, 1, 4, 64, page=8, spare=0, seed=15)
    k = torch.ones(2, 1, 4, 64, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    c.keep[0].copy_(torch.tensor([22, 20], dtype=torch.int32))   # 24 rows a sequence
    table = c.table.clone()
    table[1, 2] = 99
    c.keep[3].copy_(table)
    before = c.gv.clone()
    cfg = fa.append_config(4, rotary=fa.rotary_config(fa.DTYPE_BF16, 64, 64))
    fa.cache_append_device(c.cache, cfg, k.data_ptr(), k.data_ptr(), pos.data_ptr(), stream=stream(),
                           norm=fa.head_norm())
    torch.cuda.synchronize()
    p, r = c.place(0, torch.arange(22, 24))
    assert (c.gv.cpu()[p, r] == 1).all()
    before[p.cuda(), r.cuda()] = 1.0
    assert torch.equal(c.gv.nan_to_num(0), before.nan_to_num(0))


def test_captured_on_another_stream():
    c = Norm("bf16", 2, 8, 2, 600, 128, 128, seed=16)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c.forward()
        c.backward()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            c.forward()
            c.backward()
        for _ in range(3):
            for x in c.y + c.dx + c.dw:
                x.fill_(7.0)
            graph.replay()
            side.synchronize()
            c.check_forward()
            c.check_backward()
            c.backward()
            side.synchronize()


def test_training_through_norm_and_windowed_attention():
    """Norms, rotary positions, attention in a window with sinks and all gradients, against autograd in float64."""
    g = torch.Generator().manual_seed(17)
    b, h, hk, s, d, size, sinks, eps = 1, 2, 1, 150, 32, 40, 3, 1e-6
    q, k, v, do = (torch.randn(b, x, s, d, generator=g) for x in (h, hk, hk, h))
    w = [1 + 0.3 * torch.randn(d, generator=g) for _ in range(2)]
    pos = torch.arange(s, dtype=torch.int32)[None].repeat(b, 1)
    cfg, gp = fa.rotary_config(fa.DTYPE_F32, d, d), pos.cuda()
    gq, gk, gv, gdo, gw = q.cuda(), k.cuda(), v.cuda(), do.cuda(), [x.cuda() for x in w]
    norm = fa.head_norm(gw[0].data_ptr(), gw[1].data_ptr(), eps)
    qr, kr, out, dqr, dkr, dv = (torch.empty_like(x) for x in (gq, gk, gq, gq, gk, gv))
    dw = [torch.empty(d, device="cuda") for _ in range(2)]
    lse = torch.empty(b, h, s, device="cuda")
    c, win = fa.score_config(fa.DTYPE_F32, b, h, hk, s, s, d, causal=True), fa.window(size, sinks)
    fa.norm_rotary_device(cfg, norm, b, s, gp.data_ptr(), fa.rotary_tensor(h), gq.data_ptr(), qr.data_ptr(),
                          fa.rotary_tensor(hk), gk.data_ptr(), kr.data_ptr(), stream())
    p = [x.data_ptr() for x in (qr, kr, gv, out, lse)]
    fa.score_attention_device(c, *p, stream(), window=win)
    fa.score_attention_backward_device(c, *p, gdo.data_ptr(), dqr.data_ptr(), dkr.data_ptr(), dv.data_ptr(), stream(),
                                       window=win)
    fa.norm_rotary_backward_device(cfg, norm, b, s, gp.data_ptr(), fa.norm_grad(h), gq.data_ptr(), dqr.data_ptr(),
                                   dqr.data_ptr(), dw[0].data_ptr(), fa.norm_grad(hk), gk.data_ptr(), dkr.data_ptr(),
                                   dkr.data_ptr(), dw[1].data_ptr(), stream())
    torch.cuda.synchronize()
    f, gain = frequencies(d)
    ref = [x.double().requires_grad_() for x in (q, k, v, *w)]
    rq, rk = (rotate(normed(x, y, eps), pos, f, gain, False) for x, y in ((ref[0], ref[3]), (ref[1], ref[4])))
    z = rq @ rk.repeat_interleave(2, 1).transpose(2, 3) / math.sqrt(d)
    i, j = torch.arange(s)[:, None], torch.arange(s)[None, :]
    z = z.masked_fill((j > i) | ((i - j >= size) & (j >= sinks)), -math.inf)
    o = torch.softmax(z, -1) @ ref[2].repeat_interleave(2, 1)
    grads = torch.autograd.grad((o * do.double()).sum(), ref)
    for name, got, want in zip(("dq", "dk", "dv", "dqw", "dkw"), (dqr, dkr, dv, *dw), grads):
        # f32 throughout: some 60 products and sums a value, each within 2^-24 of the largest terms; the weights' sums
        # of up to 300 rows besides
        assert (got.double().cpu() - want).abs().max() <= 2e-5 * max(1.0, want.abs().max().item()), name
