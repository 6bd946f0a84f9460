"""The cache in 4 bits on the GPU: append, rows read back, attention over it.

What codes stand for is exact, so the cache's words are compared as they are.  Attention is compared with float64
over the values that enter its products (rounded once to f16, as probabilities are): bounds of ops_reference for f16, and
half a step of the output's type.
"""
from __future__ import annotations

import math

import pytest
import torch

import flash_attention_amd as fa
from ops_reference import attend, check, unit
from test_gpu_norm import normed
from test_gpu_rotary_tree import frequencies, rotate
from test_gpu_score import DT, filled, make, strides, to_gpu

pytestmark = pytest.mark.gpu

SHIFTS = [4 * (e // 2) + 16 * (e % 2) for e in range(8)]
NAN16 = 0x7e00


def stream():
    return torch.cuda.current_stream().cuda_stream


def quantise(x):
    """[..., d] -> codes (int64), S, O (f16 [..., d / 32]); the header's definition, operation by operation in f32."""
    y = x.float().unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(y).all(-1)
    y = y.nan_to_num(0, 60000, -60000).clamp(-60000.0, 60000.0)
    lo, hi = y.amin(-1), y.amax(-1)
    big = ((hi - lo) * 16.0 / 15.0).clamp_max(65504.0).half()
    off = (lo - big.float()).clamp_min(-65504.0).half()
    step = (big.float() * 0.0625)[..., None]
    code = torch.round((y - off.float()[..., None]) / step - 16.0).nan_to_num(0).clamp(0, 15)
    code = torch.where((step == 0) | bad[..., None], torch.zeros_like(code), code)
    nan = torch.full_like(big, math.nan)
    return code.flatten(-2).long(), torch.where(bad, nan, big), torch.where(bad, nan, off)


def stands_for(code, big, off):
    """float64 values."""
    c = code.double().unflatten(-1, (-1, 32))
    return (off.double()[..., None] + (1 + c / 16) * big.double()[..., None]).flatten(-2)


class Cache4:
    """Sequences of lens[b] filled rows, contiguous or in shuffled pages; whatever is not a row holds NaN."""

    def __init__(self, dtype, lens, hk, d, page=0, spare=8, room=0, sigma=1.0, seed=0):
        self.t, self.code = DT[dtype]
        self.g = torch.Generator().manual_seed(seed)
        b = len(lens)
        self.b, self.lens, self.hk, self.d, self.page = b, lens, hk, d, page
        rows = -(-(max(max(lens), 0) + room + spare) // 8) * 8
        if page:
            per = -(-rows // page)
            blocks, self.rows, self.capacity = b * per + 3, page, per * page
            self.table = torch.randperm(blocks, generator=self.g)[:b * per].reshape(b, per).to(torch.int32)
        else:
            blocks, self.rows, self.capacity, self.table = b, rows, rows, None
        shapes = fa.cache4_shapes(blocks, hk, self.rows, d)
        self.cpu = {n: torch.randint(-2 ** 31, 2 ** 31 - 1, shapes[n], generator=self.g, dtype=torch.int32) for n in ("k", "v")}
        for n in ("k_scale", "v_scale"):
            self.cpu[n] = torch.full(shapes[n], math.nan, dtype=torch.float16)
        self.k, self.v = [], []   # rows as kept, float64
        for i, x in enumerate(lens):
            for n, keep in (("k", self.k), ("v", self.v)):
                y = (torch.randn(hk, max(x, 0), d, generator=self.g) * sigma).to(self.t)
                q = quantise(y)
                if x > 0:
                    self.put(n, i, torch.arange(x), *q)
                keep.append(stands_for(*q))
        self.upload()

    def place(self, i, rows):
        if self.page:
            return self.table[i].long()[rows // self.page], rows % self.page
        return torch.full_like(rows, i), rows

    def put(self, n, i, rows, code, big, off):
        """Rows of sequence i: codes [heads, rows, d]."""
        p, r = self.place(i, rows)
        scales = torch.stack((big, off), -1).transpose(0, 1)   # [rows, heads, d / 32, 2]
        if n == "k":
            words = sum(code.unflatten(-1, (-1, 8))[..., e] << SHIFTS[e] for e in range(8))
            self.cpu["k"][p, :, r] = words.transpose(0, 1).to(torch.int32)
            self.cpu["k_scale"][p, :, r] = scales
        else:
            for j in range(len(rows)):
                sh = SHIFTS[int(r[j]) % 8]
                old = self.cpu["v"][p[j], :, r[j] // 8].long()
                new = (old & ~(15 << sh)) | (code[:, j] << sh)
                self.cpu["v"][p[j], :, r[j] // 8] = ((new + 2 ** 31) % 2 ** 32 - 2 ** 31).to(torch.int32)
                self.cpu["v_scale"][p[j], :, r[j] // 8, :, :, r[j] % 8] = scales[j]

    def upload(self):
        self.gpu = {n: x.cuda() for n, x in self.cpu.items()}
        self.glens = torch.tensor(self.lens, dtype=torch.int32).cuda()
        self.gtable = None if self.table is None else self.table.cuda()
        self.cache = fa.kv_cache4(self.code, self.b, self.hk, self.d, *(self.gpu[n].data_ptr() for n in
                                                                        ("k", "k_scale", "v", "v_scale")),
                                  self.glens.data_ptr(), capacity=0 if self.page else self.capacity,
                                  block_table_ptr=self.gtable.data_ptr() if self.page else 0, page_size=self.page,
                                  n_pages=self.cpu["k"].shape[0] if self.page else 0,
                                  pages_per_seq=self.table.shape[1] if self.page else 0)

    def same(self):
        """The cache on the GPU is the one on the CPU, bit by bit but for which NaN."""
        torch.cuda.synchronize()
        for n, x in self.cpu.items():
            y = self.gpu[n].cpu()
            if n.endswith("scale"):
                assert torch.equal(torch.isnan(x), torch.isnan(y)), n
                x, y = x.nan_to_num(7.0), y.nan_to_num(7.0)
            assert torch.equal(x, y), (n, (x != y).sum().item(), (x != y).nonzero()[:4].tolist())

    def append(self, k, v, rows=None):
        """k, v: [b, heads, n, d] views on the CPU."""
        n = k.shape[2]
        gk, gv = to_gpu(k), to_gpu(v)
        cfg = fa.append_config(n, k_strides=strides(gk), v_strides=strides(gv))
        fa.cache4_append_device(self.cache, cfg, gk.data_ptr(), gv.data_ptr(), stream())
        for i, x in enumerate(self.lens):
            m = min(n, self.capacity - x)
            if x < 0 or m <= 0:
                continue
            at = torch.arange(x, x + m)
            good = torch.ones(m, dtype=torch.bool)
            if self.page:
                good = (self.place(i, at)[0] >= 0) & (self.place(i, at)[0] < self.cpu["k"].shape[0])
            for name, y in (("k", k), ("v", v)):
                q = quantise(y[i, :, :m][:, good])
                self.put(name, i, at[good], *q)


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("n", (1, 3, 8, 17, 130))
@pytest.mark.parametrize("d", (32, 64, 96, 128, 160, 256))
@pytest.mark.parametrize("page", (0, 8, 32))
def test_append(dtype, n, d, page):
    c = Cache4(dtype, [20, 0, -1, 7, 31], 2, d, page=page, room=n, seed=n + d)
    g = torch.Generator().manual_seed(n)
    c.append(*(make(g, c.t, 5, 2, n, d, 1.0) for _ in range(2)))
    c.same()


@pytest.mark.parametrize("layout,pad", (("bshd", 0), ("bshd", 8), ("bhsd", 3)))
def test_append_layouts(layout, pad):
    c = Cache4("bf16", [3, 14], 3, 64, room=20, seed=1)
    g = torch.Generator().manual_seed(2)
    c.append(*(make(g, c.t, 2, 3, 20, 64, 1.0, layout, pad) for _ in range(2)))
    c.same()


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
def test_groups_of_all_kinds(dtype):
    """Constant, zero, tiny, large and huge groups, infinities, NaN, one value far from the others, halves between codes."""
    c = Cache4(dtype, [5], 1, 64, room=14, seed=3)
    g = torch.Generator().manual_seed(4)
    k = torch.randn(1, 1, 14, 64, generator=g)
    k[..., 0, :] = 3.0
    k[..., 1, :] = 0.0
    k[..., 2, :] *= 1e-6
    k[..., 3, :] *= 5000.0
    k[..., 4, :] *= 50000.0
    k[..., 5, 3] = math.inf
    k[..., 6, 40] = math.nan
    k[..., 7, 9] = -math.inf
    k[..., 8, 5] = 1000.0
    k[..., 9, :32] = torch.arange(32) / 2.0
    k[..., 10, :] = -k[..., 10, :].abs() - 300
    k[..., 11, :] *= 60000.0
    k[..., 12, :32] = 65504.0
    k[..., 12, 32:] = -65504.0
    k = k.to(c.t)
    c.append(k, k.flip(2))
    c.same()
    # and within half a step, where nothing ends
    code, big, off = quantise(k[0, 0, [0, 1, 2, 3, 8, 9, 10, 13]])
    err = (stands_for(code, big, off) - k[0, 0, [0, 1, 2, 3, 8, 9, 10, 13]].double()).abs().unflatten(-1, (-1, 32))
    room = big.double() / 32 * (1 + 2.0 ** -9) + off.double().abs() * 2.0 ** -11 + 2.0 ** -20
    assert (err <= room[..., None]).all()


def test_append_stops_at_the_capacity_and_skips_bad_pages():
    c = Cache4("bf16", [22, 20, 3], 1, 64, page=8, seed=5)
    c.table = c.table[:, :3].contiguous()   # 24 rows a sequence
    c.capacity = 24
    c.table[1, 2] = 99
    c.table[2, 1] = -1
    c.upload()
    g = torch.Generator().manual_seed(6)
    c.append(*(make(g, c.t, 3, 1, 14, 64, 1.0) for _ in range(2)))
    c.same()


def test_lengths_past_the_capacity_append_nothing():
    c = Cache4("f16", [20, 5], 1, 64, seed=7)
    c.lens = [10 ** 9, 2 ** 31 - 1]
    c.upload()
    g = torch.Generator().manual_seed(8)
    c.append(*(make(g, c.t, 2, 1, 9, 64, 1.0) for _ in range(2)))
    c.same()


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("page", (0, 8, 64))
@pytest.mark.parametrize("d,layout,pad", ((64, "bhsd", 0), (128, "bshd", 8), (96, "bshd", 3)))
def test_read(dtype, page, d, layout, pad):
    c = Cache4(dtype, [50, 9, -1], 2, d, page=page, seed=9)
    rows = torch.tensor([[0, 49, 7, 7, -1, 2 ** 31 - 1, 33], [8, 0, 1, 2, 3, c.capacity, 5], [-5] * 7], dtype=torch.int32)
    grows = rows.cuda()
    outs = [filled(make(torch.Generator(), c.t, 3, 2, 7, d, 1.0, layout, pad)) for _ in range(2)]
    cfg = fa.read_config(7, strides(outs[0]), strides(outs[1]))
    for wanted in ((1, 1), (0, 1), (1, 0)):
        for x in outs:
            x.fill_(7.0)
        fa.cache4_read_device(c.cache, cfg, grows.data_ptr(), *(x.data_ptr() if w else 0 for x, w in zip(outs, wanted)), stream())
        torch.cuda.synchronize()
        for x, w, kept in zip(outs, wanted, (c.k, c.v)):
            if not w:
                assert (x == 7).all()
                continue
            for i in range(3):
                for j in range(7):
                    r = int(rows[i, j])
                    if not 0 <= r < c.capacity:
                        assert (x[i, :, j] == 0).all()
                    else:
                        want = kept[i][:, r]
                        # one f32 operation, one rounding to the type
                        assert ((x[i, :, j].double().cpu() - want).abs() <= want.abs() * (unit(c.t) + 2.0 ** -23) + 2.0 ** -25).all()


def test_read_bad_pages():
    c = Cache4("bf16", [40], 1, 64, page=8, seed=10)
    c.table[0, 1], c.table[0, 2] = -1, 1000
    c.upload()
    rows = torch.arange(8, 24, dtype=torch.int32)[None].cuda()
    out = torch.full((1, 1, 16, 64), 7.0, dtype=c.t, device="cuda")
    fa.cache4_read_device(c.cache, fa.read_config(16), rows.data_ptr(), out.data_ptr(), out.data_ptr(), stream())
    torch.cuda.synchronize()
    assert (out == 0).all()


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
class Attention(Cache4):
    def __init__(self, dtype, lens, h, hk, n, d, page=0, mask="chain", cap=0.0, alibi=False, positions=False, window=None,
                 sigma=1.0, scale=None, pad=0, seed=0, **kw):
        super().__init__(dtype, lens, hk, d, page=page, room=n, seed=seed, **kw)
        g, b = self.g, self.b
        self.n, self.h, self.cap, self.scale = n, h, cap, scale or 1 / math.sqrt(d)
        self.q = make(g, self.t, b, h, n, d, sigma, "bhsd", pad)
        new = [make(g, self.t, b, hk, n, d, 1.0) for _ in range(2)]
        self.append(*new)
        for i, x in enumerate(lens):
            for keep, y in ((self.k, new[0]), (self.v, new[1])):
                keep[i] = torch.cat((keep[i], stands_for(*quantise(y[i]))), 1)
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
        words = -(-n // 64)
        bits = torch.zeros(b, n, words * 64, dtype=torch.int64)
        bits[:, :, :n] = self.see.long()
        self.bits = sum(bits.reshape(b, n, words, 64)[..., e] << e for e in range(64)).cuda()
        self.pos = torch.tensor([[max(x, 0) + (int(self.see[i, j].sum()) - 1 if positions else j) for j in range(n)]
                                 for i, x in enumerate(lens)], dtype=torch.int32)
        self.slopes = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)]) if alibi else None
        self.keep = [self.pos.cuda(), None if self.slopes is None else self.slopes.cuda()]
        self.window = window
        self.gq = to_gpu(self.q)
        self.out = filled(self.q)
        self.lse = torch.full((b, h, n), 7.0, device="cuda")
        self.cfg = fa.tree_config(h, n, mask_ptr=0 if mask == "chain" else self.bits.data_ptr(), softcap=cap,
                                  softmax_scale=scale, slopes_ptr=self.keep[1].data_ptr() if alibi else 0,
                                  positions_ptr=self.keep[0].data_ptr() if positions else 0, q_strides=strides(self.gq),
                                  out_strides=strides(self.out))

    def run(self, lse=True):
        fa.cache4_attention_device(self.cfg, self.cache, self.gq.data_ptr(), self.out.data_ptr(),
                                   self.lse.data_ptr() if lse else 0, stream(),
                                   window=fa.window(*self.window) if self.window else None)

    def check(self, hidden=None):
        torch.cuda.synchronize()
        for i, x in enumerate(self.lens):
            if x < 0:
                assert (self.out[i] == 0).all() and (self.lse[i] == -math.inf).all()
                continue
            see = torch.cat((torch.ones(self.n, x, dtype=torch.bool), self.see[i]), dim=1)
            pos = self.pos[i].long()
            kpos = torch.cat((torch.arange(x), pos))
            if hidden is not None:
                see = see & ~hidden[i][None, :x + self.n]
            if self.window:
                size, sinks = self.window
                see = see & ((pos[:, None] - kpos[None, :] < size) | (torch.arange(x + self.n) < sinks)[None, :])
            dist = (pos[:, None] - kpos[None, :]).abs().double()
            for j in range(self.h):
                k, v = (y[i][j * self.hk // self.h].half() for y in (self.k, self.v))
                r = attend(self.q[i, j], k, v, see, self.scale, self.cap,
                           None if self.slopes is None else -self.slopes[j].double() * dist, torch.float16)
                out, e = r["out"]
                if self.t != torch.float16:
                    e = e + unit(self.t) * (out.abs() + e)
                check(f"out {i} {j}", self.out[i, j], out, e)
                check(f"lse {i} {j}", self.lse[i, j], *r["lse"])


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("n", (1, 5, 16, 33, 64, 130, 256))
@pytest.mark.parametrize("page", (0, 8, 64))
def test_attention(dtype, n, page):
    c = Attention(dtype, [500, 0, 63, 1, 200], 4, 2, n, 64, page=page, mask="tree", seed=n)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("d", (32, 64, 96, 128, 160, 192, 224, 256))
@pytest.mark.parametrize("n,page,pad", ((1, 0, 0), (3, 16, 0), (7, 32, 8), (20, 0, 3)))
def test_head_widths(dtype, d, n, page, pad):
    """Rows of q and out on 16 bytes and not."""
    c = Attention(dtype, [300, 129], 8, 2, n, d, page=page, pad=pad, seed=d)
    c.run()
    c.check()


@pytest.mark.parametrize("page", (8, 16, 32, 128))
def test_pages(page):
    c = Attention("bf16", [333, 256, 31], 4, 1, 9, 64, page=page, seed=page)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("mask", ("chain", "any", "none"))
@pytest.mark.parametrize("mods", ({}, {"cap": 5.0}, {"alibi": True}, {"alibi": True, "positions": True, "cap": 9.0},
                                  {"cap": 700.0, "sigma": 4.0}, {"scale": 0.3}))
@pytest.mark.parametrize("page", (0, 16))
def test_masks_and_scores(dtype, mask, mods, page):
    c = Attention(dtype, [300, 40, -1, 0], 4, 2, 12, 64, mask=mask, page=page, seed=3, **mods)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("page,d,n", ((0, 64, 200), (8, 64, 50), (0, 128, 130)))
@pytest.mark.parametrize("k_off,v_off", ((5.0, 50.0), (-3.0, 1000.0), (0.0, -200.0)))
def test_groups_far_from_zero(dtype, page, d, n, k_off, v_off):
    """Against what codes stand for, unrounded.

    Values of keys off by 2^-11 |k| move scores by at most t = scale sum |q| 2^-11 |k|, and weights by e^(2 t) - 1 of
    themselves; these changes cancel in the sum, so that they weigh what values differ from v_off.  Values of V are off by
    2^-11 |v|.
    """
    c = Attention(dtype, [0], 4, 2, n, d, page=page, seed=18)
    g = torch.Generator().manual_seed(19)
    k, v = ((make(g, c.t, 1, 2, n, d, 1.0).float() + x).to(c.t) for x in (k_off, v_off))
    c.append(k, v)
    c.run()
    torch.cuda.synchronize()
    k, v = (stands_for(*quantise(x[0])) for x in (k, v))
    u = unit(torch.float16)
    for j in range(4):
        q, kx, vx = c.q[0, j], k[j // 2], v[j // 2]
        out, e = attend(q, kx, vx, c.see[0], c.scale, dtype=torch.float16)["out"]
        t = c.scale * u * torch.where(c.see[0], q.double().abs() @ kx.abs().T, 0.0).amax(1, keepdim=True)
        e = e + torch.expm1(2 * t) * (vx - v_off).abs().amax() + 1.01 * u * vx.abs().amax()
        check(f"out {j}", c.out[0, j], out, e + unit(c.t) * (out.abs() + e))


@pytest.mark.parametrize("d", (64, 128, 256))
@pytest.mark.parametrize("n,h,page", ((1, 8, 0), (3, 8, 128), (40, 8, 0), (1, 1, 16)))
def test_long_cache(d, n, h, page):
    """Keys split over many workgroups; one sequence much longer than the others."""
    c = Attention("bf16", [5000, 10, 2500], h, 1, n, d, page=page, seed=4)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("size,sinks", ((1, 0), (40, 3), (200, 100), (5000, 4)))
@pytest.mark.parametrize("n,mask,page", ((1, "chain", 0), (9, "tree", 8), (24, "tree", 64)))
def test_windows(dtype, size, sinks, n, mask, page):
    c = Attention(dtype, [1500, 0, 63, -1, 200], 4, 2, n, 64, page=page, mask=mask, positions=mask == "tree",
                  window=(size, sinks), seed=5)
    c.run()
    c.check()


@pytest.mark.parametrize("page", (0, 8))
@pytest.mark.parametrize("length", (449, 480, 6000))
def test_windows_with_sinks_far_below(length, page):
    """A bias by distance leaves sinks thousands below; last and first keys anywhere in a block of 64."""
    for size, sinks in ((100, 4), (33, 70), (5, 3)):
        c = Attention("f16", [length], 8, 8, 3, 64, page=page, alibi=True, window=(size, sinks), seed=length)
        c.run()
        c.check()


@pytest.mark.parametrize("big", (1e-30, 1e-3, 1e5, 1e30))
def test_bf16_queries_of_any_size(big):
    """Brought into f16's range by powers of two, a row each."""
    c = Attention("bf16", [100], 2, 1, 4, 64, scale=0.1 / big, seed=6)
    c.q[:, :, 1] *= big
    c.q[:, :, 0], c.q[:, :, 2:] = c.q[:, :, 0] * big, c.q[:, :, 2:] * big
    c.gq.copy_(c.q)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype,big,scale", (("bf16", 1e-36, 1e-9), ("bf16", 1.0, 1e-44), ("f16", 1.0, 1e-44), ("bf16", 1e-36, 0.1)))
@pytest.mark.parametrize("length", (0, 40, 3000))
def test_scales_that_leave_nothing_of_the_scores(dtype, big, scale, length):
    """Scores of 0, also in f32: the mean of the values, and waves without a key add nothing to it."""
    c = Attention(dtype, [length], 2, 1, 4, 64, scale=scale, seed=17)
    c.q *= big
    c.gq.copy_(c.q)
    c.run()
    c.check()


def test_queries_of_zeros_and_rows_of_different_size():
    c = Attention("bf16", [100], 2, 1, 4, 64, seed=7)
    c.q[:, :, 1] = 0
    c.q[:, :, 2] *= 2.0 ** -100
    c.q[:, :, 3, :8] *= 2.0 ** -60
    c.gq.copy_(c.q)
    c.run()
    c.check()


def test_pages_far_into_the_pool():
    """The last pages of a pool whose keys and values each take more than 2^33 bytes: the same bits as in a small pool."""
    t, code = DT["bf16"]
    hk, h, d, page, n, per = 2, 8, 128, 64, 1200, 20
    g = torch.Generator().manual_seed(20)
    k, v = (torch.randn(2, hk, n, d, generator=g).to(t).cuda() for _ in range(2))
    q = torch.randn(2, h, 3, d, generator=g).to(t).cuda()
    rows = torch.arange(n, dtype=torch.int32, device="cuda")[None].repeat(2, 1)
    results = []
    for pages in (2 * per, (1 << 27) // (hk * page) + 2 * per):
        buffers = {x: torch.empty(s, dtype=torch.int32 if x in ("k", "v") else torch.float16, device="cuda")
                   for x, s in fa.cache4_shapes(pages, hk, page, d).items()}
        table = (torch.arange(2 * per, dtype=torch.int32).reshape(2, per) + pages - 2 * per).cuda()
        lens = torch.zeros(2, dtype=torch.int32, device="cuda")
        cache = fa.kv_cache4(code, 2, hk, d, *(buffers[x].data_ptr() for x in ("k", "k_scale", "v", "v_scale")),
                             lens.data_ptr(), block_table_ptr=table.data_ptr(), page_size=page, n_pages=pages, pages_per_seq=per)
        fa.cache4_append_device(cache, fa.append_config(n), k.data_ptr(), v.data_ptr(), stream())
        lens.fill_(n - 3)
        got = [torch.full_like(q, 7.0), torch.full((2, h, 3), 7.0, device="cuda"), torch.full_like(q, 7.0),
               torch.full_like(k, 7.0), torch.full_like(v, 7.0)]
        cfg = fa.tree_config(h, 3)
        fa.cache4_attention_device(cfg, cache, q.data_ptr(), got[0].data_ptr(), got[1].data_ptr(), stream())
        fa.cache4_attention_device(cfg, cache, q.data_ptr(), got[2].data_ptr(), stream=stream(), window=fa.window(300, 5))
        fa.cache4_read_device(cache, fa.read_config(n), rows.data_ptr(), got[3].data_ptr(), got[4].data_ptr(), stream())
        torch.cuda.synchronize()
        results.append(got)
        del buffers
        torch.cuda.empty_cache()
    code_k, big, off = quantise(k.cpu())
    assert ((results[0][3].double().cpu() - stands_for(code_k, big, off)).abs() <= stands_for(code_k, big, off).abs()
            * (unit(t) + 2.0 ** -23)).all()
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("page", (8, 32))
def test_bad_pages_hold_no_keys(page):
    c = Attention("bf16", [200, 150], 4, 2, 4, 64, page=page, seed=8)
    c.table[0, 3], c.table[0, 5], c.table[1, 0] = -1, 10 ** 6, c.cpu["k"].shape[0]
    c.gtable.copy_(c.table)
    hidden = [torch.zeros(300, dtype=torch.bool) for _ in range(2)]
    hidden[0][3 * page:4 * page] = hidden[0][5 * page:6 * page] = True
    hidden[1][:page] = True
    c.run()
    c.check(hidden)


def test_lengths_beyond_the_capacity():
    """A length that the cache cannot hold: all of its rows are seen, no drafted ones."""
    c = Attention("bf16", [92], 2, 1, 4, 64, spare=0, seed=9)
    assert c.capacity == 96
    c.glens.fill_(10 ** 9)
    c.see[:] = True
    c.run()
    c.check()


@pytest.mark.parametrize("n,length", ((6, 50), (3, 3000)))
def test_rows_that_are_no_numbers_reach_those_that_see_them_alone(n, length):
    c = Attention("bf16", [length], 2, 1, n, 64, mask="tree", seed=10)
    at = length + n - 2
    p, r = c.place(0, torch.tensor([at]))
    c.gpu["v_scale"][int(p), 0, int(r) // 8, 1, 0, int(r) % 8] = math.nan   # columns 32 .. 63
    c.run()
    torch.cuda.synchronize()
    hit = c.see[0, :, n - 2].nonzero().flatten().tolist()
    out, keep = c.out.clone(), c.out
    assert hit and torch.isnan(out[0, :, hit, 32:]).all() and torch.isfinite(out[0, :, hit, :32]).all()
    rest = [i for i in range(n) if i not in hit]
    c.v[0][:, at] = 0
    see = torch.cat((torch.ones(n, length, dtype=torch.bool), c.see[0]), dim=1)
    for j in range(2):
        x, e = attend(c.q[0, j], c.k[0][0].half(), c.v[0][0].half(), see, c.scale, dtype=torch.float16)["out"]
        check("rest", keep[0, j, rest], x[rest], (e + unit(c.t) * (x.abs() + e))[rest])


def test_log_sums_are_not_needed():
    c = Attention("f16", [70], 2, 1, 2, 64, seed=11)
    c.run(lse=False)
    torch.cuda.synchronize()
    assert (c.lse == 7).all()
    first = c.out.clone()
    c.run()
    c.check()
    assert torch.equal(first, c.out)


def test_captured_and_two_streams():
    """Two graphs of a step (append and attention) and eager calls do not share partial sums."""
    cases = [Attention("bf16", [3000, 900], 8, 2, 2, 128, page=32, seed=s) for s in (12, 13)]
    other, extra = torch.cuda.Stream(), Attention("bf16", [4000], 8, 2, 2, 128, seed=14)
    side, graphs = torch.cuda.Stream(), []
    torch.cuda.synchronize()
    for c in cases:
        with torch.cuda.stream(side):
            c.run()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                c.run()
            graphs.append(graph)
    for _ in range(3):
        for c in cases + [extra]:
            c.out.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            extra.run()
        with torch.cuda.stream(side):
            for graph in graphs:
                graph.replay()
        for c in cases + [extra]:
            c.check()


def test_a_layer_as_it_is_served():
    """Norms and rotary positions, rows into the cache in 4 bits, attention in a window with sinks; prompt, then steps."""
    t, code = DT["bf16"]
    g = torch.Generator().manual_seed(15)
    b, h, hk, d, s, steps, size, sinks = 2, 4, 2, 64, 150, 3, 60, 3
    w = [(1 + 0.3 * torch.randn(d, generator=g)).to(t).cuda() for _ in range(2)]
    norm, rot = fa.head_norm(w[0].data_ptr(), w[1].data_ptr(), 1e-6), fa.rotary_config(code, d, d)
    c = Cache4("bf16", [0, 0], hk, d, page=32, room=s + steps, seed=16)
    lens, window = c.glens, fa.window(size, sinks)
    keys = torch.zeros(b, hk, 0, d, dtype=torch.float64)
    f, gain = frequencies(d)
    done = 0
    for n in [s] + [1] * steps:
        q, k, v = (torch.randn(b, x, n, d, generator=g).to(t).cuda() for x in (h, hk, hk))
        pos = torch.arange(done, done + n, dtype=torch.int32)[None].repeat(b, 1)
        gp = pos.cuda()
        raw = k.cpu()
        fa.norm_rotary_device(rot, norm, b, n, gp.data_ptr(), fa.rotary_tensor(h), q.data_ptr(), q.data_ptr(),
                              fa.rotary_tensor(hk), k.data_ptr(), k.data_ptr(), stream())
        fa.cache4_append_device(c.cache, fa.append_config(n), k.data_ptr(), v.data_ptr(), stream())
        out = torch.empty_like(q)
        fa.cache4_attention_device(fa.tree_config(h, n), c.cache, q.data_ptr(), out.data_ptr(), stream=stream(),
                                   window=window)
        rows = torch.arange(done + n, dtype=torch.int32, device="cuda")[None].repeat(b, 1)
        kk, vv = (torch.empty(b, hk, done + n, d, dtype=t, device="cuda") for _ in range(2))
        fa.cache4_read_device(c.cache, fa.read_config(done + n), rows.data_ptr(), kk.data_ptr(), vv.data_ptr(), stream())
        torch.cuda.synchronize()
        # what is kept is near the normed and rotated keys: half a step of a group (range up to 2 max) and roundings
        want = rotate(normed(raw, w[1].cpu(), 1e-6), pos, f, gain, False)
        keys = torch.cat((keys, want), 2)
        top = keys.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
        assert ((kk.double().cpu().unflatten(-1, (-1, 32)) - keys.unflatten(-1, (-1, 32))).abs() <= top * (1 / 15 + 3 * 2.0 ** -8)).all()
        i, j = torch.arange(done, done + n)[:, None], torch.arange(done + n)[None, :]
        see = (j <= i) & ((i - j < size) | (j < sinks))
        for x in range(b):
            for y in range(h):
                # rows read back are rounded to bf16, those in the products to f16: errors of scores and values of
                # 2^-8 of their terms
                kx, vx = kk[x, y // 2].double().cpu(), vv[x, y // 2].double().cpu()
                o, e = attend(q[x, y].cpu(), kx, vx, see, d ** -0.5, dtype=t)["out"]
                ez = 2.0 ** -8 * (q[x, y].double().cpu().abs() @ kx.abs().T).amax(1, keepdim=True) * d ** -0.5
                e = e + (2 * ez + 2.0 ** -8) * vx.abs().amax() * 1.1
                check("out", out[x, y], o, e)
        done += n
        lens.fill_(done)


@pytest.mark.parametrize("page", (0, 8, 32))
def test_a_cache_without_rows(page):
    """No capacity, or no pages at all: nothing is seen, and nothing is read or written."""
    t, code = DT["bf16"]
    lens = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    table = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    paged = {"block_table_ptr": table.data_ptr(), "page_size": page, "n_pages": 0, "pages_per_seq": 4} if page else {}
    some = torch.full((1024,), 7.0, device="cuda")
    buffers = [some.data_ptr()] * 4 if page else [0] * 4
    cache = fa.kv_cache4(code, 2, 1, 64, *buffers, lens.data_ptr(), capacity=0, **paged)
    q = torch.randn(2, 2, 3, 64, device="cuda").to(t)
    out, lse = torch.full_like(q, 7.0), torch.full((2, 2, 3), 7.0, device="cuda")
    k = torch.ones(2, 1, 3, 64, dtype=t, device="cuda")
    fa.cache4_append_device(cache, fa.append_config(3), k.data_ptr(), k.data_ptr(), stream())
    fa.cache4_attention_device(fa.tree_config(2, 3), cache, q.data_ptr(), out.data_ptr(), lse.data_ptr(), stream())
    torch.cuda.synchronize()
    assert (out == 0).all() and (lse == -math.inf).all() and (some == 7).all()
