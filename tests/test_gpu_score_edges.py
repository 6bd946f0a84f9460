"""Score attention on the GPU where its definition allows more than training usually asks for: any sign of
the slopes, gradients of any size, caps of any size, many small calls in one.

Bounds: tests/ops_reference.py.
"""
from __future__ import annotations

import threading

import pytest
import torch

import flash_attention_amd as fa
from ops_reference import attend, check, round_bound
from test_gpu_rotary_tree import Tree
from test_gpu_score import Call, check_batch, doc_ids, to_gpu

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


def f16_gradients(c):
    """Gradients of a call in f16 and their bounds, as ops_reference.attend has them, but for the absolute part of the
    roundings of weights and score gradients.  There it is 2^-25, half a step of the smallest numbers of f16.  Weights are
    taken 2^12 larger: 2^-37.  Score gradients too, and where the largest of a kept row (a query's for dQ, a key's for
    dK) would pass 2^15 so, all of that row are brought down with it to 2^13 at least: 2^-25 times max / 2^13."""
    b, h = c.q.shape[:2]
    sums = {"dq": [], "dk": [], "dv": []}
    for i in range(b):
        rows = {n: [] for n in sums}
        for j in range(h):
            k, v, q, do = c.k[i, j // c.group], c.v[i, j // c.group], c.q[i, j].double(), c.dout[i, j].double()
            see = c.see[i].double()
            r = attend(c.q[i, j], k, v, c.see[i], c.scale, c.cap, c.bias[j], c.t, c.dout[i, j])
            x = q @ k.double().T * c.scale
            t = torch.tanh(x / c.cap) if c.cap else torch.zeros_like(x)
            z = (c.cap * t if c.cap else x) + (0 if c.bias[j] is None else c.bias[j])
            p = torch.softmax(z.masked_fill(~c.see[i], float("-inf")), 1).nan_to_num(0)
            ds = (p * (do @ v.double().T - (do * (p @ v.double())).sum(1, keepdim=True)) * (1 - t * t)).abs()
            less = {n: (2.0 ** -25 - (2.0 ** -38 * ds.amax(d, keepdim=True)).clamp_min(2.0 ** -37)) * see
                    for n, d in (("dq", 1), ("dk", 0))}
            less = {"dq": less["dq"] @ k.double().abs() * c.scale, "dk": less["dk"].T @ q.abs() * c.scale,
                    "dv": (2.0 ** -25 - 2.0 ** -37) * see.T @ do.abs()}
            for n in sums:
                x, e = r[n][0], r[n][1] - less[n]
                if n != "dq" and j % c.group:
                    rows[n][-1] = (rows[n][-1][0] + x, rows[n][-1][1] + e)
                else:
                    rows[n].append((x, e))
        for n in sums:
            sums[n].append([torch.stack([y[m] for y in rows[n]]) for m in (0, 1)])
    full = {n: [torch.stack([y[m] for y in x]) for m in (0, 1)] for n, x in sums.items()}
    return {n: (x, round_bound(x, e, c.t)) for n, (x, e) in full.items()}


def check_f16_gradients(c):
    c.gpu["dout"] = to_gpu(c.dout)
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    for n, (x, e) in f16_gradients(c).items():
        # zeros would not pass
        assert (e < x.abs()).double().mean() > 0.75, (n, (e / x.abs()).median())
        check(n, c.outs[n], x, e)
        # All values together: errors of independent roundings, each within u of its term (u / sqrt(3) on average), add
        # up as the terms do, to u / sqrt(3) of the sum; the result is rounded once more.
        off, rounded = ((y - x).norm() for y in (c.outs[n].double().cpu(), x.to(c.t).double()))
        assert off <= 2 * (rounded + 2.0 ** -11 * x.norm()), (n, off, rounded, x.norm())


@pytest.mark.parametrize("size", (1e-2, 3e-4))
@pytest.mark.parametrize("sq,sk,d,mods", ((300, 300, 64, {"causal": True}), (300, 3000, 64, {}), (3000, 300, 64, {"alibi": True}),
                                          (400, 1300, 128, {"cap": 5.0}), (150, 1000, 256, {}), (100, 1000, 36, {})))
def test_small_f16_gradients_keep_their_accuracy(size, sq, sk, d, mods):
    """Score gradients far below the normal numbers of the type, down to parts of its smallest."""
    c = Call("f16", 1, 4, 2, sq, sk, d, seed=6, **mods)
    c.dout = (c.dout.float() * size).half()
    check_f16_gradients(c)


@pytest.mark.parametrize("sq,sk,d,mods", ((6, 3, 64, {}), (6, 3, 128, {"cap": 2.0}), (70, 40, 64, {"causal": True}), (40, 70, 256, {}),
                                          (7, 5, 36, {"alibi": True})))
def test_large_f16_gradients_stay_in_range(sq, sk, d, mods):
    """Score gradients beyond the type's largest number, whose sums are not."""
    c = Call("f16", 1, 4, 2, sq, sk, d, scale=0.01, seed=7, **mods)
    c.dout = (c.dout.float() * 1e4).half()
    check_f16_gradients(c)


def test_f16_gradients_of_all_sizes_at_once():
    """Rows of dO from 1e-3 to 1e3: each query's gradient has its own range, each key's that of its largest."""
    c = Call("f16", 2, 16, 4, 500, 500, 64, causal=True, seed=8)
    g = torch.Generator().manual_seed(9)
    size = 10.0 ** (6 * torch.rand(2, 16, 500, 1, generator=g) - 3)
    c.dout = (c.dout.float() * size).half()
    check_f16_gradients(c)


def test_many_blocks_of_small_f16_gradients():
    """Two tiles a wave."""
    c = Call("f16", 8, 16, 4, 500, 500, 64, seed=10)
    c.dout = (c.dout.float() * 1e-3).half()
    c.gpu["dout"] = to_gpu(c.dout)
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    one = Call.__new__(Call)
    one.__dict__.update(c.__dict__)
    for n in ("q", "k", "v", "dout"):
        setattr(one, n, getattr(c, n)[7:])
    one.see = c.see[7:]
    for n, (x, e) in f16_gradients(one).items():
        check(n, c.outs[n][7:], x, e)


def check_cap(c, grads=True):
    """Against the capped definition, with the bounds of uncapped scores and a quarter: scores of at most 8 differ from
    capped ones by x^3 / (3 cap^2), which changes those bounds by less than 1e-3 of them, and the rounding of the tanh adds
    8 2^-24 |x| to the error of a score, a quarter of that of its dot product at most."""
    want, cap = c.expect(grads), c.cap
    bounds = want
    if cap > 512:   # below, 16-bit types take the short tanh: ops_reference has its error, 4e-7 of the cap
        c.cap = 0.0
        bounds = c.expect(grads)
        c.cap = cap
    for n, (x, _) in want.items():
        check(n, c.lse if n == "lse" else c.outs[n], x, 1.25 * bounds[n][1])


CAPS = (500.0, 520.0, 1e4, 1e6, 1e12, 1e30)


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("d,alibi", ((64, False), (128, True), (36, False)))
def test_large_caps(dtype, cap, d, alibi):
    c = Call(dtype, 1, 4, 2, 140, 140, d, causal=True, cap=cap, alibi=alibi, seed=11)
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    check_cap(c)


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("cap", CAPS)
def test_large_caps_over_long_ranges(dtype, cap):
    c = Call(dtype, 1, 8, 2, 3, 900, 64, causal=True, q_start=880, cap=cap, seed=12)
    c.forward()
    torch.cuda.synchronize()
    check_cap(c, grads=False)
    # a tree's check has the capped bound, which allows 4e-7 of the cap: against the same call without a cap instead
    results = []
    for x in (cap, 0.0):
        t = Tree(dtype, [700, 60], 4, 2, 7, 64, page=16, cap=x, seed=13)
        t.run()
        results.append(t)
    torch.cuda.synchronize()
    if cap < 1e4:   # capped scores differ
        results[0].check()
        return
    results[1].out, results[1].lse = results[0].out, results[0].lse
    results[1].check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
def test_tiny_caps(dtype):
    """All scores are within the cap: every visible key weighs the same."""
    c = Call(dtype, 1, 2, 1, 70, 70, 64, causal=True, cap=1e-30, seed=14)
    c.forward()
    torch.cuda.synchronize()
    v = c.v.double().repeat_interleave(2, 1)
    want = v.cumsum(2) / torch.arange(1, 71)[:, None]
    u = torch.finfo(c.t).eps / 2
    check("out", c.outs["out"], want, 2 * u * (v.abs().cumsum(2) / torch.arange(1, 71)[:, None]) + 70 * 2.0 ** -24 + 2.0 ** -25)


@pytest.mark.parametrize("batch,sq,sk,d", ((131073, 64, 20, 8), (300007, 49, 49, 32), (600011, 1, 5, 64)))
def test_very_many_small_calls_in_one(batch, sq, sk, d):
    """More than 2^23 query rows in short blocks, all on the same keys: each weight and the result are rounded once, 2 u of
    the largest value, and f32 errors are far below a quarter of that."""
    g = torch.Generator(device="cuda").manual_seed(15)
    q = torch.randn(batch, 1, sq, d, generator=g, device="cuda").bfloat16()
    k, v = (torch.randn(sk, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    out, lse = torch.full_like(q, 7.0), torch.full((batch, 1, sq), 7.0, device="cuda")
    c = fa.score_config(fa.DTYPE_BF16, batch, 1, 1, sq, sk, d, strides={"k": (0, d, 0), "v": (0, d, 0)})
    fa.score_attention_device(c, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
                              torch.cuda.current_stream().cuda_stream)
    kt, vd = k.double().t().contiguous(), v.double()
    for lo in range(0, batch, 40000):
        z = q[lo:lo + 40000].reshape(-1, d).double() @ kt / d ** 0.5
        want = torch.softmax(z, 1) @ vd
        assert (out[lo:lo + 40000].reshape(-1, d) - want).abs().max() <= 2.25 * 2.0 ** -8 * vd.abs().max()
        assert (lse[lo:lo + 40000].reshape(-1) - torch.logsumexp(z, 1)).abs().max() <= 1e-4


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("b,h,hk,sq,sk,d", ((2, 8, 2, 300, 300, 128), (1, 8, 2, 3, 3000, 64), (2, 4, 4, 130, 150, 36), (8, 16, 4, 500, 500, 64)))
def test_same_bits_every_time(dtype, b, h, hk, sq, sk, d):
    """Forward and backward, whatever order the workgroups run in."""
    c = Call(dtype, b, h, hk, sq, sk, d, causal=True, q_start=sk - sq, alibi=True, seed=16)
    first = None
    for _ in range(4):
        for x in (*c.outs.values(), c.lse):
            x.fill_(7.0)
        c.forward()
        c.backward()
        torch.cuda.synchronize()
        now = [x.clone() for x in (*c.outs.values(), c.lse)]
        first = first or now
        assert all(torch.equal(x, y) for x, y in zip(now, first))
