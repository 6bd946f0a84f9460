"""Attention with modified scores on the GPU against its definition in float64.

Bounds: tests/ops_reference.py.  Every type, head layout and mask, forward and
backward, with lengths that fill no tile, rows that see no key, infinities and
NaN where nothing may look, and outputs whose surroundings stay as they were.
"""
from __future__ import annotations

import math

import pytest
import torch

import flash_attention_amd as fa
from ops_reference import attend, check, round_bound, visible

pytestmark = pytest.mark.gpu

DT = {"f32": (torch.float32, fa.DTYPE_F32), "bf16": (torch.bfloat16, fa.DTYPE_BF16),
      "f16": (torch.float16, fa.DTYPE_F16)}


def strides(x):
    return (x.stride(0), x.stride(2), x.stride(1))


def make(gen, dtype, b, h, s, d, sigma=1.0, layout="bhsd", pad=0):
    """[b, h, s, d] view; layout: the order in memory; pad: columns between rows."""
    shape = (b, h, s, d + pad) if layout == "bhsd" else (b, s, h, d + pad)
    x = (torch.randn(shape, generator=gen) * sigma).to(dtype)
    x = x if layout == "bhsd" else x.transpose(1, 2)
    return x[..., :d]


def to_gpu(x):
    """The same view of a copy of the whole storage."""
    base = torch.empty(0, dtype=x.dtype).set_(x.untyped_storage())
    return torch.as_strided(base.cuda(), x.shape, x.stride(), x.storage_offset())


def filled(x):
    """The same view of a storage full of sevens, on the GPU."""
    n = x.untyped_storage().nbytes() // x.element_size()
    return torch.as_strided(torch.full((n,), 7.0, dtype=x.dtype, device="cuda"), x.shape, x.stride(), x.storage_offset())


class Call:
    """One call's tensors on the CPU and the GPU, its config, and the expectation."""

    def __init__(self, dtype, b, h, hk, sq, sk, d, causal=False, cap=0.0, alibi=False, q_start=0, prefix=None,
                 q_doc=None, k_doc=None, sigma=1.0, layout="bhsd", pad=0, scale=None, seed=0):
        self.t, code = DT[dtype]
        g = torch.Generator().manual_seed(seed)
        self.q, self.k, self.v = (make(g, self.t, b, n, s, d, w, layout, pad)
                                  for n, s, w in ((h, sq, sigma), (hk, sk, sigma), (hk, sk, 1.0)))
        self.dout = make(g, self.t, b, h, sq, d, 1.0, layout, pad)
        self.scale = scale or 1.0 / math.sqrt(d)
        self.cap, self.group = cap, h // hk
        self.slopes = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)]) if alibi else None
        dist = (torch.arange(sq)[:, None] + q_start - torch.arange(sk)[None, :]).abs().double()
        self.bias = [-self.slopes[i].double() * dist for i in range(h)] if alibi else [None] * h
        self.see = [visible(sq, sk, causal, q_start, prefix[i] if prefix else None, q_doc[i] if q_doc is not None else None,
                            k_doc[i] if k_doc is not None else None) for i in range(b)]
        ints = [None if x is None else torch.as_tensor(x, dtype=torch.int32).cuda() for x in (prefix, q_doc, k_doc)]
        self.keep = ints + [None if self.slopes is None else self.slopes.cuda()]
        p = [0 if x is None else x.data_ptr() for x in self.keep]
        self.gpu = {n: to_gpu(getattr(self, n)) for n in ("q", "k", "v", "dout")}
        st = {n: strides(x) for n, x in self.gpu.items()}
        self.outs = {}
        for n, like in (("out", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v")):
            self.outs[n] = filled(getattr(self, like))
            st[n] = strides(self.outs[n])
        self.lse = torch.full((b, h, sq), 7.0, device="cuda")
        self.cfg = fa.score_config(code, b, h, hk, sq, sk, d, causal=causal, softmax_scale=scale, softcap=cap,
                                   q_start=q_start, slopes_ptr=p[3], q_doc_ptr=p[1], k_doc_ptr=p[2], prefix_ptr=p[0],
                                   strides=st)

    def forward(self, lse=True):
        fa.score_attention_device(self.cfg, *(self.gpu[n].data_ptr() for n in ("q", "k", "v")),
                                  self.outs["out"].data_ptr(), self.lse.data_ptr() if lse else 0,
                                  torch.cuda.current_stream().cuda_stream)

    def backward(self, dq=True, dk=True, dv=True):
        o = self.outs
        fa.score_attention_backward_device(
            self.cfg, *(self.gpu[n].data_ptr() for n in ("q", "k", "v")), o["out"].data_ptr(), self.lse.data_ptr(),
            self.gpu["dout"].data_ptr(), *(o[n].data_ptr() if w else 0 for n, w in (("dq", dq), ("dk", dk), ("dv", dv))),
            torch.cuda.current_stream().cuda_stream)

    def expect(self, grads=True):
        b, h = self.q.shape[:2]
        res = {n: ([], []) for n in ("out", "lse", "dq", "dk", "dv")}
        for i in range(b):
            rows = {n: ([], []) for n in res}
            for j in range(h):
                r = attend(self.q[i, j], self.k[i, j // self.group], self.v[i, j // self.group], self.see[i], self.scale,
                           self.cap, self.bias[j], self.t, self.dout[i, j] if grads else None)
                for n, (x, e) in r.items():
                    if n in ("dk", "dv") and j % self.group:
                        rows[n][0][-1] = rows[n][0][-1] + x
                        rows[n][1][-1] = rows[n][1][-1] + e
                    else:
                        rows[n][0].append(x)
                        rows[n][1].append(e)
            for n in res:
                if rows[n][0]:
                    res[n][0].append(torch.stack(rows[n][0]))
                    res[n][1].append(torch.stack(rows[n][1]))
        full = {n: (torch.stack(x), torch.stack(e)) for n, (x, e) in res.items() if x}
        for n in ("dq", "dk", "dv"):
            if n in full:
                full[n] = (full[n][0], round_bound(*full[n], self.t))
        return full

    def run_and_check(self, grads=True):
        self.forward()
        if grads:
            self.backward()
        torch.cuda.synchronize()
        for n, (x, e) in self.expect(grads).items():
            check(n, self.lse if n == "lse" else self.outs[n], x, e)


def doc_ids(b, s, lengths, pad=0):
    rows = []
    for i in range(b):
        ids = []
        for n, length in enumerate(lengths[i % len(lengths)]):
            ids += [n] * length
        ids = (ids + [len(lengths[i % len(lengths)])] * s)[:s]
        if pad:
            ids[s - pad:] = [-1] * pad
        rows.append(ids)
    return torch.tensor(rows, dtype=torch.int32)


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("d", (8, 40, 64, 100, 128, 200, 256))
def test_causal_every_head_width(dtype, d):
    Call(dtype, 1, 2, 1, 150, 150, d, causal=True, seed=d).run_and_check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("sq,sk", ((1, 1), (1, 300), (129, 1), (127, 65), (260, 200), (65, 333)))
@pytest.mark.parametrize("causal", (False, True))
def test_lengths(dtype, sq, sk, causal):
    Call(dtype, 2, 2, 2, sq, sk, 64, causal=causal, seed=sq + sk).run_and_check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("h,hk", ((4, 1), (6, 3), (8, 8), (16, 8)))
def test_grouped_heads_and_layouts(dtype, h, hk):
    for layout, pad in (("bhsd", 0), ("bshd", 0), ("bshd", 8), ("bhsd", 3)):
        Call(dtype, 2, h, hk, 90, 90, 64, causal=True, layout=layout, pad=pad, seed=h).run_and_check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("cap", (1.0, 30.0))
@pytest.mark.parametrize("d", (64, 128, 256))
def test_softcap(dtype, cap, d):
    Call(dtype, 1, 2, 1, 140, 140, d, causal=True, cap=cap, sigma=3.0, seed=3).run_and_check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("causal", (False, True))
@pytest.mark.parametrize("cap", (0.0, 20.0))
def test_distance_bias(dtype, causal, cap):
    Call(dtype, 1, 4, 2, 140, 170, 64, causal=causal, alibi=True, cap=cap, q_start=20, seed=4).run_and_check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("causal", (False, True))
def test_documents(dtype, causal):
    ids = doc_ids(2, 330, ([10, 1, 63, 128, 64], [300]), pad=9)
    Call(dtype, 2, 2, 1, 330, 330, 64, causal=causal, q_doc=ids, k_doc=ids, seed=5).run_and_check()


@pytest.mark.parametrize("causal", (False, True))
def test_documents_in_any_order(causal):
    """Ids that come back, queries of documents without keys, other ids for queries and keys."""
    g = torch.Generator().manual_seed(6)
    qd = torch.randint(-1, 4, (2, 200), generator=g, dtype=torch.int32)
    kd = torch.randint(-1, 3, (2, 150), generator=g, dtype=torch.int32)
    Call("bf16", 2, 2, 1, 200, 150, 64, causal=causal, q_doc=qd, k_doc=kd, seed=6).run_and_check()
    Call("f32", 2, 2, 1, 200, 150, 64, causal=causal, cap=5.0, q_doc=qd, k_doc=kd, seed=6).run_and_check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("prefix", ((0, 1), (64, 130), (1000, -5)))
def test_prefix(dtype, prefix):
    Call(dtype, 2, 2, 1, 180, 180, 64, causal=True, prefix=list(prefix), seed=7).run_and_check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("q_start", (-70, -1, 50, 400))
def test_query_position(dtype, q_start):
    """Negative positions see nothing (rows of zeros), far ones everything."""
    Call(dtype, 1, 2, 1, 140, 190, 64, causal=True, q_start=q_start, seed=8).run_and_check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
def test_scale_and_peaked_rows(dtype):
    Call(dtype, 1, 2, 1, 140, 140, 64, causal=True, scale=0.31, sigma=3.0, seed=9).run_and_check()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("sk", (700, 2000))
@pytest.mark.parametrize("sq", (1, 3, 17))
@pytest.mark.parametrize("mods", ({}, {"cap": 20.0}, {"alibi": True}, {"prefix": [900, 1500]}))
def test_short_query_blocks(dtype, sk, sq, mods):
    """Decode steps: keys split over workgroups and waves, partial sums joined."""
    Call(dtype, 2, 8, 2, sq, sk, 128, causal=True, q_start=sk - sq, seed=10, **mods).run_and_check(grads=False)


@pytest.mark.parametrize("dtype,d", (("bf16", 256), ("f16", 96), ("f32", 256), ("f32", 40), ("bf16", 20)))
def test_short_query_blocks_of_other_widths(dtype, d):
    Call(dtype, 1, 8, 1, 5, 1100, d, causal=True, q_start=600, seed=11).run_and_check(grads=False)
    Call(dtype, 1, 2, 1, 130, 1100, d, cap=9.0, seed=11).run_and_check(grads=False)


def test_short_query_blocks_with_documents():
    kd = doc_ids(2, 900, ([200, 300, 400],))
    qd = torch.tensor([[1, 1, 2, -1], [5, 0, 0, 2]], dtype=torch.int32)
    Call("bf16", 2, 4, 2, 4, 900, 64, q_doc=qd, k_doc=kd, seed=12).run_and_check(grads=False)


def test_no_keys():
    c = Call("bf16", 1, 2, 1, 40, 0, 64, seed=1)
    c.forward()
    torch.cuda.synchronize()
    assert (c.outs["out"] == 0).all() and (c.lse == -math.inf).all()
    c.backward()
    torch.cuda.synchronize()
    assert (c.outs["dq"] == 0).all()


def test_no_queries():
    c = Call("bf16", 1, 2, 1, 0, 40, 64, seed=1)
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    assert (c.outs["dk"] == 0).all() and (c.outs["dv"] == 0).all()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("what", ("k", "v"))
@pytest.mark.parametrize("value", (math.nan, math.inf, -math.inf))
@pytest.mark.parametrize("sq", (150, 10))
def test_hidden_infinities_do_not_reach_a_row(dtype, what, value, sq):
    """One key's row holds the value: causal rows before it come out as if it were not there."""
    at = 60 if sq > 60 else 5
    c = Call(dtype, 1, 2, 1, sq, sq, 64, causal=True, seed=13)
    x = c.expect()
    getattr(c, what)[0, 0, at] = value
    c.gpu[what] = to_gpu(getattr(c, what))
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    check("out", c.outs["out"][:, :, :at], x["out"][0][:, :, :at], x["out"][1][:, :, :at])
    check("lse", c.lse[:, :, :at], x["lse"][0][:, :, :at], x["lse"][1][:, :, :at])
    check("dq", c.outs["dq"][:, :, :at], x["dq"][0][:, :, :at], x["dq"][1][:, :, :at])
    if what == "v":
        assert not torch.isfinite(c.outs["out"][:, :, at:]).any()
        if math.isinf(value):
            assert (c.outs["out"][:, :, at:] == value).all()


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("sq", (300, 16))
def test_padding_may_hold_anything(dtype, sq):
    """Tokens of negative documents: NaN in all of their rows, and nothing else notices."""
    ids = doc_ids(1, sq, ([sq // 3],), pad=sq // 4)
    real = sq - sq // 4
    c = Call(dtype, 1, 2, 1, sq, sq, 64, causal=True, q_doc=ids, k_doc=ids, seed=14)
    x = c.expect()
    for n in ("q", "k", "v", "dout"):
        getattr(c, n)[:, :, real:] = math.nan
        c.gpu[n] = to_gpu(getattr(c, n))
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    for n in ("out", "dq", "dk", "dv"):
        check(n, c.outs[n][:, :, :real], x[n][0][:, :, :real], x[n][1][:, :, :real])
        assert (c.outs[n][:, :, real:] == 0).all(), n
    assert (c.lse[:, :, real:] == -math.inf).all()


def test_infinite_gradients_stay_in_their_rows():
    """An infinite dO row reaches the keys that its query sees, no others."""
    c = Call("bf16", 1, 2, 1, 150, 150, 64, causal=True, seed=15)
    x = c.expect()
    c.dout[0, 0, 70] = math.inf
    c.gpu["dout"] = to_gpu(c.dout)
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    for n in ("dk", "dv"):
        check(n, c.outs[n][:, :, 71:], x[n][0][:, :, 71:], x[n][1][:, :, 71:])
    assert not torch.isfinite(c.outs["dv"][0, 0, :71]).any()
    check("dq", c.outs["dq"][:, :, :70], x["dq"][0][:, :, :70], x["dq"][1][:, :, :70])


def test_surroundings_stay_as_they_were():
    """Padding columns, and tokens of a longer buffer, keep their values."""
    c = Call("bf16", 1, 2, 1, 100, 100, 64, causal=True, layout="bshd", pad=8, seed=16)
    whole = {n: torch.empty(0, dtype=x.dtype, device="cuda").set_(x.untyped_storage()).view(-1, 72)
             for n, x in c.outs.items()}
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    for n, w in whole.items():
        assert (w[:, 64:] == 7.0).all(), n


def test_same_bits_every_time_and_one_gradient_at_a_time():
    c = Call("bf16", 2, 8, 2, 300, 300, 128, causal=True, cap=20.0, seed=17)
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    first = {n: x.clone() for n, x in c.outs.items()}
    for only in ("dq", "dk", "dv"):
        for n in ("dq", "dk", "dv"):
            c.outs[n].fill_(7.0)
        c.forward(lse=True)
        c.backward(**{n: n == only for n in ("dq", "dk", "dv")})
        torch.cuda.synchronize()
        for n in ("out", "dq", "dk", "dv"):
            if n in ("out", only):
                assert torch.equal(c.outs[n], first[n]), (only, n)
            else:
                assert (c.outs[n] == 7.0).all(), (only, n)


def test_without_lse_and_misaligned_pointers():
    c = Call("bf16", 1, 2, 1, 130, 130, 64, causal=True, seed=18)
    c.forward(lse=False)
    torch.cuda.synchronize()
    assert (c.lse == 7.0).all()
    x = c.expect(grads=False)
    check("out", c.outs["out"], *x["out"])
    for n in ("q", "k", "v"):   # one element off: no vector access is aligned
        t = c.gpu[n]
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        buf[1:] = t.reshape(-1)
        c.gpu[n] = buf[1:].view(t.shape)
    out = torch.empty(c.outs["out"].numel() + 1, dtype=torch.bfloat16, device="cuda")
    c.outs["out"] = out[1:].view(c.outs["out"].shape)
    c.forward()
    torch.cuda.synchronize()
    check("out", c.outs["out"], *x["out"])


def test_gradients_against_differences():
    """Directional derivatives of sum(dO . O) by central differences of the float32 forward pass."""
    c = Call("f32", 1, 2, 1, 70, 70, 32, causal=True, cap=3.0, alibi=True, seed=19)
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    g = torch.Generator().manual_seed(20)
    for n in ("q", "k", "v"):
        step = torch.randn(getattr(c, n).shape, generator=g).double()
        step = step / step.norm()
        want = (c.outs["d" + n].double().cpu() * step).sum().item()
        base, vals, h = getattr(c, n), [], 1e-4
        for sign in (1.0, -1.0):
            # the definition in float64: forward differences of the float32 kernel would drown in rounding
            moved = Call.__new__(Call)
            moved.__dict__.update(c.__dict__)
            setattr(moved, n, base.double() + sign * h * step)
            out = moved.expect(grads=False)["out"][0]
            vals.append((out * c.dout.double()).sum().item())
        got = (vals[0] - vals[1]) / (2 * h)
        # third-order term of the difference ~ h^2, float32 gradients ~ 1e-6 of their norm
        assert abs(got - want) <= 1e-5 * max(1.0, c.outs["d" + n].double().norm().item()), (n, got, want)


def test_long_rows_against_float64():
    """Sums over 5000 keys, documents and capped scores, one head."""
    ids = doc_ids(1, 5000, ([1700, 900, 2400],))
    c = Call("bf16", 1, 1, 1, 5000, 5000, 64, causal=True, cap=30.0, q_doc=ids, k_doc=ids, sigma=2.0, seed=21)
    c.run_and_check()


def test_captured_graph_replays():
    """Forward and backward in one graph, replayed on new inputs with eager work between."""
    c = Call("bf16", 2, 4, 2, 200, 200, 64, causal=True, cap=10.0,
             q_doc=doc_ids(2, 200, ([70, 90],)), k_doc=doc_ids(2, 200, ([70, 90],)), seed=22)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c.forward()
        c.backward()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        c.forward()
        c.backward()
    other = Call("bf16", 1, 4, 2, 333, 333, 64, causal=True, seed=23)
    for turn in range(3):
        for n in ("q", "k", "v", "dout"):
            c.gpu[n].copy_(torch.randn(c.gpu[n].shape, device="cuda"))
        for x in c.outs.values():
            x.fill_(7.0)
        graph.replay()
        with torch.cuda.stream(side):   # eager calls on the capture's stream in between
            other.forward()
            other.backward()
        torch.cuda.synchronize()
        replayed = {n: x.clone() for n, x in c.outs.items()}
        c.forward()
        c.backward()
        torch.cuda.synchronize()
        for n, x in c.outs.items():
            assert torch.equal(x, replayed[n]), (turn, n)


def test_two_streams_at_once():
    a = Call("bf16", 1, 4, 2, 300, 300, 64, causal=True, seed=24)
    b = Call("bf16", 1, 4, 2, 1, 3000, 128, causal=True, q_start=2999, seed=25)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, c in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                c.forward()
                if c is a:
                    c.backward()
    torch.cuda.synchronize()
    for c, grads in ((a, True), (b, False)):
        for n, (x, e) in c.expect(grads).items():
            check(n, c.lse if n == "lse" else c.outs[n], x, e)


def check_batch(c, i, grads=True):
    """One batch entry of a larger call."""
    one = Call.__new__(Call)
    one.__dict__.update(c.__dict__)
    for n in ("q", "k", "v", "dout"):
        setattr(one, n, getattr(c, n)[i:i + 1])
    one.see = c.see[i:i + 1]
    for n, (x, e) in one.expect(grads).items():
        check(n, (c.lse if n == "lse" else c.outs[n])[i:i + 1], x, e)


@pytest.mark.parametrize("dtype,d", (("bf16", 64), ("f16", 64), ("bf16", 128), ("f16", 128)))
@pytest.mark.parametrize("mods", ({}, {"cap": 20.0}, {"alibi": True}, {"cap": 20.0, "alibi": True}))
def test_many_blocks(dtype, d, mods):
    """Workgroups enough for two tiles a wave, and gradients whose group is not split."""
    c = Call(dtype, 8, 16, 4, 500, 500, d, causal=d == 64, seed=26, **mods)
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    check_batch(c, 7)


@pytest.mark.parametrize("causal", (False, True))
@pytest.mark.parametrize("sq,sk", ((770, 770), (770, 500), (400, 1100)))
def test_many_blocks_of_documents(causal, sq, sk):
    """More blocks than run at once: they go in the order of their lengths.  Every entry has documents of its own."""
    lengths = ([300, 20, 450], [5, 700], [64, 64, 128, 192, 322], [sk])
    ids = [doc_ids(4, n, lengths, pad=n // 9) for n in (sq, sk)]
    c = Call("bf16", 4, 16, 8, sq, sk, 64, causal=causal, q_doc=ids[0], k_doc=ids[1], seed=27)
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    for i in range(4):
        check_batch(c, i)


def test_more_blocks_of_documents_than_are_ordered():
    """1100 blocks of 128 queries: the tables of their order hold 1024."""
    ids = doc_ids(220, 640, ([100, 300, 90, 150], [640], [7, 600]))
    c = Call("bf16", 220, 2, 1, 640, 640, 64, causal=True, q_doc=ids, k_doc=ids, seed=28)
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    for i in (0, 1, 219):
        check_batch(c, i)


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("h,hk,sq", ((4, 1, 70), (4, 4, 90), (2, 1, 40)))
@pytest.mark.parametrize("mods", ({}, {"cap": 20.0, "alibi": True}))
def test_blocks_of_rows_that_share_a_long_range(dtype, h, hk, sq, mods):
    """Few workgroups of queries over many keys: the keys are split, one block of rows or several."""
    Call(dtype, 1, h, hk, sq, 2500, 64, causal=True, q_start=2430, seed=29, **mods).run_and_check(grads=False)


def test_small_gradients_in_f16():
    """dO of 1e-4: products with weights below the normal numbers of the type."""
    c = Call("f16", 1, 2, 1, 300, 300, 64, causal=True, seed=30)
    c.dout = (c.dout.float() * 1e-4).half()
    c.gpu["dout"] = to_gpu(c.dout)
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    tiny = 2.0 ** -24   # half a step of the numbers below 2^-14, times 2 for the two factors of a product
    x = c.expect()
    for n in ("dq", "dk", "dv"):
        # each of up to 300 products carries a rounding of its weight's gradient (dS), up to `tiny` / 2 absolutely,
        # against an operand below 4.5 times the scale, once for each of the group's two heads
        slack = 300 * 2 * tiny * 4.5 * (c.scale if n != "dv" else 1e-4)
        check(n, c.outs[n], x[n][0], x[n][1] + slack)


def test_two_graphs_and_eager_calls_at_once():
    """Two captured steps replay on streams of their own while an eager one runs: each has its own workspace."""
    ids = doc_ids(4, 600, ([200, 400], [500, 90]))
    cases = [Call("bf16", 4, 16, 4, 600, 600, 64, causal=True, q_doc=ids, k_doc=ids, seed=s) for s in (31, 32, 33)]
    side, graphs = torch.cuda.Stream(), []
    for c in cases[:2]:
        with torch.cuda.stream(side):
            c.forward()
            c.backward()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            c.forward()
            c.backward()
        graphs.append(graph)
    first = None
    for _ in range(3):
        for c in cases:
            for x in c.outs.values():
                x.fill_(7.0)
        torch.cuda.synchronize()
        for stream, graph in zip((side, torch.cuda.Stream()), graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        cases[2].forward()
        cases[2].backward()
        torch.cuda.synchronize()
        if first is None:
            first = [{n: x.clone() for n, x in c.outs.items()} for c in cases]
            for c in cases:
                check_batch(c, 3)
        for c, f in zip(cases, first):
            for n, x in c.outs.items():
                assert torch.equal(x, f[n]), n


@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
def test_wide_blocks_of_rows_that_share_a_range(dtype):
    """256 columns: keys are split from 1024 on; the gradients take the forward pass's lse."""
    Call(dtype, 1, 2, 2, 150, 1100, 256, causal=True, q_start=950, seed=34).run_and_check()
