"""Sliding windows, norms of queries and keys, a cache in 4 bits: timed cases.

Each case is one pass through one of these operators as a training or serving
program makes it, with tensors on the GPU and on torch's current stream:

  window        softmax attention in a sliding window with a few first keys that stay visible (sinks)
  window_train  its forward and backward pass: output and the gradients of Q, K, V
  window_cache  new tokens of a batch of sequences in such a window over a key / value cache
  norm          queries and keys of a layer: norm of each head, then rotary positions
  norm_train    its forward and backward pass: gradients of Q, K and of the norms' weights
  norm_append   the same for new tokens, keys and values written to the cache
  c4_attention  new tokens of a batch of sequences over a cache held in 4 bits
  c4_fill       keys and values into such a cache, and these rows read back

``own`` chooses between the package's kernels and a plain form out of
elementary torch operations in 32 bits.  ``exact`` is the definition in 64
bits, written apart from both.

Inputs are N(0, 1) (keys, queries and weights as said at the cases).  Cache
lengths come from the case, so that its work is known; the values and page
tables from the seed.
"""
from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_EPS = 1e-6      # of the norms
_BASE = 10000.0  # of the rotary angles


def _fa():
    p = os.path.join(_ROOT, "flash-attention-cpu_amd")
    if p not in sys.path:
        sys.path.insert(0, p)
    import flash_attention_amd
    return flash_attention_amd


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _case(kind, dtype, batch, heads, kv_heads, d, name=None, **more):
    c = {"kind": kind, "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "d": d, **more}
    if name is not None:
        c["name"] = name
    return c


def _window(kind, dtype, batch, heads, kv_heads, sq, sk, d, size, sinks, name=None, causal=True, softcap=0.0,
            alibi=False, layout="bhsd"):
    return _case(kind, dtype, batch, heads, kv_heads, d, name, sq=sq, sk=sk, size=size, sinks=sinks, causal=causal,
                 softcap=softcap, alibi=alibi, layout=layout)


def _norm(kind, dtype, batch, heads, kv_heads, seq, d, rot, name=None, interleaved=False, layout="bshd", start=0):
    return _case(kind, dtype, batch, heads, kv_heads, d, name, seq=seq, rot=rot, interleaved=interleaved,
                 layout=layout, start=start)


def _cached(kind, dtype, batch, heads, kv_heads, n, length, d, name=None, page=0, size=0, sinks=0, softcap=0.0,
            tree=False, rot=0):
    return _case(kind, dtype, batch, heads, kv_heads, d, name, n=n, length=length, page=page, size=size, sinks=sinks,
                 softcap=softcap, tree=tree, rot=rot)


def listed():
    return [
        # prefill of a local layer, grouped heads, a few sinks
        _window("window", "bf16", 1, 32, 8, 8192, 8192, 128, 1024, 4, "window_layer"),
        # training of a local layer, heads next to each other in memory: the largest call
        _window("window_train", "bf16", 2, 16, 4, 4096, 4096, 128, 512, 64, "window_train", layout="bshd"),
        # training of a local encoder in f32: both sides, short ragged rows
        _window("window_train", "f32", 2, 8, 8, 777, 777, 64, 100, 0, "window_both_f32", causal=False),
        # decode steps of a batch of long contexts in pages
        _cached("window_cache", "bf16", 16, 32, 8, 1, 32768, 128, "window_decode", page=64, size=4096, sinks=4),
        # queries and keys of a layer's prefill
        _norm("norm", "bf16", 1, 32, 8, 8192, 128, 128, "norm_layer"),
        # and in training
        _norm("norm_train", "bf16", 2, 16, 4, 4096, 128, 128, "norm_train"),
        # training in f32: interleaved pairs, half of the head
        _norm("norm_train", "f32", 2, 16, 16, 1000, 80, 40, "norm_half_f32", interleaved=True, layout="bhsd"),
        # one new token a sequence, into a paged cache: a unit of latency
        _cached("norm_append", "f16", 32, 16, 2, 1, 500, 128, "norm_step", page=16, rot=128),
        # decode steps of a batch of long contexts
        _cached("c4_attention", "bf16", 8, 32, 8, 1, 32768, 128, "c4_decode"),
        # a drafted tree over short contexts in pages, capped scores
        _cached("c4_attention", "f16", 4, 16, 2, 25, 3000, 128, "c4_tree", page=16, softcap=50.0, tree=True),
        # one sequence, narrow heads, a window with sinks
        _cached("c4_attention", "bf16", 1, 8, 8, 4, 20000, 64, "c4_window", size=2000, sinks=4),
        # prompts into the cache, and back out of it
        _cached("c4_fill", "bf16", 4, 32, 8, 2048, 1000, 128, "c4_fill", page=64),
    ]


def _log_int(rng, lo, hi):
    """A whole number spread over the logarithm of lo .. hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = [work(c) for c in listed()]
    flops, moved = max(w["flops"] for w in most), max(w["bytes"] for w in most)
    while True:
        kind = rng.choice(("window", "window", "window_train", "window_train", "window_cache", "norm", "norm_train",
                           "norm_append", "c4_attention", "c4_attention", "c4_fill"))
        dtype = rng.choice(("bf16", "f16") if kind.startswith("c4") else ("bf16", "bf16", "f16", "f32"))
        d = rng.choice((64, 128, 128, 96, 256) if kind.startswith("c4") else (64, 64, 128, 128, 80, 96, 256))
        kv = rng.choice((1, 2, 4, 8))
        heads = kv * rng.choice((1, 2, 4, 8))
        batch = rng.choice((1, 1, 2, 3, 8))
        cap = rng.choice((0.0, 0.0, 30.0, 50.0))
        size, sinks = _log_int(rng, 16, 8192), rng.choice((0, 1, 4, 16, 100))
        if kind in ("window", "window_train"):
            s = _log_int(rng, 100, 16384 if kind == "window" else 8192)
            chunk = kind == "window" and rng.random() < 0.3   # a prompt's later part against all of its keys
            c = _window(kind, dtype, batch, heads, kv, _log_int(rng, 1, s) if chunk else s, s, d, size, sinks,
                        causal=chunk or rng.random() < 0.8, softcap=cap, alibi=cap == 0.0 and rng.random() < 0.3,
                        layout=rng.choice(("bhsd", "bshd")))
        elif kind in ("norm", "norm_train"):
            c = _norm(kind, dtype, batch, heads, kv, _log_int(rng, 1, 16384), d, rng.choice((d, d, d // 2)),
                      interleaved=rng.random() < 0.5, layout=rng.choice(("bhsd", "bshd")),
                      start=rng.choice((0, 0, 5000, 200000)))
        else:
            fill = kind in ("norm_append", "c4_fill")
            c = _cached(kind, dtype, batch, heads, kv,
                        _log_int(rng, 1, 4096) if fill else rng.choice((1, 1, 2, 7, 16, 25, 48, 64, 100)),
                        _log_int(rng, 30, 2000 if fill else 65536), d, page=rng.choice((0, 16, 64, 256)),
                        size=size if kind == "window_cache" or rng.random() < 0.4 else 0, sinks=sinks,
                        softcap=0.0 if fill else cap, tree=not fill and rng.random() < 0.4,
                        rot=rng.choice((d, d // 2)) if kind == "norm_append" else 0)
        w = work(c)
        # f32 products run at a sixteenth of the 16-bit rate
        if w["flops"] * (16 if c["dtype"] == "f32" else 1) <= flops and 1e5 <= w["bytes"] <= moved:
            return c


# ---------------------------------------------------------------------------
# What a case consists of besides values
# ---------------------------------------------------------------------------
def _cache_lengths(c):
    rng = random.Random(c["length"] * 1000003 + c["batch"])
    return [c["length"]] + [max(1, int(c["length"] * rng.uniform(0.4, 1.0))) for _ in range(c["batch"] - 1)]


def _ancestors(c, b):
    """n x n truth values, token i sees token j (itself and its ancestors), and each token's depth."""
    rng = random.Random(c["n"] * 1000003 + b)
    vis = np.tril(np.ones((c["n"], c["n"]), dtype=bool))
    depth = list(range(c["n"]))
    if c["tree"]:
        vis = np.eye(c["n"], dtype=bool)
        for i in range(1, c["n"]):
            parent = rng.randrange(max(0, i - 6), i)
            vis[i] |= vis[parent]
            depth[i] = depth[parent] + 1
    return vis, depth


def _slopes(heads):
    return [2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)]


def _start(c):
    """Position of query 0: a chunk of queries stands at the end of the keys."""
    return c["sk"] - c["sq"]


def _window_pairs(c):
    """Visible (query, key) pairs of one head of one sequence."""
    i = np.arange(c["sq"], dtype=np.int64) + _start(c)
    end = np.minimum(i + (1 if c["causal"] else c["size"]), c["sk"])
    low = np.maximum(i - c["size"] + 1, 0)
    sinks = np.minimum(c["sinks"], i + 1 if c["causal"] else c["sk"])
    return int((np.maximum(end - low, 0) + np.minimum(sinks, low)).sum()
               + (0 if c["causal"] else np.maximum(sinks - end, 0).sum()))


def _cache_seen(c, b, length):
    """[n, length + n] truth values: what the new tokens of sequence b see."""
    vis, depth = _ancestors(c, b)
    at = np.concatenate((np.arange(length), length + np.array(depth)))
    seen = np.concatenate((np.ones((c["n"], length), dtype=bool), vis), axis=1)
    if c["size"]:
        far = (length + np.array(depth))[:, None] - at[None, :] >= c["size"]
        seen &= ~far | (np.arange(length + c["n"]) < c["sinks"])[None, :]
    return seen


def work(case):
    c = case
    e = _SIZE[c["dtype"]]
    kv_row = c["kv_heads"] * c["d"]
    if c["kind"] in ("window", "window_train"):
        q, kv = c["batch"] * c["heads"] * c["sq"] * c["d"], c["batch"] * c["sk"] * kv_row
        pairs, train = c["batch"] * _window_pairs(c), c["kind"] == "window_train"
        if not train and c["sq"] < c["sk"]:   # keys that no query of the chunk sees
            kv = c["batch"] * min(c["sk"], c["sq"] + c["size"] + c["sinks"]) * kv_row
        return {"bytes": e * (2 + 2 * train) * (q + kv), "flops": (14 if train else 4) * c["d"] * pairs * c["heads"]}
    if c["kind"] in ("norm", "norm_train"):
        n = c["batch"] * c["seq"] * (c["heads"] + c["kv_heads"]) * c["d"]
        return {"bytes": (4 if c["kind"] == "norm_train" else 2) * e * n + 4 * c["batch"] * c["seq"],
                "flops": (20 if c["kind"] == "norm_train" else 7) * n}
    new = c["batch"] * c["n"]
    q = new * c["heads"] * c["d"]
    if c["kind"] == "norm_append":
        return {"bytes": e * (2 * q + 4 * new * kv_row), "flops": 7 * (q + new * kv_row)}
    if c["kind"] == "c4_fill":
        # 16 bits in, five written, five read, 16 out
        return {"bytes": 2 * new * kv_row * (2 * e + 2 * 0.625), "flops": 16 * new * kv_row}
    pairs = rows = 0
    for b, length in enumerate(_cache_lengths(c)):
        seen = _cache_seen(c, b, length)
        pairs += int(seen.sum())
        rows += int(seen.any(axis=0).sum())
    row = 1.25 if c["kind"] == "c4_attention" else 2 * e
    return {"bytes": 2 * e * q + row * rows * kv_row, "flops": 4 * c["d"] * pairs * c["heads"]}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _tensor(g, c, heads, seq, layout="bhsd"):
    """[batch, heads, seq, d] as seen, stored in the case's layout."""
    shape = (c["batch"], heads, seq, c["d"]) if layout == "bhsd" else (c["batch"], seq, heads, c["d"])
    x = torch.randn(shape, device="cuda", generator=g).to(_TORCH[c["dtype"]])
    return x if layout == "bhsd" else x.transpose(1, 2)


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _weights(g, c):
    """Weights of the two norms, around 1 as trained ones are."""
    return {x: (1.0 + 0.2 * torch.randn(c["d"], device="cuda", generator=g)).to(_TORCH[c["dtype"]])
            for x in ("qw", "kw")}


def _window_inputs(c, seed):
    g = _generator(seed)
    s = {"q": _tensor(g, c, c["heads"], c["sq"], c["layout"]),
         "k": _tensor(g, c, c["kv_heads"], c["sk"], c["layout"]),
         "v": _tensor(g, c, c["kv_heads"], c["sk"], c["layout"])}
    if c["kind"] == "window_train":
        s["dout"] = _tensor(g, c, c["heads"], c["sq"], c["layout"])
    s["slopes"] = torch.tensor(_slopes(c["heads"]), device="cuda") if c["alibi"] else None
    return s


def _norm_inputs(c, seed):
    g = _generator(seed)
    # projections of different size, as heads have them
    s = {"q": (_tensor(g, c, c["heads"], c["seq"], c["layout"]) * 3.0),
         "k": (_tensor(g, c, c["kv_heads"], c["seq"], c["layout"]) * 0.5), **_weights(g, c)}
    s["pos"] = torch.arange(c["seq"], device="cuda", dtype=torch.int32)[None, :].repeat(c["batch"], 1) + c["start"]
    if c["kind"] == "norm_train":
        s["dqout"] = _tensor(g, c, c["heads"], c["seq"], c["layout"])
        s["dkout"] = _tensor(g, c, c["kv_heads"], c["seq"], c["layout"])
    return s


def _cache_inputs(c, seed):
    """The cache holds capacity rows a sequence, in pages of a common pool (page > 0) or one after another."""
    g = _generator(seed)
    lens = _cache_lengths(c)
    cap = -(-(max(lens) + c["n"]) // 8) * 8
    t = _TORCH[c["dtype"]]
    s = {"q": _tensor(g, c, c["heads"], c["n"]), "table": None, "lens": _int32(lens), "host_lens": lens}
    blocks, rows = c["batch"], cap
    if c["page"]:
        per = -(-cap // c["page"])
        order = np.random.default_rng(seed).permutation(c["batch"] * per).reshape(c["batch"], per)
        s["table"] = _int32(order.tolist())
        blocks, rows = c["batch"] * per, c["page"]
    if c["kind"] in ("norm_append", "c4_fill"):
        s["knew"], s["vnew"] = _tensor(g, c, c["kv_heads"], c["n"]), _tensor(g, c, c["kv_heads"], c["n"])
    if c["kind"] == "norm_append":
        s.update(_weights(g, c))
    trees = [_ancestors(c, b) for b in range(c["batch"])]
    s["pos"] = _int32([[n + x for x in depth] for n, (_, depth) in zip(lens, trees)])
    s["seen"] = torch.tensor(np.stack([v for v, _ in trees]), device="cuda")
    words = -(-c["n"] // 64)
    bits = np.zeros((c["batch"], c["n"], words * 64), dtype=np.uint64)
    bits[:, :, :c["n"]] = np.stack([v for v, _ in trees])
    packed = (bits.reshape(c["batch"], c["n"], words, 64) << np.arange(64, dtype=np.uint64)).sum(axis=-1,
                                                                                                dtype=np.uint64)
    s["mask"] = torch.from_numpy(packed.view(np.int64)).cuda()
    if not c["kind"].startswith("c4"):
        shape = (blocks, rows, c["kv_heads"], c["d"])
        s["kcache"] = torch.randn(shape, device="cuda", generator=g).to(t)
        s["vcache"] = torch.randn(shape, device="cuda", generator=g).to(t)
        return s
    shape = (blocks, c["kv_heads"], rows, c["d"])
    if c["kind"] == "c4_fill":   # no rows yet
        k = v = torch.zeros(shape, device="cuda", dtype=t)
    else:
        k = torch.randn(shape, device="cuda", generator=g).to(t)
        v = torch.randn(shape, device="cuda", generator=g).to(t)
    s["k4"], s["ks"] = _pack_k(*_quantise(k))
    s["v4"], s["vs"] = _pack_v(*_quantise(v))
    s["rows"] = s["lens"][:, None] + torch.arange(c["n"], device="cuda", dtype=torch.int32)[None, :]
    return s


# The cache in 4 bits.  32 columns of a row share a step: S (16 steps, 16 bits) and O; the code c stands for
# O + (1 + c / 16) S.  Keys: 8 columns a word; values: 8 rows of a column a word; entry e of the eight in the
# bits from 4 (e / 2) + 16 (e % 2) on.
_SHIFTS = [4 * (e // 2) + 16 * (e % 2) for e in range(8)]


def _quantise(x):
    """[..., d] -> codes [..., d] (int32), S and O [..., d / 32] (f16)."""
    y = x.float().unflatten(-1, (-1, 32))
    lo, hi = y.amin(dim=-1), y.amax(dim=-1)
    big = ((hi - lo) * 16.0 / 15.0).half()
    off = (lo - big.float()).half()
    step = big.float()[..., None] * 0.0625
    code = torch.round((y - off.float()[..., None]) / torch.where(step == 0, torch.ones_like(step), step) - 16.0)
    code = torch.where(step == 0, torch.zeros_like(code), code.clamp(0.0, 15.0))
    return code.flatten(-2).to(torch.int32), big, off


def _join(codes):
    """[..., 8] codes -> words."""
    w = torch.zeros_like(codes[..., 0])
    for e, sh in enumerate(_SHIFTS):
        w |= codes[..., e] << sh
    return w


def _split(words):
    """words -> [..., 8] codes."""
    return torch.stack([(words >> sh) & 15 for sh in _SHIFTS], dim=-1)


def _pack_k(codes, big, off):
    """[blocks, heads, rows, d / 8] words and [blocks, heads, rows, d / 32, (S, O)]."""
    return _join(codes.unflatten(-1, (-1, 8))), torch.stack((big, off), dim=-1)


def _pack_v(codes, big, off):
    """[blocks, heads, rows / 8, d] words and [blocks, heads, rows / 8, d / 32, (S, O), 8]."""
    w = _join(codes.unflatten(2, (-1, 8)).transpose(3, 4).contiguous())
    p = torch.stack((big, off), dim=-1).unflatten(2, (-1, 8))   # [blocks, heads, rows / 8, 8, d / 32, 2]
    return w, p.permute(0, 1, 2, 4, 5, 3).contiguous()


def _unpack_k(words, scales):
    """f32 values [..., rows, d] of keys."""
    c = _split(words).flatten(-2).float().unflatten(-1, (-1, 32))
    return (scales[..., 1:2].float() + (1.0 + c * 0.0625) * scales[..., 0:1].float()).flatten(-2)


def _unpack_v(words, scales):
    """f32 values [..., rows, d] of values."""
    c = _split(words).transpose(-1, -2).float().unflatten(-1, (-1, 32))   # [..., rows / 8, 8, d / 32, 32]
    p = scales.float().transpose(-1, -3)   # [..., rows / 8, 8, (S, O), d / 32]
    x = p[..., 1, :, None] + (1.0 + c * 0.0625) * p[..., 0, :, None]
    return x.flatten(-2).flatten(-3, -2)


_INPUTS = {"window": _window_inputs, "window_train": _window_inputs, "norm": _norm_inputs, "norm_train": _norm_inputs,
           "window_cache": _cache_inputs, "norm_append": _cache_inputs, "c4_attention": _cache_inputs,
           "c4_fill": _cache_inputs}


def _strides(x):
    """Element strides of a [batch, heads, seq, d] view as (batch, seq, head)."""
    return (x.stride(0), x.stride(2), x.stride(1))


def prepare(case, seed):
    c = case
    s = _INPUTS[c["kind"]](c, seed)
    s["case"] = c
    if not own:
        return s
    fa = _fa()
    fa.init()
    dtype = {"f32": fa.DTYPE_F32, "bf16": fa.DTYPE_BF16, "f16": fa.DTYPE_F16}[c["dtype"]]

    def ptr(x):
        return 0 if x is None else x.data_ptr()

    if "size" in c:
        s["window"] = fa.window(c["size"], c["sinks"]) if c["size"] else None
    if c["kind"] in ("window", "window_train"):
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(c["batch"], c["heads"], c["sq"], device="cuda")
        strides = {x: _strides(s[x]) for x in ("q", "k", "v", "out")}
        if c["kind"] == "window_train":
            for x in ("q", "k", "v"):
                s["d" + x] = torch.empty_like(s[x])
            strides.update({x: _strides(s[x]) for x in ("dout", "dq", "dk", "dv")})
        s["cfg"] = fa.score_config(dtype, c["batch"], c["heads"], c["kv_heads"], c["sq"], c["sk"], c["d"],
                                   causal=c["causal"], softcap=c["softcap"], q_start=_start(c),
                                   slopes_ptr=ptr(s["slopes"]), strides=strides)
        return s
    if "rot" in c and c["rot"]:
        s["rot"] = fa.rotary_config(dtype, c["d"], c["rot"], interleaved=c.get("interleaved", False), base=_BASE)
        s["norm"] = fa.head_norm(s["qw"].data_ptr(), s["kw"].data_ptr(), _EPS)
    if c["kind"] in ("norm", "norm_train"):
        s["qout"], s["kout"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        s["qt"] = fa.rotary_tensor(c["heads"], _strides(s["q"]), _strides(s["qout"]))
        s["kt"] = fa.rotary_tensor(c["kv_heads"], _strides(s["k"]), _strides(s["kout"]))
        if c["kind"] == "norm_train":
            s["dq"], s["dk"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
            s["dqw"], s["dkw"] = torch.empty(c["d"], device="cuda"), torch.empty(c["d"], device="cuda")
            s["qg"] = fa.norm_grad(c["heads"], _strides(s["q"]), _strides(s["dqout"]), _strides(s["dq"]))
            s["kg"] = fa.norm_grad(c["kv_heads"], _strides(s["k"]), _strides(s["dkout"]), _strides(s["dk"]))
        return s
    paged = {"block_table_ptr": ptr(s["table"]), "page_size": c["page"],
             "pages_per_seq": s["table"].shape[1] if c["page"] else 0}
    if c["kind"].startswith("c4"):
        blocks, rows = s["k4"].shape[0], s["k4"].shape[2]
        s["cache"] = fa.kv_cache4(dtype, c["batch"], c["kv_heads"], c["d"], ptr(s["k4"]), ptr(s["ks"]), ptr(s["v4"]),
                                  ptr(s["vs"]), ptr(s["lens"]), capacity=0 if c["page"] else rows,
                                  n_pages=blocks if c["page"] else 0, **paged)
    else:
        kc, vc = s["kcache"], s["vcache"]
        s["cache"] = fa.kv_cache(dtype, c["batch"], c["kv_heads"], c["d"], ptr(kc), ptr(vc),
                                 k_strides=(kc.stride(0), kc.stride(1), kc.stride(2)),
                                 v_strides=(vc.stride(0), vc.stride(1), vc.stride(2)), lens_ptr=ptr(s["lens"]),
                                 capacity=0 if c["page"] else kc.shape[1], n_pages=kc.shape[0] if c["page"] else 0,
                                 **paged)
    s["out"] = torch.empty_like(s["q"])
    if c["kind"] in ("window_cache", "c4_attention"):
        s["cfg"] = fa.tree_config(c["heads"], c["n"], mask_ptr=ptr(s["mask"]) if c["tree"] else 0,
                                  softcap=c["softcap"], positions_ptr=ptr(s["pos"]) if c["tree"] else 0)
    elif c["kind"] == "norm_append":
        s["append"] = fa.append_config(c["n"], rotary=s["rot"], k_strides=_strides(s["knew"]),
                                       v_strides=_strides(s["vnew"]),
                                       q_layout=fa.rotary_tensor(c["heads"], _strides(s["q"]), _strides(s["out"])))
    else:
        s["append"] = fa.append_config(c["n"], k_strides=_strides(s["knew"]), v_strides=_strides(s["vnew"]))
        s["kread"], s["vread"] = torch.empty_like(s["knew"]), torch.empty_like(s["vnew"])
        s["read"] = fa.read_config(c["n"], _strides(s["kread"]), _strides(s["vread"]))
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    c = state["case"]
    if own:
        return _run_own(state)
    if c["kind"] in ("window", "window_train"):
        return _plain_window(state)
    if c["kind"] in ("norm", "norm_train"):
        return _plain_norm(state)
    if c["kind"] == "norm_append":
        return _plain_append(state)
    if c["kind"] == "c4_fill":
        return _plain_fill(state)
    return _plain_cache(state)


def _run_own(s):
    c, fa = s["case"], _fa()
    stream = torch.cuda.current_stream().cuda_stream
    if c["kind"] in ("window", "window_train"):
        q, k, v = s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr()
        fa.score_attention_device(s["cfg"], q, k, v, s["out"].data_ptr(), s["lse"].data_ptr(), stream,
                                  window=s["window"])
        if c["kind"] == "window":
            return {"out": s["out"], "lse": s["lse"]}
        fa.score_attention_backward_device(s["cfg"], q, k, v, s["out"].data_ptr(), s["lse"].data_ptr(),
                                           s["dout"].data_ptr(), s["dq"].data_ptr(), s["dk"].data_ptr(),
                                           s["dv"].data_ptr(), stream, window=s["window"])
        return {"out": s["out"], "lse": s["lse"], "dq": s["dq"], "dk": s["dk"], "dv": s["dv"]}
    if c["kind"] in ("norm", "norm_train"):
        fa.norm_rotary_device(s["rot"], s["norm"], c["batch"], c["seq"], s["pos"].data_ptr(), s["qt"],
                              s["q"].data_ptr(), s["qout"].data_ptr(), s["kt"], s["k"].data_ptr(),
                              s["kout"].data_ptr(), stream)
        if c["kind"] == "norm":
            return {"q": s["qout"], "k": s["kout"]}
        fa.norm_rotary_backward_device(s["rot"], s["norm"], c["batch"], c["seq"], s["pos"].data_ptr(), s["qg"],
                                       s["q"].data_ptr(), s["dqout"].data_ptr(), s["dq"].data_ptr(),
                                       s["dqw"].data_ptr(), s["kg"], s["k"].data_ptr(), s["dkout"].data_ptr(),
                                       s["dk"].data_ptr(), s["dkw"].data_ptr(), stream)
        return {"q": s["qout"], "k": s["kout"], "dq": s["dq"], "dk": s["dk"], "dqw": s["dqw"], "dkw": s["dkw"]}
    q, out = s["q"].data_ptr(), s["out"].data_ptr()
    if c["kind"] == "norm_append":
        fa.cache_append_device(s["cache"], s["append"], s["knew"].data_ptr(), s["vnew"].data_ptr(),
                               s["pos"].data_ptr(), q, out, stream=stream, norm=s["norm"])
        return {"q": s["out"], "k": s["kcache"], "v": s["vcache"]}
    if c["kind"] == "c4_fill":
        fa.cache4_append_device(s["cache"], s["append"], s["knew"].data_ptr(), s["vnew"].data_ptr(), stream=stream)
        fa.cache4_read_device(s["cache"], s["read"], s["rows"].data_ptr(), s["kread"].data_ptr(),
                              s["vread"].data_ptr(), stream=stream)
        return {"k": s["kread"], "v": s["vread"]}
    call = fa.cache4_attention_device if c["kind"] == "c4_attention" else fa.tree_attention_device
    call(s["cfg"], s["cache"], q, out, stream=stream, window=s["window"])
    return {"out": s["out"]}


# ---------------------------------------------------------------------------
# Plain form
# ---------------------------------------------------------------------------
def _plain_softmax(s, seen):
    """Probabilities and log of the sum over the seen keys of each row; rows that see none get zeros."""
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    l = p.sum(dim=-1, keepdim=True)
    return p / torch.where(l == 0, torch.ones_like(l), l), (m + torch.log(l)).squeeze(-1)


def _plain_window(state):
    c, train = state["case"], state["case"]["kind"] == "window_train"
    q, k, v, slopes = state["q"], state["k"], state["v"], state["slopes"]
    group, scale, cap = c["heads"] // c["kv_heads"], c["d"] ** -0.5, c["softcap"]
    qpos = torch.arange(c["sq"], device="cuda") + _start(c)
    kpos = torch.arange(c["sk"], device="cuda")
    distance = (qpos[:, None] - kpos[None, :]).abs()
    seen = (distance < c["size"]) | (kpos < c["sinks"])[None, :]
    if c["causal"]:
        seen = seen & (kpos[None, :] <= qpos[:, None])
    distance = distance.float() if c["alibi"] else None
    lse = torch.empty(c["batch"], c["heads"], c["sq"], device="cuda")
    res = {"out": torch.empty_like(q), "lse": lse}
    if train:
        res.update(dq=torch.empty_like(q), dk=torch.empty_like(k), dv=torch.empty_like(v))
    for b in range(c["batch"]):
        for hk in range(c["kv_heads"]):
            kf, vf = k[b, hk].float(), v[b, hk].float()
            kt, vt = kf.t().contiguous(), vf.t().contiguous()
            dk, dv = torch.zeros_like(kf), torch.zeros_like(vf)
            for h in range(hk * group, (hk + 1) * group):
                qf = q[b, h].float()
                y = torch.matmul(qf, kt) * scale
                if cap:
                    y = cap * torch.tanh(y / cap)
                p, res["lse"][b, h] = _plain_softmax(y - slopes[h] * distance if c["alibi"] else y, seen)
                o = torch.matmul(p, vf)
                res["out"][b, h] = o.to(q.dtype)
                if train:
                    do = state["dout"][b, h].float()
                    dv += torch.matmul(p.t().contiguous(), do)
                    ds = p * (torch.matmul(do, vt) - (do * o).sum(dim=-1, keepdim=True))
                    if cap:
                        ds = ds * (1.0 - (y / cap) ** 2)
                    ds = ds * scale
                    res["dq"][b, h] = torch.matmul(ds, kf).to(q.dtype)
                    dk += torch.matmul(ds.t().contiguous(), qf)
            if train:
                res["dk"][b, hk], res["dv"][b, hk] = dk.to(k.dtype), dv.to(v.dtype)
    return res


def _plain_turn(x, pos, c, sign=1.0):
    """x: [batch, heads, seq, d] in 32 bits, pos: [batch, seq]."""
    rot = c["rot"]
    f = _BASE ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = pos.double()[:, None, :, None] * f   # far positions: 32 bits lose the angle
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float() * sign
    out = x.clone()
    if c.get("interleaved", False):
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        out[..., :rot // 2], out[..., rot // 2:rot] = a * cos - b * sin, a * sin + b * cos
    return out


def _plain_normed(x, weight):
    """x / its root mean square, in 32 bits, and that times the weights."""
    xf = x.float()
    y = xf * torch.rsqrt((xf * xf).mean(dim=-1, keepdim=True) + _EPS)
    return y, y * weight.float()


def _plain_norm(state):
    c = state["case"]
    res = {}
    for x in ("q", "k"):
        res[x] = _plain_turn(_plain_normed(state[x], state[x + "w"])[1], state["pos"], c).to(state[x].dtype)
    if c["kind"] == "norm_train":
        for x in ("q", "k"):
            xf, w = state[x].float(), state[x + "w"].float()
            r = torch.rsqrt((xf * xf).mean(dim=-1, keepdim=True) + _EPS)
            g = _plain_turn(state[f"d{x}out"].float(), state["pos"], c, -1.0)
            y = xf * r
            res[f"d{x}w"] = (g * y).sum(dim=(0, 1, 2), dtype=torch.float64).float()
            g = g * w
            res["d" + x] = (r * (g - y * (g * y).mean(dim=-1, keepdim=True))).to(state[x].dtype)
    return res


def _rows_at(c, state, b, rows):
    """(block, row) of a sequence's rows."""
    if c["page"]:
        return state["table"][b].long()[rows // c["page"]], rows % c["page"]
    return torch.full_like(rows, b), rows


def _plain_append(state):
    c = state["case"]
    q = _plain_turn(_plain_normed(state["q"], state["qw"])[1], state["pos"], c).to(state["q"].dtype)
    k = _plain_turn(_plain_normed(state["knew"], state["kw"])[1], state["pos"], c).to(state["q"].dtype)
    for b, length in enumerate(state["host_lens"]):
        at = _rows_at(c, state, b, torch.arange(length, length + c["n"], device="cuda"))
        state["kcache"][at[0], at[1]] = k[b].transpose(0, 1)
        state["vcache"][at[0], at[1]] = state["vnew"][b].transpose(0, 1)
    return {"q": q, "k": state["kcache"], "v": state["vcache"]}


def _plain_fill(state):
    """Keys and values as the cache holds them (its buffers are the library's own)."""
    t = state["knew"].dtype
    return {"k": _unpack_k(*_pack_k(*_quantise(state["knew"]))).to(t), "v": _unpack_codes(state["vnew"]).to(t)}


def _unpack_codes(x):
    code, big, off = _quantise(x)
    c = code.float().unflatten(-1, (-1, 32))
    return (off.float()[..., None] + (1.0 + c * 0.0625) * big.float()[..., None]).flatten(-2)


def _cache_rows(state, b, first, end):
    """Keys [kv_heads, d, rows] and values [kv_heads, rows, d] of a sequence's rows in 32 bits."""
    c = state["case"]
    rows = torch.arange(first, end, device="cuda")
    if c["kind"] == "window_cache":
        at = _rows_at(c, state, b, rows)
        k, v = state["kcache"][at[0], at[1]].float(), state["vcache"][at[0], at[1]].float()
        return k.permute(1, 2, 0).contiguous(), v.transpose(0, 1).contiguous()
    blk, row = _rows_at(c, state, b, rows)
    k = _unpack_k(state["k4"][blk, :, row], state["ks"][blk, :, row])           # [rows, kv_heads, d]
    first8 = first // 8 * 8
    rows8 = torch.arange(first8, end, 8, device="cuda")
    blk, row = _rows_at(c, state, b, rows8)
    v = _unpack_v(state["v4"][blk, :, row // 8].transpose(0, 1), state["vs"][blk, :, row // 8].transpose(0, 1))
    return k.permute(1, 2, 0).contiguous(), v[:, first - first8:end - first8].contiguous()


def _plain_cache(state):
    c, q = state["case"], state["q"]
    group, cap, n = c["heads"] // c["kv_heads"], c["softcap"], c["n"]
    res = torch.empty_like(q)
    for b, length in enumerate(state["host_lens"]):
        # the sinks, and the rows from the first that the window of some token reaches
        first = max(0, length - c["size"] + 1) if c["size"] else 0
        parts = [(0, min(c["sinks"], first)), (first, length + n)] if first and c["sinks"] else [(first, length + n)]
        got = [_cache_rows(state, b, *p) for p in parts]
        kf, vf = torch.cat([k for k, _ in got], dim=2), torch.cat([v for _, v in got], dim=1)
        rows = torch.cat([torch.arange(*p, device="cuda") for p in parts])
        keys = rows.numel()
        qf = q[b].float().reshape(c["kv_heads"], group * n, c["d"])
        s = torch.matmul(qf, kf).reshape(c["heads"], n, keys) * c["d"] ** -0.5
        if cap:
            s = cap * torch.tanh(s / cap)
        seen = torch.cat((torch.ones(n, keys - n, dtype=torch.bool, device="cuda"), state["seen"][b]), dim=1)
        if c["size"]:
            pos = state["pos"][b].long()
            at = torch.cat((rows[:keys - n], pos))
            seen = seen & ((pos[:, None] - at[None, :] < c["size"]) | (rows < c["sinks"])[None, :])
        p, _ = _plain_softmax(s, seen)
        o = torch.matmul(p.reshape(c["kv_heads"], group * n, keys), vf)
        res[b] = o.reshape(c["heads"], n, c["d"]).to(q.dtype)
    return {"out": res}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    c = case
    s = _INPUTS[c["kind"]](c, seed)
    if c["kind"] in ("window", "window_train"):
        return _exact_window(c, s)
    if c["kind"] in ("norm", "norm_train"):
        return _exact_norm(c, s)
    if c["kind"] == "norm_append":
        out = {"q": _exact_normed(c, s["q"], s["qw"], s["pos"]), "k": s["kcache"].double(), "v": s["vcache"].double()}
        knew = _exact_normed(c, s["knew"], s["kw"], s["pos"])
        for b, length in enumerate(_cache_lengths(c)):
            blk, row = zip(*(_exact_place(c, s, b, length + i) for i in range(c["n"])))
            blk, row = torch.tensor(blk, device=knew.device), torch.tensor(row, device=knew.device)
            out["k"][blk, row] = knew[b].transpose(0, 1)
            out["v"][blk, row] = s["vnew"][b].transpose(0, 1).double()
        return out
    if c["kind"] == "c4_fill":
        return {"k": _exact_stored(s["knew"]), "v": _exact_stored(s["vnew"])}
    return _exact_cache(c, s)


def _exact_place(c, s, b, row):
    if not c["page"]:
        return b, row
    if "host_table" not in s:
        s["host_table"] = s["table"].tolist()
    return s["host_table"][b][row // c["page"]], row % c["page"]


def _exact_weights(z, hidden):
    """softmax over the keys that are not hidden, and its log-sum; a row of hidden keys has weight nowhere."""
    z = torch.where(hidden, torch.full_like(z, -math.inf), z)
    lse = torch.logsumexp(z, dim=-1)
    return torch.exp(z - lse[..., None]).nan_to_num_(0.0), lse


def _exact_window(c, s):
    dev = s["q"].device
    i = torch.arange(c["sk"] - c["sq"], c["sk"], device=dev)[:, None]
    j = torch.arange(c["sk"], device=dev)[None, :]
    hidden = ((i - j >= c["size"]) | (j - i >= c["size"])) & (j >= c["sinks"])
    if c["causal"]:
        hidden = hidden | (j > i)
    per = c["heads"] // c["kv_heads"]
    o = {"out": torch.empty(s["q"].shape, dtype=torch.float64, device=dev),
         "lse": torch.empty(c["batch"], c["heads"], c["sq"], dtype=torch.float64, device=dev)}
    if c["kind"] == "window_train":
        for x in ("q", "k", "v"):
            o["d" + x] = torch.zeros(s[x].shape, dtype=torch.float64, device=dev)
    for b in range(c["batch"]):
        for h in range(c["heads"]):
            Q, K, V = s["q"][b, h].double(), s["k"][b, h // per].double(), s["v"][b, h // per].double()
            x = (Q @ K.t().contiguous()) / math.sqrt(c["d"])
            slope = 1.0
            if c["softcap"]:
                th = torch.tanh(x / c["softcap"])
                x, slope = c["softcap"] * th, 1.0 - th * th
            if c["alibi"]:
                x = x - float(s["slopes"][h]) * (i - j).abs().double()
            P, o["lse"][b, h] = _exact_weights(x, hidden)
            o["out"][b, h] = P @ V
            if c["kind"] == "window_train":
                dO = s["dout"][b, h].double()
                o["dv"][b, h // per] += P.t().contiguous() @ dO
                dP = dO @ V.t().contiguous()
                dX = P * (dP - (P * dP).sum(-1, keepdim=True)) * slope / math.sqrt(c["d"])
                o["dq"][b, h] = dX @ K
                o["dk"][b, h // per] += dX.t().contiguous() @ Q
    return o


def _exact_turn(c, y, pos, sign=1.0):
    half = c["rot"] // 2
    freq = torch.tensor([_BASE ** (-2.0 * p / c["rot"]) for p in range(half)], dtype=torch.float64, device=y.device)
    t = sign * pos.double()[:, None, :, None] * freq
    turn = torch.polar(torch.ones_like(t), t)
    if c.get("interleaved", False):
        z = torch.complex(y[..., 0:c["rot"]:2].contiguous(), y[..., 1:c["rot"]:2].contiguous()) * turn
        head = torch.stack((z.real, z.imag), dim=-1).flatten(-2)
    else:
        z = torch.complex(y[..., :half].contiguous(), y[..., half:c["rot"]].contiguous()) * turn
        head = torch.cat((z.real, z.imag), dim=-1)
    return torch.cat((head, y[..., c["rot"]:]), dim=-1)


def _exact_normed(c, x, w, pos):
    y = x.double()
    return _exact_turn(c, y / torch.sqrt(y.square().mean(-1, keepdim=True) + _EPS) * w.double(), pos)


def _exact_norm(c, s):
    o = {x: _exact_normed(c, s[x], s[x + "w"], s["pos"]) for x in ("q", "k")}
    if c["kind"] == "norm_train":
        for x in ("q", "k"):
            y = s[x].double()
            size = torch.sqrt(y.square().mean(-1, keepdim=True) + _EPS)
            back = _exact_turn(c, s[f"d{x}out"].double(), s["pos"], -1.0)
            o[f"d{x}w"] = (back * y / size).sum(dim=(0, 1, 2))
            back = back * s[x + "w"].double()
            o["d" + x] = back / size - y * (back * y).sum(-1, keepdim=True) / (c["d"] * size ** 3)
    return o


def _exact_stored(x):
    """What 4 bits hold of x [..., d]."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for g in range(0, x.shape[-1], 32):
        y = x[..., g:g + 32].double()
        lo = y.min(dim=-1, keepdim=True).values
        big = ((y.max(dim=-1, keepdim=True).values - lo) / 15 * 16).half().double()
        off = (lo - big).half().double()
        code = torch.clip(torch.round((y - off) / big * 16 - 16), 0, 15)
        code = torch.where(big > 0, code, torch.zeros_like(code))
        out[..., g:g + 32] = off + big + code * big / 16
    return out


def _exact_cache(c, s):
    dev, n, per = s["q"].device, c["n"], c["heads"] // c["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=dev)
    if c["kind"] == "window_cache":
        K, V = s["kcache"].transpose(1, 2).double(), s["vcache"].transpose(1, 2).double()
    else:
        K, V = (torch.empty(s["k4"].shape[:3] + (c["d"],), dtype=torch.float64, device=dev) for _ in range(2))
        for e in range(8):
            at = 4 * (e // 2) + 16 * (e % 2)
            scale = s["ks"].double().repeat_interleave(4, dim=3)
            K[..., e::8] = scale[..., 1] + scale[..., 0] * (1 + ((s["k4"] >> at) & 15).double() / 16)
            scale = s["vs"][..., e].double().repeat_interleave(32, dim=3)
            V[:, :, e::8] = scale[..., 1] + scale[..., 0] * (1 + ((s["v4"] >> at) & 15).double() / 16)
    for b, length in enumerate(_cache_lengths(c)):
        place = [_exact_place(c, s, b, r) for r in range(length + n)]
        page = torch.tensor([p for p, _ in place], device=dev)
        row = torch.tensor([r for _, r in place], device=dev)
        hidden = ~torch.tensor(_cache_seen(c, b, length), device=dev)
        for hk in range(c["kv_heads"]):
            Kh, Vh = K[page, hk, row], V[page, hk, row]
            for h in range(hk * per, (hk + 1) * per):
                x = (s["q"][b, h].double() @ Kh.t().contiguous()) / math.sqrt(c["d"])
                if c["softcap"]:
                    x = c["softcap"] * torch.tanh(x / c["softcap"])
                out[b, h] = _exact_weights(x, hidden)[0] @ Vh
    return {"out": out}
