"""Score attention, tree attention over a cache and rotary positions: timed cases.

Each case is one pass through one of these operators as a training or serving
program makes it, with tensors on the GPU and on torch's current stream:

  score   softmax attention whose scores are capped by a tanh, get a bias that
          falls with the distance, a document mask or a prefix mask (forward;
          one query and many keys is a decode step)
  train   its forward and backward pass: output and the gradients of Q, K, V
  rotary  rotary positions on the queries and keys of a layer (or, inverse, on
          their gradients)
  tree    attention of a tree of drafted tokens over a cache, contiguous or paged
  step    a layer's share of a verification step: rotary positions on the
          queries, the drafted keys (rotated) and values into the cache, tree
          attention

``own`` chooses between the package's kernels and a plain form out of
elementary torch operations in 32 bits.  ``exact`` is the definition in 64
bits, written apart from both.

Inputs are N(0, 1), queries and keys N(0, sigma) in the 16-bit or f32 type of
the case.  Document lengths, cache lengths and drafted trees come from the
case, so that its work is known; the values and page tables from the seed.
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


def _fa():
    p = os.path.join(_ROOT, "flash-attention-cpu_amd")
    if p not in sys.path:
        sys.path.insert(0, p)
    import flash_attention_amd
    return flash_attention_amd


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _score(kind, dtype, batch, heads, kv_heads, sq, sk, d, name=None, layout="bhsd", causal=True, softcap=0.0,
           alibi=False, docs=0, prefix=0, sigma=1.0):
    c = {"kind": kind, "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "sq": sq, "sk": sk,
         "d": d, "layout": layout, "causal": causal, "softcap": softcap, "alibi": alibi, "docs": docs,
         "prefix": prefix, "sigma": sigma}
    if name is not None:
        c["name"] = name
    return c


def _rotary(dtype, batch, heads, kv_heads, seq, d, rot, name=None, interleaved=False, scaling="none", inverse=False,
            start=0, layout="bshd"):
    c = {"kind": "rotary", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "seq": seq, "d": d,
         "rot": rot, "interleaved": interleaved, "scaling": scaling, "inverse": inverse, "start": start,
         "layout": layout}
    if name is not None:
        c["name"] = name
    return c


def _tree(kind, dtype, batch, heads, kv_heads, n, length, d, name=None, page=0, softcap=0.0, alibi=False, rot=0):
    c = {"kind": kind, "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "n": n,
         "length": length, "d": d, "page": page, "softcap": softcap, "alibi": alibi, "rot": rot}
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # a causal layer's prefill, grouped heads, capped scores
        _score("score", "bf16", 1, 32, 8, 2048, 2048, 128, "cap_layer", softcap=30.0, sigma=3.0),
        # one long row of packed documents, heads next to each other in memory
        _score("score", "bf16", 1, 16, 4, 16384, 16384, 128, "docs_long", layout="bshd", docs=2000),
        # one decode step of one sequence against a long cache tensor: bias by distance
        _score("score", "f16", 1, 32, 8, 1, 32768, 128, "alibi_decode", alibi=True),
        # training on packed documents with capped scores: the largest call
        _score("train", "bf16", 2, 16, 4, 4096, 4096, 128, "train_docs_cap", layout="bshd", docs=1500, softcap=50.0,
               sigma=2.0),
        # training with a bias by distance: narrow heads, a length that fills no tile
        _score("train", "f16", 1, 16, 16, 1500, 1500, 64, "train_alibi_ragged", alibi=True),
        # training of a prefix model in f32, short ragged rows
        _score("train", "f32", 2, 8, 8, 777, 777, 64, "train_prefix_f32", prefix=200),
        # queries and keys of a layer, scaled for a long context
        _rotary("bf16", 1, 32, 8, 8192, 128, 128, "rotary_layer", scaling="yarn"),
        # gradients of a layer's queries and keys: interleaved pairs, half of the head
        _rotary("f32", 2, 16, 16, 1000, 80, 40, "rotary_grad", interleaved=True, inverse=True, layout="bhsd"),
        # one sequence, a small tree: a unit of latency
        _tree("tree", "bf16", 1, 32, 8, 16, 1024, 128, "tree_small"),
        # a batch of long contexts in pages, a tree of 64 tokens
        _tree("tree", "bf16", 8, 32, 8, 64, 16384, 128, "tree_paged", page=64),
        # a verification step with capped scores: rotary, append, attention
        _tree("step", "f16", 4, 16, 2, 25, 3000, 128, "tree_step", page=16, softcap=50.0, rot=128),
    ]


def _log_int(rng, lo, hi):
    """A whole number spread over the logarithm of lo .. hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    limit = work(listed()[3])["flops"]
    while True:
        kind = rng.choice(("score", "score", "decode", "train", "train", "rotary", "tree", "tree", "step"))
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        d = rng.choice((64, 64, 128, 128, 80, 96, 256))
        kv = rng.choice((1, 2, 4, 8))
        heads = kv * rng.choice((1, 2, 4, 8))
        batch = rng.choice((1, 1, 2, 3, 8))
        cap = rng.choice((0.0, 0.0, 30.0, 50.0))
        alibi = cap == 0.0 and rng.random() < 0.5
        if kind in ("score", "train"):
            s = _log_int(rng, 100, 16384 if kind == "score" else 4096)
            mask = rng.choice(("causal", "docs", "docs", "prefix", "none", "cross"))
            sk = _log_int(rng, 100, 4096) if mask == "cross" else s
            c = _score(kind, dtype, batch, heads, kv, s, sk, d, layout=rng.choice(("bhsd", "bshd")),
                       causal=mask in ("causal", "prefix") or (mask == "docs" and rng.random() < 0.7), softcap=cap,
                       alibi=alibi, docs=_log_int(rng, 50, 4000) if mask == "docs" else 0,
                       prefix=_log_int(rng, 10, s) if mask == "prefix" else 0, sigma=rng.choice((1.0, 2.0, 3.0)))
        elif kind == "decode":
            c = _score("score", dtype, batch, heads, kv, 1, _log_int(rng, 500, 65536), d, softcap=cap, alibi=alibi)
        elif kind == "rotary":
            c = _rotary(dtype, batch, heads, kv, _log_int(rng, 1, 16384), d, rng.choice((d, d, d // 2)),
                        interleaved=rng.random() < 0.5, scaling=rng.choice(("none", "linear", "ntk", "yarn")),
                        inverse=rng.random() < 0.4, start=rng.choice((0, 0, 5000, 200000)),
                        layout=rng.choice(("bhsd", "bshd")))
        else:
            c = _tree(kind, dtype, batch, heads, kv, rng.choice((1, 2, 7, 16, 25, 48, 64, 100)),
                      _log_int(rng, 30, 32768), d, page=rng.choice((0, 16, 64, 256)), softcap=cap, alibi=alibi,
                      rot=rng.choice((d, d // 2)) if kind == "step" else 0)
        w = work(c)
        # f32 products run at a sixteenth of the 16-bit rate
        if w["flops"] * (16 if c["dtype"] == "f32" else 1) <= limit and 2e5 <= w["bytes"] <= 8e8:
            return c


# ---------------------------------------------------------------------------
# What a case consists of besides values
# ---------------------------------------------------------------------------
def _positions_of_queries(c):
    """Position of query 0 among the keys: decode steps stand behind the cache."""
    return c["sk"] - 1 if c["sq"] == 1 else 0


def _doc_ids(c):
    """Document of each token, one list a batch row; -1 marks padding at the end of a row."""
    rng = random.Random(c["docs"] * 1000003 + c["sq"])
    rows = []
    for _ in range(c["batch"]):
        ids, doc = [], 0
        end = c["sq"] - (c["sq"] // 50 if rng.random() < 0.5 else 0)
        while len(ids) < end:
            ids += [doc] * min(end - len(ids), max(1, int(c["docs"] * rng.uniform(0.3, 1.7))))
            doc += 1
        rows.append(ids + [-1] * (c["sq"] - end))
    return rows


def _prefixes(c):
    rng = random.Random(c["prefix"] * 1000003 + c["sk"])
    return [max(1, int(c["prefix"] * rng.uniform(0.5, 1.0))) for _ in range(c["batch"])]


def _cache_lengths(c):
    rng = random.Random(c["length"] * 1000003 + c["batch"])
    return [c["length"]] + [max(1, int(c["length"] * rng.uniform(0.4, 1.0))) for _ in range(c["batch"] - 1)]


def _parents(c, b):
    """A drafted tree: token 0 is the root, later tokens hang on earlier ones."""
    rng = random.Random(c["n"] * 1000003 + b)
    return [-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, c["n"])]


def _ancestors(c, b):
    """n x n truth values, token i sees token j (itself and its ancestors), and each token's depth."""
    par = _parents(c, b)
    vis = np.zeros((c["n"], c["n"]), dtype=bool)
    depth = []
    for i, p in enumerate(par):
        if p >= 0:
            vis[i] = vis[p]
        vis[i, i] = True
        depth.append(0 if p < 0 else depth[p] + 1)
    return vis, depth


def _slopes(heads):
    return [2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)]


def _visible_pairs(c):
    """Visible (query, key) pairs of one head, all batch rows together."""
    if c["kind"] in ("tree", "step"):
        return sum(n * c["n"] + int(_ancestors(c, b)[0].sum()) for b, n in enumerate(_cache_lengths(c)))
    sq, sk = c["sq"], c["sk"]
    if c["docs"]:
        total = 0
        for ids in _doc_ids(c):
            count = {}
            for i in ids:
                count[i] = count.get(i, 0) + 1
            total += sum(n * (n + 1) // 2 if c["causal"] else n * n for i, n in count.items() if i >= 0)
        return total
    if sq == 1 or not c["causal"]:
        return c["batch"] * sq * sk
    if c["prefix"]:
        return sum(sum(min(sk, max(i + 1, f)) for i in range(sq)) for f in _prefixes(c))
    n = min(sq, sk)
    return c["batch"] * (n * (n + 1) // 2 + max(0, sq - sk) * sk)


def work(case):
    c = case
    e = _SIZE[c["dtype"]]
    if c["kind"] == "rotary":
        n = c["batch"] * c["seq"] * (c["heads"] + c["kv_heads"])
        return {"bytes": 2 * e * n * c["d"] + 4 * c["batch"] * c["seq"], "flops": 3 * n * c["rot"]}
    pairs = _visible_pairs(c)
    if c["kind"] in ("tree", "step"):
        rows = sum(_cache_lengths(c)) + c["batch"] * c["n"]
        q = c["batch"] * c["n"] * c["heads"] * c["d"]
        kv = rows * c["kv_heads"] * c["d"]
        new = 2 * c["batch"] * c["n"] * c["kv_heads"] * c["d"] if c["kind"] == "step" else 0
        return {"bytes": e * (2 * q + 2 * kv + new), "flops": 4 * c["d"] * pairs * c["heads"]}
    q = c["batch"] * c["heads"] * c["sq"] * c["d"]
    kv = c["batch"] * c["kv_heads"] * c["sk"] * c["d"]
    if c["kind"] == "score":
        return {"bytes": e * (2 * q + 2 * kv), "flops": 4 * c["d"] * pairs * c["heads"]}
    return {"bytes": e * (4 * q + 4 * kv), "flops": 14 * c["d"] * pairs * c["heads"]}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _tensor(g, c, heads, seq, sigma=1.0, layout="bhsd"):
    """[batch, heads, seq, d] as seen, stored in the case's layout."""
    shape = (c["batch"], heads, seq, c["d"]) if layout == "bhsd" else (c["batch"], seq, heads, c["d"])
    x = (torch.randn(shape, device="cuda", generator=g) * sigma).to(_TORCH[c["dtype"]])
    return x if layout == "bhsd" else x.transpose(1, 2)


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _score_inputs(c, seed):
    g = _generator(seed)
    lay = c["layout"]
    s = {"q": _tensor(g, c, c["heads"], c["sq"], c["sigma"], lay),
         "k": _tensor(g, c, c["kv_heads"], c["sk"], c["sigma"], lay),
         "v": _tensor(g, c, c["kv_heads"], c["sk"], 1.0, lay)}
    if c["kind"] == "train":
        s["dout"] = _tensor(g, c, c["heads"], c["sq"], 1.0, lay)
    s["slopes"] = torch.tensor(_slopes(c["heads"]), device="cuda") if c["alibi"] else None
    s["docs"] = _int32(_doc_ids(c)) if c["docs"] else None
    s["prefix"] = _int32(_prefixes(c)) if c["prefix"] else None
    return s


def _rotary_inputs(c, seed):
    g = _generator(seed)
    pos = torch.arange(c["seq"], device="cuda", dtype=torch.int32)[None, :].repeat(c["batch"], 1) + c["start"]
    return {"q": _tensor(g, c, c["heads"], c["seq"], 1.0, c["layout"]),
            "k": _tensor(g, c, c["kv_heads"], c["seq"], 1.0, c["layout"]), "pos": pos}


def _tree_inputs(c, seed):
    """The cache holds capacity rows a sequence, in pages of a common pool (page > 0) or one after another."""
    g = _generator(seed)
    lens = _cache_lengths(c)
    cap = max(lens) + c["n"]
    t = _TORCH[c["dtype"]]
    s = {"q": _tensor(g, c, c["heads"], c["n"])}
    if c["page"]:
        per = -(-cap // c["page"])
        order = np.random.default_rng(seed).permutation(c["batch"] * per).reshape(c["batch"], per)
        s["table"] = _int32(order.tolist())
        shape = (c["batch"] * per, c["page"], c["kv_heads"], c["d"])
    else:
        s["table"] = None
        shape = (c["batch"], cap, c["kv_heads"], c["d"])
    s["kcache"] = torch.randn(shape, device="cuda", generator=g).to(t)
    s["vcache"] = torch.randn(shape, device="cuda", generator=g).to(t)
    if c["kind"] == "step":
        s["knew"] = _tensor(g, c, c["kv_heads"], c["n"])
        s["vnew"] = _tensor(g, c, c["kv_heads"], c["n"])
    trees = [_ancestors(c, b) for b in range(c["batch"])]
    s["lens"] = _int32(lens)
    s["pos"] = _int32([[n + d for d in depth] for n, (_, depth) in zip(lens, trees)])
    s["seen"] = torch.tensor(np.stack([v for v, _ in trees]), device="cuda")
    words = -(-c["n"] // 64)
    bits = np.zeros((c["batch"], c["n"], words * 64), dtype=np.uint64)
    bits[:, :, :c["n"]] = np.stack([v for v, _ in trees])
    packed = (bits.reshape(c["batch"], c["n"], words, 64) << np.arange(64, dtype=np.uint64)).sum(axis=-1,
                                                                                                dtype=np.uint64)
    s["mask"] = torch.from_numpy(packed.view(np.int64)).cuda()
    s["slopes"] = torch.tensor(_slopes(c["heads"]), device="cuda") if c["alibi"] else None
    return s


_INPUTS = {"score": _score_inputs, "train": _score_inputs, "rotary": _rotary_inputs, "tree": _tree_inputs,
           "step": _tree_inputs}
# Rotary tables of the cases: base, and the scaling's factor over an original length
_ROT_BASE = 10000.0
_ROT_FACTOR = 8.0
_ROT_LEN = 4096


def _strides(x):
    """Element strides of a [batch, heads, seq, d] view as (batch, seq, head)."""
    return (x.stride(0), x.stride(2), x.stride(1))


def prepare(case, seed):
    c = case
    s = _INPUTS[c["kind"]](c, seed)
    s["case"] = c
    s["host_lens"] = _cache_lengths(c) if c["kind"] in ("tree", "step") else None
    if not own:
        return s
    fa = _fa()
    fa.init()
    dtype = {"f32": fa.DTYPE_F32, "bf16": fa.DTYPE_BF16, "f16": fa.DTYPE_F16}[c["dtype"]]

    def ptr(x):
        return 0 if x is None else x.data_ptr()

    if c["kind"] in ("score", "train"):
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(c["batch"], c["heads"], c["sq"], device="cuda")
        strides = {x: _strides(s[x]) for x in ("q", "k", "v", "out")}
        if c["kind"] == "train":
            for x in ("q", "k", "v"):
                s["d" + x] = torch.empty_like(s[x])
            strides.update({x: _strides(s[x]) for x in ("dout", "dq", "dk", "dv")})
        s["cfg"] = fa.score_config(dtype, c["batch"], c["heads"], c["kv_heads"], c["sq"], c["sk"], c["d"],
                                   causal=c["causal"], softcap=c["softcap"], q_start=_positions_of_queries(c),
                                   slopes_ptr=ptr(s["slopes"]), q_doc_ptr=ptr(s["docs"]), k_doc_ptr=ptr(s["docs"]),
                                   prefix_ptr=ptr(s["prefix"]), strides=strides)
        return s
    if c["kind"] in ("rotary", "step"):
        scaling = {"none": fa.ROTARY_NONE, "linear": fa.ROTARY_LINEAR, "ntk": fa.ROTARY_NTK,
                   "yarn": fa.ROTARY_YARN}[c.get("scaling", "none")]
        rot = fa.rotary_config(dtype, c["d"], c["rot"], interleaved=c.get("interleaved", False), base=_ROT_BASE,
                               scaling=scaling, factor=_ROT_FACTOR, original_len=_ROT_LEN)
        s["rot"] = rot
    if c["kind"] == "rotary":
        s["qout"], s["kout"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        s["qt"] = fa.rotary_tensor(c["heads"], _strides(s["q"]), _strides(s["qout"]))
        s["kt"] = fa.rotary_tensor(c["kv_heads"], _strides(s["k"]), _strides(s["kout"]))
        return s
    kc, vc = s["kcache"], s["vcache"]
    s["cache"] = fa.kv_cache(dtype, c["batch"], c["kv_heads"], c["d"], kc.data_ptr(), vc.data_ptr(),
                             k_strides=(kc.stride(0), kc.stride(1), kc.stride(2)),
                             v_strides=(vc.stride(0), vc.stride(1), vc.stride(2)), lens_ptr=s["lens"].data_ptr(),
                             capacity=0 if c["page"] else kc.shape[1], block_table_ptr=ptr(s["table"]),
                             page_size=c["page"], n_pages=kc.shape[0] if c["page"] else 0,
                             pages_per_seq=s["table"].shape[1] if c["page"] else 0)
    s["out"] = torch.empty_like(s["q"])
    s["cfg"] = fa.tree_config(c["heads"], c["n"], mask_ptr=s["mask"].data_ptr(), softcap=c["softcap"],
                              slopes_ptr=ptr(s["slopes"]), positions_ptr=s["pos"].data_ptr())
    if c["kind"] == "step":
        s["qrot"] = torch.empty_like(s["q"])
        s["append"] = fa.append_config(c["n"], rotary=s["rot"], k_strides=_strides(s["knew"]),
                                       v_strides=_strides(s["vnew"]),
                                       q_layout=fa.rotary_tensor(c["heads"], _strides(s["q"]), _strides(s["qrot"])))
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    c = state["case"]
    if own:
        return _run_own(state)
    if c["kind"] in ("score", "train"):
        return _plain_score(state)
    if c["kind"] == "rotary":
        q = _plain_rotary(state["q"], state["pos"], c, c["inverse"])
        return {"q": q, "k": _plain_rotary(state["k"], state["pos"], c, c["inverse"])}
    return _plain_tree(state)


def _run_own(s):
    c, fa = s["case"], _fa()
    stream = torch.cuda.current_stream().cuda_stream
    if c["kind"] in ("score", "train"):
        q, k, v = s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr()
        fa.score_attention_device(s["cfg"], q, k, v, s["out"].data_ptr(), s["lse"].data_ptr(), stream)
        if c["kind"] == "score":
            return {"out": s["out"], "lse": s["lse"]}
        fa.score_attention_backward_device(s["cfg"], q, k, v, s["out"].data_ptr(), s["lse"].data_ptr(),
                                           s["dout"].data_ptr(), s["dq"].data_ptr(), s["dk"].data_ptr(),
                                           s["dv"].data_ptr(), stream)
        return {"out": s["out"], "lse": s["lse"], "dq": s["dq"], "dk": s["dk"], "dv": s["dv"]}
    if c["kind"] == "rotary":
        fa.rotary_device(s["rot"], c["batch"], c["seq"], s["pos"].data_ptr(), s["qt"], s["q"].data_ptr(),
                         s["qout"].data_ptr(), s["kt"], s["k"].data_ptr(), s["kout"].data_ptr(), stream,
                         inverse=c["inverse"])
        return {"q": s["qout"], "k": s["kout"]}
    if c["kind"] == "tree":
        fa.tree_attention_device(s["cfg"], s["cache"], s["q"].data_ptr(), s["out"].data_ptr(), stream=stream)
        return {"out": s["out"]}
    pos = s["pos"].data_ptr()
    fa.cache_append_device(s["cache"], s["append"], s["knew"].data_ptr(), s["vnew"].data_ptr(), pos,
                           s["q"].data_ptr(), s["qrot"].data_ptr(), stream=stream)
    fa.tree_attention_device(s["cfg"], s["cache"], s["qrot"].data_ptr(), s["out"].data_ptr(), stream=stream)
    return {"out": s["out"], "k": s["kcache"], "v": s["vcache"]}


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


def _plain_score(state):
    c, train = state["case"], state["case"]["kind"] == "train"
    q, k, v, slopes = state["q"], state["k"], state["v"], state["slopes"]
    group, scale, cap, start = c["heads"] // c["kv_heads"], c["d"] ** -0.5, c["softcap"], _positions_of_queries(c)
    qpos = torch.arange(c["sq"], device="cuda") + start
    kpos = torch.arange(c["sk"], device="cuda")
    lse = torch.empty(c["batch"], c["heads"], c["sq"], device="cuda")
    res = {"out": torch.empty_like(q), "lse": lse}
    if train:
        res.update(dq=torch.empty_like(q), dk=torch.empty_like(k), dv=torch.empty_like(v))
    for b in range(c["batch"]):
        seen = torch.ones(c["sq"], c["sk"], dtype=torch.bool, device="cuda")
        if c["causal"]:
            seen = kpos[None, :] <= qpos[:, None]
            if c["prefix"]:
                seen = seen | (kpos < state["prefix"][b])[None, :]
        if c["docs"]:
            ids = state["docs"][b]
            seen = seen & (ids[:, None] == ids[None, :]) & (ids >= 0)[:, None]
        distance = (qpos[:, None] - kpos[None, :]).abs().float() if c["alibi"] else None
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


def _plain_frequencies(rot, scaling):
    """Angle a position of each column pair (64 bits) and the factor on the rotated values."""
    i = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda")
    base = _ROT_BASE
    if scaling == "ntk":
        base = base * _ROT_FACTOR ** (rot / (rot - 2))
    f = base ** (-i / rot)
    if scaling == "linear":
        f = f / _ROT_FACTOR
    if scaling != "yarn":
        return f, 1.0
    # YaRN: pairs that turn more than 32 times over the trained length keep their angle, those
    # below one turn are interpolated, a ramp over the pair's index lies between
    def pair(turns):
        return rot * math.log(_ROT_LEN / (turns * 2 * math.pi)) / (2 * math.log(_ROT_BASE))
    lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot - 1)
    ramp = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
    return f / _ROT_FACTOR * ramp + f * (1.0 - ramp), 0.1 * math.log(_ROT_FACTOR) + 1.0


def _plain_rotary(x, pos, c, inverse=False):
    """x: [batch, heads, seq, d], pos: [batch, seq]."""
    rot = c["rot"]
    f, m = _plain_frequencies(rot, c.get("scaling", "none"))
    angle = pos.double()[:, None, :, None] * f   # far positions: 32 bits lose the angle
    cos, sin = torch.cos(angle).float() * m, torch.sin(angle).float() * (-m if inverse else m)
    xf = x.float()
    out = xf.clone()
    if c.get("interleaved", False):
        a, b = xf[..., 0:rot:2], xf[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = xf[..., :rot // 2], xf[..., rot // 2:rot]
        out[..., :rot // 2], out[..., rot // 2:rot] = a * cos - b * sin, a * sin + b * cos
    return out.to(x.dtype)


def _plain_tree(state):
    c, q = state["case"], state["q"]
    kc, vc, group, cap = state["kcache"], state["vcache"], c["heads"] // c["kv_heads"], c["softcap"]
    n = c["n"]
    if c["kind"] == "step":
        q = _plain_rotary(q, state["pos"], c)
        knew = _plain_rotary(state["knew"], state["pos"], c)
    res = {"out": torch.empty_like(state["q"])}
    for b, length in enumerate(state["host_lens"]):
        rows = torch.arange(length + n, device="cuda")
        if c["page"]:
            at = (state["table"][b].long()[rows // c["page"]], rows % c["page"])
        else:
            at = (torch.full_like(rows, b), rows)
        if c["kind"] == "step":
            kc[at[0][length:], at[1][length:]] = knew[b].transpose(0, 1)
            vc[at[0][length:], at[1][length:]] = state["vnew"][b].transpose(0, 1)
        kf = kc[at[0], at[1]].float().permute(1, 2, 0).contiguous()   # [kv_heads, d, keys]
        vf = vc[at[0], at[1]].float().transpose(0, 1).contiguous()
        qf = q[b].float().reshape(c["kv_heads"], group * n, c["d"])
        s = torch.matmul(qf, kf).reshape(c["heads"], n, length + n) * c["d"] ** -0.5
        if cap:
            s = cap * torch.tanh(s / cap)
        if c["alibi"]:
            kpos = torch.cat((rows[:length], state["pos"][b].long()))
            s = s - state["slopes"][:, None, None] * (state["pos"][b].long()[:, None] - kpos[None, :]).abs().float()
        seen = torch.cat((torch.ones(n, length, dtype=torch.bool, device="cuda"), state["seen"][b]), dim=1)
        p, _ = _plain_softmax(s, seen)
        o = torch.matmul(p.reshape(c["kv_heads"], group * n, length + n), vf)
        res["out"][b] = o.reshape(c["heads"], n, c["d"]).to(q.dtype)
    if c["kind"] == "step":
        res.update(k=kc, v=vc)
    return res


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = _INPUTS[case["kind"]](case, seed)
    if case["kind"] in ("score", "train"):
        return _exact_score(case, s)
    if case["kind"] == "rotary":
        sign = -1.0 if case["inverse"] else 1.0
        return {x: _exact_rotary(case, s[x], s["pos"], sign) for x in ("q", "k")}
    return _exact_tree(case, s)


def _exact_weights(z, hidden):
    """softmax over the keys that are not hidden, and its log-sum; a row of hidden keys has weight nowhere."""
    z = torch.where(hidden, torch.full_like(z, -math.inf), z)
    lse = torch.logsumexp(z, dim=-1)
    return torch.exp(z - lse[..., None]).nan_to_num_(0.0), lse


def _exact_score(c, s):
    dev = s["q"].device
    i = torch.arange(c["sq"], device=dev)[:, None] + (c["sk"] - 1 if c["sq"] == 1 else 0)
    j = torch.arange(c["sk"], device=dev)[None, :]
    per = c["heads"] // c["kv_heads"]
    o = {"out": torch.empty(s["q"].shape, dtype=torch.float64, device=dev),
         "lse": torch.empty(c["batch"], c["heads"], c["sq"], dtype=torch.float64, device=dev)}
    if c["kind"] == "train":
        for x in ("q", "k", "v"):
            o["d" + x] = torch.zeros(s[x].shape, dtype=torch.float64, device=dev)
    for b in range(c["batch"]):
        hidden = torch.zeros(c["sq"], c["sk"], dtype=torch.bool, device=dev)
        if c["causal"]:
            hidden |= (j > i) & (j >= (int(s["prefix"][b]) if c["prefix"] else 0))
        if c["docs"]:
            own_doc = s["docs"][b]
            hidden |= (own_doc[:, None] != own_doc[None, :]) | (own_doc < 0)[None, :]
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
            if c["kind"] == "train":
                dO = s["dout"][b, h].double()
                o["dv"][b, h // per] += P.t().contiguous() @ dO
                dP = dO @ V.t().contiguous()
                dX = P * (dP - (P * dP).sum(-1, keepdim=True)) * slope / math.sqrt(c["d"])
                o["dq"][b, h] = dX @ K
                o["dk"][b, h // per] += dX.t().contiguous() @ Q
    return o


def _exact_rotary(c, x, pos, sign=1.0):
    rot, half = c["rot"], c["rot"] // 2
    kind = c.get("scaling", "none")
    freq, gain = [], 1.0
    for p in range(half):
        w = _ROT_BASE ** (-2.0 * p / rot)
        if kind == "linear":
            w /= _ROT_FACTOR
        elif kind == "ntk":
            w = (_ROT_BASE * _ROT_FACTOR ** (rot / (rot - 2.0))) ** (-2.0 * p / rot)
        elif kind == "yarn":
            def index(turns):
                return rot * math.log(_ROT_LEN / (2.0 * math.pi * turns)) / (2.0 * math.log(_ROT_BASE))
            first, last = max(0, math.floor(index(32.0))), min(rot - 1, math.ceil(index(1.0)))
            part = min(1.0, max(0.0, (p - first) / max(0.001, last - first)))
            w = part * w / _ROT_FACTOR + (1.0 - part) * w
            gain = 1.0 + 0.1 * math.log(_ROT_FACTOR)
        freq.append(w)
    t = sign * pos.double()[:, None, :, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.full_like(t, gain), t)
    y = x.double()
    if c.get("interleaved", False):
        z = torch.complex(y[..., 0:rot:2].contiguous(), y[..., 1:rot:2].contiguous()) * turn
        head = torch.stack((z.real, z.imag), dim=-1).flatten(-2)
    else:
        z = torch.complex(y[..., :half].contiguous(), y[..., half:rot].contiguous()) * turn
        head = torch.cat((z.real, z.imag), dim=-1)
    return torch.cat((head, y[..., rot:]), dim=-1)


def _exact_tree(c, s):
    dev, n, per = s["q"].device, c["n"], c["heads"] // c["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=dev)
    q = s["q"].double()
    kcache, vcache = s["kcache"], s["vcache"]
    if c["kind"] == "step":
        # the cache and the queries hold the rounded rotated values
        q = _exact_rotary(c, s["q"], s["pos"]).to(s["q"].dtype).double()
        knew = _exact_rotary(c, s["knew"], s["pos"])
        kcache, vcache = kcache.double(), vcache.double()
    for b, length in enumerate(_cache_lengths(c)):
        place = []
        for r in range(length + n):
            place.append((int(r // c["page"]), r % c["page"]) if c["page"] else (b, r))
        page = torch.tensor([p for p, _ in place], device=dev)
        if c["page"]:
            page = s["table"][b].long()[page]
        row = torch.tensor([r for _, r in place], device=dev)
        if c["kind"] == "step":
            kcache[page[length:], row[length:]] = knew[b].transpose(0, 1)
            vcache[page[length:], row[length:]] = s["vnew"][b].double().transpose(0, 1)
        hidden = torch.zeros(n, length + n, dtype=torch.bool, device=dev)
        hidden[:, length:] = ~s["seen"][b]
        for h in range(c["heads"]):
            K, V = kcache[page, row, h // per], vcache[page, row, h // per]
            if c["kind"] == "step":
                K = K.to(s["q"].dtype)
            x = (q[b, h] @ K.double().t().contiguous()) / math.sqrt(c["d"])
            if c["softcap"]:
                x = c["softcap"] * torch.tanh(x / c["softcap"])
            if c["alibi"]:
                at = torch.cat((torch.arange(length, device=dev), s["pos"][b].long()))
                x = x - float(s["slopes"][h]) * (s["pos"][b].long()[:, None] - at[None, :]).abs().double()
            out[b, h] = _exact_weights(x, hidden)[0] @ V.double()
    if c["kind"] == "step":
        return {"out": out, "k": kcache, "v": vcache}
    return {"out": out}
