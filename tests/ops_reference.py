"""The score, tree and rotary operators in float64 on the CPU, with the bounds that their tests use.

``score_case`` computes output, log-sums and gradients of one call and, for
each, how far a kernel may be off: u is half a step of the type (one rounding,
relative), every f32 operation is within 2^-24, and

  z error    an f32 dot product of d terms in any order and a few operations
             on the score: (d + 8) 2^-24 sum |q||k| scale, plus the rounding of the exponent's
             argument (2^-23 of the largest |z|, twice) and 4e-7 of the cap
  weights    2 e_z relatively (the row's sum moves too), u where they are
             rounded for a product, and 2^-25 absolutely where f16 has subnormals
             (forward: of weights taken 2^7 times larger)
  sums       n terms in f32: n 2^-24 of the sum of absolute values
"""
from __future__ import annotations

import math

import torch

EPS32 = 2.0 ** -24


def unit(dtype):
    """Half a step of the type, relative to the value (bf16 2^-8, f16 2^-11, f32 2^-24)."""
    return torch.finfo(dtype).eps / 2


def visible(sq, sk, causal, q_start=0, prefix=None, q_doc=None, k_doc=None):
    i = torch.arange(sq)[:, None] + q_start
    j = torch.arange(sk)[None, :]
    see = torch.ones(sq, sk, dtype=torch.bool)
    if causal:
        see = j <= i
        if prefix is not None:
            see = see | (j < prefix)
    if q_doc is not None:
        see = see & (q_doc[:, None] == k_doc[None, :]) & (q_doc >= 0)[:, None]
    return see


def attend(q, k, v, see, scale, cap=0.0, bias=None, dtype=torch.float32, dout=None):
    """One head in float64: a dict of (value, bound) for out, lse and, with dout, dq, dk, dv."""
    u = 0.0 if dtype == torch.float32 else unit(dtype)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    q, k, v = q.double(), k.double(), v.double()
    n, m, d = q.shape[0], k.shape[0], q.shape[1]
    x = q @ k.T * scale
    ez = (d + 8) * EPS32 * (q.abs() @ k.abs().T) * scale
    t = torch.tanh(x / cap) if cap else torch.zeros_like(x)
    y = cap * t if cap else x
    z = y if bias is None else y + bias
    ez = ez + 2 * 2 * EPS32 * (z.abs() + (0 if bias is None else bias.abs()) + 16) + 4e-7 * cap
    # errors of scores below the row's maximum by more than 40 do not matter: their weight is 0 to f32
    z = torch.where(see, z, torch.full_like(z, -math.inf))
    ez = torch.where(see, ez, torch.zeros_like(ez))
    lse = torch.logsumexp(z, dim=1)
    empty = torch.isinf(lse)
    p = torch.where(see, torch.exp(z - torch.where(empty, torch.zeros_like(lse), lse)[:, None]), torch.zeros_like(z))
    rowe = (p * ez).sum(1)   # error of lse
    elz = rowe + 4 * EPS32 * (lse.nan_to_num(0, 0, 0).abs() + 16) + m * EPS32
    out = p @ v
    ep = p * (ez + elz[:, None])
    eo = (ep + p * u + tiny / 64) @ v.abs() + (m + 4) * EPS32 * (p @ v.abs())
    res = {"out": (out, eo + unit(dtype) * (out.abs() + eo) + tiny), "lse": (lse, elz)}
    if dout is None:
        return res
    do = dout.double()
    delta = (do * out).sum(1)
    # O enters delta rounded to the type
    edelta = (do.abs() * (eo + unit(dtype) * (out.abs() + eo) + tiny)).sum(1) + d * EPS32 * (do.abs() * out.abs()).sum(1)
    dp = do @ v.T
    edp = (d + 4) * EPS32 * (do.abs() @ v.abs().T)
    slope = 1 - t * t
    eslope = 2 * (ez / cap + 3e-7) if cap else torch.zeros_like(x)
    ds = p * (dp - delta[:, None]) * slope
    eds = (ep * (dp - delta[:, None]).abs() + p * (edp + edelta[:, None])) * slope + p * (dp - delta[:, None]).abs() * eslope
    eds = eds + 4 * EPS32 * ds.abs()
    eds = eds + u * (ds.abs() + eds) + tiny
    eds = torch.where(see, eds, torch.zeros_like(eds))
    dv = p.T @ do
    edv = (ep + u * p + tiny * see).T @ do.abs() + (n + 4) * EPS32 * (p.T @ do.abs())
    dq = ds @ k * scale
    edq = (eds @ k.abs() + (m + 4) * EPS32 * (ds.abs() @ k.abs())) * scale
    dk = ds.T @ q * scale
    edk = (eds.T @ q.abs() + (n + 4) * EPS32 * (ds.abs().T @ q.abs())) * scale
    # left unrounded: the heads of a group are added before the rounding
    res.update(dq=(dq, edq), dk=(dk, edk), dv=(dv, edv))
    return res


def round_bound(value, bound, dtype):
    """Bound of a sum that is rounded to the type at its end."""
    return bound + unit(dtype) * (value.abs() + bound) + (2.0 ** -25 if dtype == torch.float16 else 0.0) + 1e-37


def check(name, got, value, bound):
    """got within bound of value, infinities and NaN in the same places."""
    got = got.double().cpu()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    special = ~torch.isfinite(value)
    assert torch.equal(torch.isnan(got), torch.isnan(value)), f"{name}: NaN in other places"
    same = torch.where(torch.isnan(value), torch.zeros_like(value), value)
    assert torch.equal(got[special & ~torch.isnan(value)], same[special & ~torch.isnan(value)]), f"{name}: infinities"
    err = torch.where(special, torch.zeros_like(value), (got - value).abs())
    worst = (err / bound.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3g} of its bound (largest error {err.max().item():.3g})"
    return worst
