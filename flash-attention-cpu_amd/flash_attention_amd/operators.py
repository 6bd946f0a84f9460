"""Attention with modified scores, rotary positions and the key / value cache.

Python view of the fa_score_*, fa_rotary*, fa_cache_append and
fa_tree_attention entry points of include/fa_hip.h, which defines what they
compute.  They have no counterpart in the reference crate.

Calls take raw device pointers and a HIP stream, as attention_device does,
and return when queued.  What does not change from call to call -- sizes,
layouts, masks, tables -- is in config objects that a program makes once and
keeps; they hold the pointers they are given, not the memory behind them, so
the tensors of masks, slopes, lengths and caches have to outlive them.
Strides are (batch, token, head) element strides; None means contiguous.
"""
from __future__ import annotations

import ctypes

_P = ctypes.c_void_p
_SZ = ctypes.c_size_t
_I = ctypes.c_int
_F = ctypes.c_float


class Strides(ctypes.Structure):
    """fa_strides: element strides between batches, tokens and heads."""

    _fields_ = [("batch", ctypes.c_int64), ("seq", ctypes.c_int64), ("head", ctypes.c_int64)]


class ScoreConfig(ctypes.Structure):
    """fa_score_config."""

    _fields_ = [("dtype", _I), ("causal", _I), ("batch", _SZ), ("heads", _SZ), ("kv_heads", _SZ), ("seq_len_q", _SZ),
                ("seq_len_k", _SZ), ("d_head", _SZ), ("q_start", ctypes.c_int64), ("softmax_scale", _F),
                ("softcap", _F), ("slopes", _P), ("q_doc", _P), ("k_doc", _P), ("prefix", _P),
                *((n, Strides) for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"))]


class RotaryConfig(ctypes.Structure):
    """fa_rotary_config; turns and gain may be overwritten with another scheme's."""

    _fields_ = [("dtype", _I), ("interleaved", _I), ("d_head", _SZ), ("rot_dim", _SZ), ("gain", _F),
                ("turns", ctypes.c_double * 128)]


class RotaryTensor(ctypes.Structure):
    """fa_rotary_tensor."""

    _fields_ = [("heads", _SZ), ("src", Strides), ("dst", Strides)]


class KvCache(ctypes.Structure):
    """fa_kv_cache."""

    _fields_ = [("dtype", _I), ("batch", _SZ), ("kv_heads", _SZ), ("d_head", _SZ), ("k", _P), ("v", _P),
                ("k_strides", Strides), ("v_strides", Strides), ("lens", _P), ("capacity", _SZ), ("block_table", _P),
                ("page_size", _SZ), ("n_pages", _SZ), ("pages_per_seq", _SZ)]


class AppendConfig(ctypes.Structure):
    """fa_append_config."""

    _fields_ = [("n_tokens", _SZ), ("k", Strides), ("v", Strides), ("rotary", ctypes.POINTER(RotaryConfig)),
                ("q_layout", ctypes.POINTER(RotaryTensor))]


class TreeConfig(ctypes.Structure):
    """fa_tree_config."""

    _fields_ = [("heads", _SZ), ("n_tokens", _SZ), ("softmax_scale", _F), ("softcap", _F), ("slopes", _P),
                ("positions", _P), ("mask", _P), ("mask_shared", _I), ("q", Strides), ("out", Strides)]


def declare(lib: ctypes.CDLL) -> None:
    """Argument types of the operators' entry points."""
    ptr = ctypes.POINTER
    for name, args in {
        "fa_score_forward": [_P, ptr(ScoreConfig), _P, _P, _P, _P, _P],
        "fa_score_backward": [_P, ptr(ScoreConfig)] + [_P] * 9,
        "fa_rotary_init": [ptr(RotaryConfig), _I, _SZ, _SZ, _I, ctypes.c_double, _I, ctypes.c_double,
                           ctypes.c_double],
        "fa_rotary": [_P, ptr(RotaryConfig), _SZ, _SZ, _P, _I, ptr(RotaryTensor), _P, _P, ptr(RotaryTensor), _P, _P],
        "fa_cache_append": [_P, ptr(KvCache), ptr(AppendConfig), _P, _P, _P, _P, _P],
        "fa_tree_attention": [_P, ptr(TreeConfig), ptr(KvCache), _P, _P, _P],
    }.items():
        f = getattr(lib, name, None)   # None: a library built before there were operators
        if f is not None:
            f.argtypes = args
            f.restype = _I


def _lib():
    global _lib
    from . import lib
    loaded = lib()
    if not hasattr(loaded, "fa_score_forward"):
        from . import FA_ERR_MODULE, LIB_PATH, FaError
        raise FaError(FA_ERR_MODULE, f"{LIB_PATH} has no operators; build it anew with flash-attention-cpu_amd/build.py")

    def known():
        return loaded
    _lib = known
    return loaded


def _check(status: int) -> None:
    if status:
        from . import _check as check
        check(status)


def _strides(s) -> Strides:
    return Strides() if s is None else Strides(*(int(x) for x in s))


def _ptr(x):
    return int(x) or None


def score_config(dtype: int, batch: int, heads: int, kv_heads: int, seq_len_q: int, seq_len_k: int, d_head: int,
                 causal: bool = False, softmax_scale: float | None = None, softcap: float = 0.0, q_start: int = 0,
                 slopes_ptr: int = 0, q_doc_ptr: int = 0, k_doc_ptr: int = 0, prefix_ptr: int = 0,
                 strides: dict | None = None) -> ScoreConfig:
    """What a layer's score attention is made of.  strides: layouts of q, k, v,
    out, dout, dq, dk, dv, those that are not contiguous [batch, heads, seq, d]."""
    strides = strides or {}
    unknown = set(strides) - {"q", "k", "v", "out", "dout", "dq", "dk", "dv"}
    if unknown:
        raise ValueError(f"strides of unknown tensors: {sorted(unknown)}")
    c = ScoreConfig(int(dtype), 1 if causal else 0, batch, heads, kv_heads, seq_len_q, seq_len_k, d_head, int(q_start),
                    float(softmax_scale or 0.0), float(softcap), _ptr(slopes_ptr), _ptr(q_doc_ptr), _ptr(k_doc_ptr),
                    _ptr(prefix_ptr))
    for name, s in strides.items():
        setattr(c, name, _strides(s))
    return c


def score_attention_device(cfg: ScoreConfig, q_ptr: int, k_ptr: int, v_ptr: int, out_ptr: int, lse_ptr: int = 0,
                           stream: int = 0) -> None:
    """Queue softmax attention with modified scores (fa_score_forward)."""
    _check(_lib().fa_score_forward(stream, cfg, q_ptr, k_ptr, v_ptr, out_ptr, lse_ptr))


def score_attention_backward_device(cfg: ScoreConfig, q_ptr: int, k_ptr: int, v_ptr: int, out_ptr: int, lse_ptr: int,
                                    dout_ptr: int, dq_ptr: int, dk_ptr: int, dv_ptr: int, stream: int = 0) -> None:
    """Queue its gradients (fa_score_backward); out and lse are the forward's.  A
    gradient whose pointer is 0 is not computed."""
    _check(_lib().fa_score_backward(stream, cfg, q_ptr, k_ptr, v_ptr, out_ptr, lse_ptr, dout_ptr, dq_ptr, dk_ptr,
                                    dv_ptr))


def rotary_config(dtype: int, d_head: int, rot_dim: int | None = None, interleaved: bool = False,
                  base: float = 10000.0, scaling: int = 0, factor: float = 1.0,
                  original_len: float = 0.0) -> RotaryConfig:
    """Angles of a rotary scheme (fa_rotary_init); scaling: ROTARY_NONE, _LINEAR, _NTK or _YARN."""
    c = RotaryConfig()
    _check(_lib().fa_rotary_init(c, int(dtype), d_head, d_head if rot_dim is None else rot_dim, 1 if interleaved else 0,
                                 float(base), int(scaling), float(factor), float(original_len)))
    return c


def rotary_tensor(heads: int, in_strides=None, out_strides=None) -> RotaryTensor:
    """Head rows a token and layouts of one tensor of a rotary call."""
    return RotaryTensor(heads, _strides(in_strides), _strides(out_strides))


def rotary_device(cfg: RotaryConfig, batch: int, seq_len: int, positions_ptr: int, q_layout: RotaryTensor, q_ptr: int,
                  q_out_ptr: int, k_layout: RotaryTensor | None = None, k_ptr: int = 0, k_out_ptr: int = 0,
                  stream: int = 0, inverse: bool = False) -> None:
    """Queue rotary positions of one or two tensors (fa_rotary); inverse: their gradients."""
    _check(_lib().fa_rotary(stream, cfg, batch, seq_len, positions_ptr, 1 if inverse else 0, q_layout, q_ptr,
                            q_out_ptr, k_layout, k_ptr, k_out_ptr))


def kv_cache(dtype: int, batch: int, kv_heads: int, d_head: int, k_ptr: int, v_ptr: int, lens_ptr: int,
             k_strides=None, v_strides=None, capacity: int = 0, block_table_ptr: int = 0, page_size: int = 0,
             n_pages: int = 0, pages_per_seq: int = 0) -> KvCache:
    """A cache of capacity rows a sequence, or (block_table_ptr) in pages."""
    return KvCache(int(dtype), batch, kv_heads, d_head, _ptr(k_ptr), _ptr(v_ptr), _strides(k_strides),
                   _strides(v_strides), _ptr(lens_ptr), capacity, _ptr(block_table_ptr), page_size, n_pages,
                   pages_per_seq)


def append_config(n_tokens: int, rotary: RotaryConfig | None = None, k_strides=None, v_strides=None,
                  q_layout: RotaryTensor | None = None) -> AppendConfig:
    """An append of n tokens a sequence; rotary: keys (and queries, with q_layout) are rotated on the way."""
    c = AppendConfig(n_tokens, _strides(k_strides), _strides(v_strides))
    if rotary is not None:
        c.rotary = ctypes.pointer(rotary)
    if q_layout is not None:
        c.q_layout = ctypes.pointer(q_layout)
    return c


def cache_append_device(cache: KvCache, cfg: AppendConfig, k_ptr: int, v_ptr: int, positions_ptr: int = 0,
                        q_ptr: int = 0, q_out_ptr: int = 0, stream: int = 0) -> None:
    """Queue the append of drafted keys and values behind each sequence's rows (fa_cache_append)."""
    _check(_lib().fa_cache_append(stream, cache, cfg, k_ptr, v_ptr, positions_ptr, q_ptr, q_out_ptr))


def tree_config(heads: int, n_tokens: int, mask_ptr: int = 0, mask_shared: bool = False,
                softmax_scale: float | None = None, softcap: float = 0.0, slopes_ptr: int = 0, positions_ptr: int = 0,
                q_strides=None, out_strides=None) -> TreeConfig:
    """Attention of n drafted tokens; no mask: a chain, each token sees itself and those before it."""
    return TreeConfig(heads, n_tokens, float(softmax_scale or 0.0), float(softcap), _ptr(slopes_ptr),
                      _ptr(positions_ptr), _ptr(mask_ptr), 1 if mask_shared else 0, _strides(q_strides),
                      _strides(out_strides))


def tree_attention_device(cfg: TreeConfig, cache: KvCache, q_ptr: int, out_ptr: int, lse_ptr: int = 0,
                          stream: int = 0) -> None:
    """Queue attention of drafted tokens over the cache (fa_tree_attention)."""
    _check(_lib().fa_tree_attention(stream, cfg, cache, q_ptr, out_ptr, lse_ptr))
