"""Norms and rotary positions of query and key heads (include/hq_rotary.h): what an attention layer does between its
projections (nebula_amd.hq, nebula_amd.decoder) and its scores (nebula_amd.attn).

    rot = Rotary(64, base=1e6, layout="half", scaling=Stretch(4.0, 32768))     # once
    q, k = rotate(q, k, rot, positions, q_weight=wq, k_weight=wk)               # before attn.prompt
    q = cache.append_rotated(layer, rot, q, k, v, rows, cu, q_weight=wq, ...)   # in place of cache.append

Tensors are float16 or bfloat16 [tokens, heads, head_dim] on the GPU, with any row and head strides that are
multiples of 8 elements; the norms' weights float32 [head_dim]. Only the first `dim` elements of a head are
rotated. torch supplies memory and streams only; every computation on the device runs in the HIP library.
"""
from __future__ import annotations

import ctypes
import math
import struct
from dataclasses import dataclass
from typing import Optional

import numpy as np

from . import attn, hq

LAYOUTS = {"half": 1, "interleaved": 2}

# Every symbol include/hq_rotary.h declares.
EXPORTS = ("hq_rotate", "hq_cache_append_rotated")


class RotaryDesc(ctypes.Structure):
    _fields_ = [("turns", ctypes.c_void_p), ("dim", ctypes.c_uint32), ("layout", ctypes.c_int), ("scale", ctypes.c_float)]


class RotaryHeads(ctypes.Structure):
    _fields_ = [("In", ctypes.c_void_p), ("Out", ctypes.c_void_p), ("in_row", ctypes.c_int64), ("in_head", ctypes.c_int64),
                ("out_row", ctypes.c_int64), ("out_head", ctypes.c_int64), ("weight", ctypes.c_void_p), ("heads", ctypes.c_uint32),
                ("eps", ctypes.c_float)]


# hq_rotary_heads as bytes, packed by every call.
_HEADS = struct.Struct("@PPqqqqPIf")
assert _HEADS.size == ctypes.sizeof(RotaryHeads)

_bound: Optional[ctypes.CDLL] = None


def _lib() -> ctypes.CDLL:
    global _bound
    if _bound is not None:
        return _bound
    L = hq.lib()
    u32, i64, vp, i32 = ctypes.c_uint32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_int
    rot, heads, cache = ctypes.POINTER(RotaryDesc), ctypes.c_char_p, ctypes.POINTER(attn.KVCacheDesc)
    for name, types in {"hq_rotate": [rot, heads, heads, u32, u32, i32, vp, vp],
                        "hq_cache_append_rotated": [cache, u32, rot, heads, heads, vp, i64, i64, u32, vp, vp, u32, vp]}.items():
        f = getattr(L, name)
        f.restype, f.argtypes = i32, types
    _bound = L
    return L


# ---------------------------------------------------------------- frequencies
@dataclass(frozen=True)
class Linear:
    """Positions divided by factor."""
    factor: float


@dataclass(frozen=True)
class Base:
    """The base raised so that the slowest pair turns 1 / factor as far: base * factor^(R / (R - 2))."""
    factor: float


@dataclass(frozen=True)
class Stretch:
    """By parts: pairs that turn at least `fast` times within `original` positions keep their frequency, those that turn at
    most `slow` times take positions / factor, a linear ramp over the pairs between them; the rotated part is
    multiplied by `scale` (None: 0.1 log(factor) + 1)."""
    factor: float
    original: int
    fast: float = 32.0
    slow: float = 1.0
    scale: Optional[float] = None


def frequencies(dim: int, base: float = 10000.0, scaling=None):
    """(radians per position of the dim / 2 pairs as float64, factor of the rotated part): base^(-2 i / dim), scaled."""
    if dim < 16 or dim % 16:
        raise ValueError(f"dim={dim} must be a positive multiple of 16")
    if not (base > 0 and math.isfinite(base)):
        raise ValueError(f"base={base} must be positive and finite")
    i = np.arange(dim // 2, dtype=np.float64)
    f = float(base) ** (-2.0 * i / dim)
    if scaling is None:
        return f, 1.0
    s = float(scaling.factor)
    if not (s > 0 and math.isfinite(s)):
        raise ValueError(f"factor={s} must be positive and finite")
    if isinstance(scaling, Linear):
        return f / s, 1.0
    if isinstance(scaling, Base):
        return (float(base) * s ** (dim / (dim - 2))) ** (-2.0 * i / dim), 1.0
    if isinstance(scaling, Stretch):
        if scaling.original < 1 or not scaling.fast > scaling.slow > 0 or base <= 1:
            raise ValueError(f"{scaling}: need original >= 1, fast > slow > 0 and a base above 1 (got {base})")
        pair = lambda turns: dim * math.log(scaling.original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(pair(scaling.fast)), 0), min(math.ceil(pair(scaling.slow)), dim - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        scale = (0.1 * math.log(s) + 1.0 if s > 1 else 1.0) if scaling.scale is None else float(scaling.scale)
        return f / s * ramp + f * (1.0 - ramp), scale
    raise TypeError(f"scaling must be Linear, Base or Stretch, got {scaling!r}")


class Rotary:
    """How heads are rotated: their first dim elements (a multiple of 16), in pairs (i, i + dim / 2), layout "half", or
    (2 i, 2 i + 1), "interleaved", pair i by position * base^(-2 i / dim) radians, scaled by scaling (Linear, Base or
    Stretch). angles, float64 [dim / 2] radians per position, and scale stand for frequencies of the caller's own."""

    def __init__(self, dim: int, base: float = 10000.0, layout: str = "half", scaling=None, angles=None, scale: Optional[float] = None,
                 device="cuda"):
        import torch

        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {tuple(LAYOUTS)}, got {layout!r}")
        f, factor = frequencies(dim, base, scaling)
        if angles is not None:
            f = np.asarray(angles, dtype=np.float64)
            if f.shape != (dim // 2,) or not np.isfinite(f).all():
                raise ValueError(f"angles must be {dim // 2} finite numbers")
        self.dim, self.layout, self.scale = dim, layout, factor if scale is None else float(scale)
        self.turns = torch.from_numpy(f / (2 * math.pi)).to(device)
        self.device_index = self.turns.get_device()
        self._desc = RotaryDesc(self.turns.data_ptr(), dim, LAYOUTS[layout], self.scale)
        self._ref = ctypes.byref(self._desc)


# ---------------------------------------------------------------- calls
def _weight(name: str, w, D: int, dev: int) -> int:
    """Address of a norm's weight (None: 0)."""
    if w is None:
        return 0
    if w.get_device() != dev or w.dtype != (hq._torch or hq._load()).float32 or not w.is_contiguous() or w.numel() != D:
        raise ValueError(f"{name} must be a contiguous float32 tensor of {D} entries on the call's device, got {w.dtype} {tuple(w.shape)} on {w.device}")
    return w.data_ptr()


def _heads(name: str, x, shape, out, weight, eps: float, dev: int) -> bytes:
    """hq_rotary_heads of a tensor that is checked."""
    T, H, D = shape
    row, head, _ = x.stride()
    op = orow = ohead = 0
    if out is not None:
        op = out.data_ptr()
        orow, ohead, _ = out.stride()
        if H == 1:
            ohead = 0
    if T == 1:
        row = orow = 0
    return _HEADS.pack(x.data_ptr(), op, row, head if H > 1 else 0, orow, ohead, 0 if weight is None else _weight(name, weight, D, dev), H, eps)


def _check_heads(name: str, x, shape, dtype, dev: int) -> None:
    if len(shape) != 3 or x.dtype != dtype or x.get_device() != dev or dev < 0:
        raise ValueError(f"{name} must be a {dtype} tensor [tokens, heads, head_dim] on the call's GPU, got {x.dtype} {tuple(shape)} on {x.device}")
    if x.stride()[2] != 1:
        raise ValueError(f"{name} must have unit stride along its last dimension, got strides {x.stride()}")


def _output(name: str, x, shape, out):
    """The output tensor for x, checked or made."""
    if out is None:
        if attn._empty_like is None:
            attn._int32()
        return attn._empty_like(x, memory_format=attn._dense)
    if out.shape != shape:
        raise ValueError(f"{name} has shape {tuple(out.shape)}, expected {tuple(shape)}")
    _check_heads(name, out, shape, x.dtype, x.get_device())
    return out


def _check_rotary(rotary: Rotary, dev: int) -> None:
    if rotary.device_index != dev:
        raise ValueError(f"the rotary is on device {rotary.device_index}, the call on {dev}")


def rotate(q, k, rotary: Rotary, positions, q_weight=None, k_weight=None, eps: float = 1e-6, out_q=None, out_k=None, stream=None):
    """q and k (None: q alone) [tokens, heads, head_dim], each head normed (with a weight: x * weight / sqrt(mean(x^2) + eps))
    and rotated by its token's position; positions: int32 [tokens]. Returns (q', k'), or q' without k. out_q may be q
    and out_k k (in place), neither the other's."""
    shape, dtype, dev = q.shape, q.dtype, q.get_device()
    _check_heads("q", q, shape, dtype, dev)
    _check_rotary(rotary, dev)
    T, _, D = shape
    out_q = _output("out_q", q, shape, out_q)
    kb = None
    if k is not None:
        ks = k.shape
        _check_heads("k", k, ks, dtype, dev)
        if ks[0] != T or ks[2] != D:
            raise ValueError(f"k has shape {tuple(ks)}, q {tuple(shape)}: the same tokens and head_dim are needed")
        out_k = _output("out_k", k, ks, out_k)
        kb = _heads("k_weight", k, ks, out_k, k_weight, eps, dev)
    st = (_bound or _lib()).hq_rotate(rotary._ref, _heads("q_weight", q, shape, out_q, q_weight, eps, dev), kb, T, D, hq._dt(q),
                                      attn._ints("positions", positions, T, dev) or None, hq._stream_ptr(stream))
    if st:
        hq.check(st)
    return out_q if k is None else (out_q, out_k)


def append(cache, layer: int, rotary: Rotary, q, k, v, rows, cu_seqlens=None, q_weight=None, k_weight=None, eps: float = 1e-6, out=None,
           stream=None):
    """KVCache.append_rotated."""
    shape, dtype, dev, D = k.shape, cache.k.dtype, cache.device_index, cache.head_dim
    _check_heads("k", k, shape, dtype, dev)
    T, H, _ = shape
    if shape != (T, cache.kv_heads, D):
        raise ValueError(f"k has shape {tuple(shape)}, the cache holds {cache.kv_heads} heads of {D}")
    if v.shape != shape:
        raise ValueError(f"v has shape {tuple(v.shape)}, k {tuple(shape)}")
    _check_heads("v", v, shape, dtype, dev)
    _check_rotary(rotary, dev)
    qb = None
    if q is not None:
        qs = q.shape
        _check_heads("q", q, qs, dtype, dev)
        if qs[0] != T or qs[2] != D:
            raise ValueError(f"q has shape {tuple(qs)}: {T} tokens with head_dim {D} are needed")
        out = _output("out", q, qs, out)
        qb = _heads("q_weight", q, qs, out, q_weight, eps, dev)
    n = rows.numel()
    vr, vh, _ = v.stride()
    st = (_bound or _lib()).hq_cache_append_rotated(cache._ref, layer, rotary._ref, qb, _heads("k_weight", k, shape, None, k_weight, eps, dev), v.data_ptr(),
                                                    vr if T > 1 else 0, vh if H > 1 else 0, T, cache._list("rows", rows),
                                                    None if cu_seqlens is None else attn._ints("cu_seqlens", cu_seqlens, n + 1, dev), n,
                                                    hq._stream_ptr(stream))
    if st:
        hq.check(st)
    return out if q is not None else None
