"""A state space layer's mixer between its projections (include/hq_ssm.h): the short causal convolution and the
selective scan, for packed prompts and for single tokens, with the states that sequences keep (nebula_amd.decoder
runs them between a layer's fused projections).

    states = StateCache.create(layers, rows, channels, width, heads, head_dim, state_dim, dtype)
    for each layer:
        xbc = states.conv(layer, xbc, weight, rows, cu, bias=bias, held=held)
        y = states.scan(layer, x, dt, A, B, C, rows, cu, D=D, z=z, dt_bias=dt_bias, held=held)

x, B and C [tokens, heads or groups, dim] are views of xbc. Activations are float16 or bfloat16 on the GPU, weights and
states of the scan float32. Lists of rows, lengths and offsets are int32 device tensors: no call waits for the device. What
a call meets there (a bad row) goes to states.status; states.check() waits and raises. torch supplies memory and streams
only; every computation runs in the HIP library.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional

from . import attn, hq

HEAD_DIMS, STATE_DIMS, WIDTHS = (64, 128), (64, 128, 256), (2, 3, 4)
MAX_BATCH = 1024

# Every symbol include/hq_ssm.h declares.
EXPORTS = ("hq_ssm_conv", "hq_ssm_workspace_bytes", "hq_describe_ssm", "hq_ssm_scan")


class StateCacheDesc(ctypes.Structure):
    _fields_ = [("conv", ctypes.c_void_p), ("ssm", ctypes.c_void_p), ("conv_layer", ctypes.c_int64), ("conv_row", ctypes.c_int64),
                ("ssm_layer", ctypes.c_int64), ("ssm_row", ctypes.c_int64), ("layers", ctypes.c_uint32), ("rows", ctypes.c_uint32),
                ("channels", ctypes.c_uint32), ("width", ctypes.c_uint32), ("heads", ctypes.c_uint32), ("head_dim", ctypes.c_uint32),
                ("state_dim", ctypes.c_uint32), ("dtype", ctypes.c_int), ("status", ctypes.c_void_p), ("refused", ctypes.c_void_p)]


class ScanIO(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("X", "B", "C", "dt", "Z", "Y", "A", "D", "dt_bias")] + \
               [(n, ctypes.c_int64) for n in ("x_row", "x_head", "b_row", "b_group", "c_row", "c_group", "dt_row", "z_row", "z_head",
                                              "y_row", "y_head")] + \
               [("tokens", ctypes.c_uint32), ("groups", ctypes.c_uint32), ("dt_f32", ctypes.c_int), ("softplus", ctypes.c_int)]


# hq_ssm_io as bytes, packed by every call.
_IO = struct.Struct("@9P11qIIii")
assert _IO.size == ctypes.sizeof(ScanIO)

_bound: Optional[ctypes.CDLL] = None


def _lib() -> ctypes.CDLL:
    global _bound
    if _bound is not None:
        return _bound
    L = hq.lib()
    u32, i64, sz, vp, i32 = ctypes.c_uint32, ctypes.c_int64, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_int
    cache = ctypes.POINTER(StateCacheDesc)
    args = {
        "hq_ssm_conv": [cache, u32, vp, i64, vp, i64, vp, vp, i32, u32, vp, vp, vp, u32, vp],
        "hq_ssm_workspace_bytes": [u32, u32, i32, u32, u32, u32, u32, u32, ctypes.POINTER(sz)],
        "hq_describe_ssm": [u32, u32, i32, u32, u32, u32, u32, u32, ctypes.c_char_p, sz],
        "hq_ssm_scan": [cache, u32, ctypes.c_char_p, vp, vp, vp, u32, u32, vp, sz, vp],
    }
    for name, types in args.items():
        f = getattr(L, name)
        f.restype, f.argtypes = i32, types
    _bound = L
    return L


def _floats(name: str, t, n: int, dev: int) -> int:
    """Address of a contiguous float32 tensor of n entries on GPU dev (None: 0)."""
    if t is None:
        return 0
    if t.get_device() != dev or t.dtype != (hq._torch or hq._load()).float32 or not t.is_contiguous() or t.numel() != n:
        raise ValueError(f"{name} must be a contiguous float32 tensor of {n} entries on the call's device, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _heads(name: str, t, shape, dtype, dev: int):
    """(address, row stride, head stride) of a [tokens, heads, dim] operand; an axis of one entry may have any stride: 0 stands for it."""
    if t.shape != shape or t.dtype != dtype or t.get_device() != dev:
        raise ValueError(f"{name} must be {dtype} {tuple(shape)} on device {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    row, head, one = t.stride()
    if one != 1:
        raise ValueError(f"{name} must have unit stride along its last dimension, got strides {t.stride()}")
    return t.data_ptr(), row if shape[0] > 1 else 0, head if shape[1] > 1 else 0


def _rows(name: str, t, shape, dtype, dev: int):
    """(address, row stride) of a [tokens, channels] operand; that of one token is the channels."""
    if t.shape != shape or t.dtype != dtype or t.get_device() != dev:
        raise ValueError(f"{name} must be {dtype} {tuple(shape)} on device {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    row, one = t.stride()
    if one != 1 or (shape[0] > 1 and row < shape[1]):
        raise ValueError(f"{name} must have unit stride along its channels and rows apart, got strides {t.stride()}")
    return t.data_ptr(), row if shape[0] > 1 else shape[1]


def _torch_calls():
    attn._int32()
    return attn._empty_like


class StateCache:
    """The states of sequences, over the caller's tensors.

    conv: [layers, rows, width - 1, channels] float16 or bfloat16, the last inputs of the convolution, oldest first;
    ssm: [layers, rows, heads, head_dim, state_dim] float32; either may be None where it is not used. status: int32 [1], zero, made
    if not given. refused: int32 [rows] or None, a KVCache's: the states of rows whose reserve() was refused stay as they
    are, so that a step of both kinds of layers can be run again.

    A sequence is a row. held[i] is how many tokens rows[i] holds before a call: with 0 its states are taken as zero, whatever is
    there, so that a row needs no clearing; held None: all continue."""

    def __init__(self, conv=None, ssm=None, status=None, refused=None):
        import torch

        if conv is None and ssm is None:
            raise ValueError("conv or ssm is needed")
        for name, t, dims in (("conv", conv, 4), ("ssm", ssm, 5)):
            if t is None:
                continue
            if t.dim() != dims or not t.is_cuda:
                raise ValueError(f"{name} must be a device tensor of {dims} dimensions, got {tuple(t.shape)} on {t.device}")
            if min(t.shape) > 0 and not t[0, 0].is_contiguous():
                raise ValueError(f"{name}: a row of a layer must be contiguous, got strides {t.stride()}")
        if ssm is not None and ssm.dtype != torch.float32:
            raise ValueError(f"ssm must be float32, got {ssm.dtype}")
        first = conv if conv is not None else ssm
        if conv is not None and ssm is not None and (conv.shape[:2] != ssm.shape[:2] or conv.device != ssm.device):
            raise ValueError(f"conv and ssm must have the same layers, rows and device, got {tuple(conv.shape)} and {tuple(ssm.shape)}")
        self.layers, self.rows = first.shape[:2]
        self.device_index = dev = first.get_device()
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=first.device)
        attn._ints("status", status, 1, dev)
        attn._ints("refused", refused, self.rows, dev)
        self.conv_state, self.ssm_state, self.status, self.refused = conv, ssm, status, refused
        d = StateCacheDesc(layers=self.layers, rows=self.rows, status=status.data_ptr(), refused=refused.data_ptr() if refused is not None else None)
        self.channels = self.width = self.heads = self.head_dim = self.state_dim = 0
        self.dtype = None
        if conv is not None:
            self.channels, self.width, self.dtype = conv.shape[3], conv.shape[2] + 1, conv.dtype
            d.conv, d.dtype, d.channels, d.width = conv.data_ptr(), hq._dt(conv), self.channels, self.width
            d.conv_layer, d.conv_row = self._strides(conv)
        if ssm is not None:
            self.heads, self.head_dim, self.state_dim = ssm.shape[2:]
            d.ssm, d.heads, d.head_dim, d.state_dim = ssm.data_ptr(), self.heads, self.head_dim, self.state_dim
            d.ssm_layer, d.ssm_row = self._strides(ssm)
        # One descriptor for each type of activations: without conv a scan's x has either.
        self._refs = {}
        for t, code in (hq._torch or hq._load()).dtypes.items():
            if self.dtype in (None, t):
                own = StateCacheDesc.from_buffer_copy(d)
                own.dtype = code
                self._refs[t] = ctypes.byref(own)

    @staticmethod
    def _strides(t):
        """Layer and row stride; an axis of one entry may have any: a dense one stands for it."""
        row = t.stride(1) if t.shape[1] > 1 else t[0, 0].numel()
        return (t.stride(0) if t.shape[0] > 1 else row * t.shape[1]), row

    @classmethod
    def create(cls, layers: int, rows: int, channels: int, width: int, heads: int, head_dim: int, state_dim: int, dtype=None, refused=None,
               device="cuda") -> "StateCache":
        """States of `rows` sequences, zero."""
        import torch

        return cls(torch.zeros(layers, rows, width - 1, channels, dtype=dtype or torch.bfloat16, device=device),
                   torch.zeros(layers, rows, heads, head_dim, state_dim, dtype=torch.float32, device=device), refused=refused)

    def _sequences(self, T: int, rows, cu_seqlens, held):
        """Addresses of the lists, and how many sequences."""
        dev, n, cp = self.device_index, T, None
        if cu_seqlens is not None:
            n, cp = max(cu_seqlens.numel() - 1, 0), attn._ints("cu_seqlens", cu_seqlens, None, dev)
        return None if rows is None else attn._ints("rows", rows, n, dev), None if held is None else attn._ints("held", held, n, dev), cp, n

    def conv(self, layer: int, x, weight, rows=None, cu_seqlens=None, bias=None, silu: bool = True, held=None, out=None, stream=None):
        """Causal convolution of each channel of x [tokens, channels] with weight [channels, width] (float32), plus bias
        [channels], through u / (1 + exp(-u)) if silu: tokens [cu_seqlens[i], cu_seqlens[i + 1]) are rows[i]'s next ones
        (cu_seqlens None: one token a row; rows None: row i). The rows' last inputs are kept. Returns out, apart from x."""
        T, C = shape = x.shape
        dtype, dev = x.dtype, self.device_index
        ref = self._refs.get(dtype)
        if ref is None or self.conv_state is None or C != self.channels:
            raise ValueError(f"x is {dtype} of {C} channels, the states {self.dtype} of {self.channels}")
        xp, ldx = _rows("x", x, shape, dtype, dev)
        if out is None:
            out = (attn._empty_like or _torch_calls())(x, memory_format=attn._dense)
        yp, ldy = _rows("out", out, shape, dtype, dev)
        rp, hp, cp, n = self._sequences(T, rows, cu_seqlens, held)
        st = (_bound or _lib()).hq_ssm_conv(ref, layer, xp, ldx, yp, ldy, _floats("weight", weight, C * self.width, dev),
                                            None if bias is None else _floats("bias", bias, C, dev), silu, T, rp, hp, cp, n, hq._stream_ptr(stream))
        if st:
            hq.check(st)
        return out

    def scan(self, layer: int, x, dt, A, B, C, rows=None, cu_seqlens=None, D=None, z=None, dt_bias=None, softplus: bool = True, held=None,
             max_len: int = 0, out=None, stream=None, workspace=None):
        """Selective scan: per token and head, with s = dt + dt_bias (log(1 + exp(s)) if softplus),
            S = exp(A s) S + s x B^T;  y = S C + D x,  times z / (1 + exp(-z)) with a gate z.
        x, z and out [tokens, heads, head_dim], B and C [tokens, groups, state_dim], dt [tokens, heads] float32 or x's type; A (not
        positive), D and dt_bias float32 [heads]. Sequences as in conv(); their states S are kept. max_len: no sequence has more
        new tokens (a hint for the split: several prompts of one length take up to twice as long without it). Single tokens and a
        long chunk are faster as two calls. out may be z."""
        dtype = x.dtype
        ref = self._refs.get(dtype)
        if ref is None or self.ssm_state is None:
            raise ValueError(f"x is {dtype}, the states {self.dtype}")
        dev, H, xs, bs = self.device_index, self.heads, x.shape, B.shape
        if len(xs) != 3 or len(bs) != 3 or xs != (xs[0], H, self.head_dim) or bs != (xs[0], bs[1], self.state_dim):
            raise self._shapes(x, B, C, z)
        xp, xr, xh = _heads("x", x, xs, dtype, dev)
        bp, br, bh = _heads("B", B, bs, dtype, dev)
        cp, cr, ch = _heads("C", C, bs, dtype, dev)
        zp, zr, zh = (0, 0, 0) if z is None else _heads("z", z, xs, dtype, dev)
        T, f32 = xs[0], dt.dtype
        f32 = f32 == (hq._torch or hq._load()).float32 or (None if f32 != dtype else False)
        if f32 is None or dt.get_device() != dev or dt.shape != (T, H) or (H > 1 and dt.stride(1) != 1):
            raise ValueError(f"dt must be [{T}, {H}] float32 or {dtype} with unit stride along the heads, got {dt.dtype} {tuple(dt.shape)} on {dt.device}")
        if out is None:
            out = (attn._empty_like or _torch_calls())(x, memory_format=attn._dense)
        yp, yr, yh = _heads("out", out, xs, dtype, dev)
        rp, hp, cup, n = self._sequences(T, rows, cu_seqlens, held)
        wp, wb = (None, 0) if workspace is None else hq._ws(workspace)
        io = _IO.pack(xp, bp, cp, dt.data_ptr(), zp, yp, _floats("A", A, H, dev), _floats("D", D, H, dev), _floats("dt_bias", dt_bias, H, dev),
                      xr, xh, br, bh, cr, ch, dt.stride(0) if T > 1 else H, zr, zh, yr, yh, T, bs[1], f32, softplus)
        st = (_bound or _lib()).hq_ssm_scan(ref, layer, io, rp, hp, cup, n, max_len, wp, wb, hq._stream_ptr(stream))
        if st:
            hq.check(st)
        return out

    def _shapes(self, x, B, C, z):
        return ValueError(f"x {tuple(x.shape)}, z or out {None if z is None else tuple(z.shape)}, B {tuple(B.shape)}, C {tuple(C.shape)}: need "
                          f"[tokens, {self.heads}, {self.head_dim}] and [tokens, groups, {self.state_dim}]")

    def check(self) -> None:
        """Waits for the device, all its streams, and raises HQError if a call met a fault there since the last check."""
        import torch

        torch.cuda.synchronize(self.device_index)
        got = int(self.status.item())
        if got:
            self.status.zero_()
            torch.cuda.synchronize(self.device_index)  # not after what a call on another stream reports next
            raise hq.HQError(hq.HQ_ERR_DEVICE, "states: " + "; ".join(text for bit, text in attn.FAULTS.items() if got & bit))


def workspace_bytes(tokens: int, sequences: int, heads: int, groups: int, head_dim: int, state_dim: int, max_len: int = 0, single: bool = False) -> int:
    """Workspace of one scan on the current device (single: one without cu_seqlens), and of every one of as many sequences with
    fewer tokens: it does not fall as tokens and max_len grow."""
    b = ctypes.c_size_t(0)
    hq.check(_lib().hq_ssm_workspace_bytes(tokens, sequences, int(not single), heads, groups, head_dim, state_dim, max_len, ctypes.byref(b)))
    return int(b.value)


def describe(tokens: int, sequences: int, heads: int, groups: int, head_dim: int, state_dim: int, max_len: int = 0, single: bool = False) -> str:
    """The kernels such a scan runs."""
    buf = ctypes.create_string_buffer(512)
    hq.check(_lib().hq_describe_ssm(tokens, sequences, int(not single), heads, groups, head_dim, state_dim, max_len, buf, len(buf)))
    return buf.value.decode()
