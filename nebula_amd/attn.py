"""Attention and its paged key/value cache (include/hq_attn.h): what stands between a decoder
layer's q | k | v projections (nebula_amd.hq, nebula_amd.decoder) and its output projection.

    cache = KVCache.create(layers, pages, page_tokens, kv_heads, head_dim, rows, max_pages, dtype)
    cache.reserve(rows, counts)                    # once a step: room for its new tokens
    for each layer:
        cache.append(layer, k, v, rows, cu)        # the layer's new keys and values (append_rotated: normed and rotated)
        y = paged(q, cache, layer, rows, cu)       # or prompt(...), shared_prefix(...)
    cache.fork(parents, children); cache.free(rows); cache.compact()

Tensors are float16 or bfloat16 on the GPU, q and outputs [tokens, heads, head_dim], k and v [tokens,
kv_heads, head_dim], with any row and head strides that are multiples of 8 elements (views of wider
projections, for example). Lists of rows, lengths and offsets are int32 device tensors: no call waits
for the device. What a call meets there (no free page, a bad row) goes to cache.status; cache.check()
waits and raises. torch supplies memory and streams only; every computation runs in the HIP library.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional

from . import hq

KIND_PROMPT, KIND_PAGED, KIND_SHARED = 1, 2, 3
HEAD_DIMS = (64, 128, 256)
BAD_ROW, NO_PAGES, ROW_FULL, BAD_PAGE = 1, 2, 4, 8
MAX_BATCH = 1024
FAULTS = {BAD_ROW: "a row number out of range, repeated, or not as the call needs it", NO_PAGES: "too few free pages",
          ROW_FULL: "a sequence would pass its row of the table",
          BAD_PAGE: "a page number out of range, or tokens for a page that several rows hold"}

# Every symbol include/hq_attn.h declares.
EXPORTS = (
    "hq_attn_workspace_bytes", "hq_describe_attn", "hq_attn_prompt", "hq_attn_paged", "hq_attn_shared_prefix",
    "hq_cache_workspace_bytes", "hq_cache_reserve", "hq_cache_append", "hq_cache_fork", "hq_cache_free",
    "hq_cache_copy_pages", "hq_cache_compact",
)


class AttnIO(ctypes.Structure):
    _fields_ = [("Q", ctypes.c_void_p), ("O", ctypes.c_void_p), ("lse", ctypes.c_void_p), ("q_row", ctypes.c_int64),
                ("q_head", ctypes.c_int64), ("o_row", ctypes.c_int64), ("o_head", ctypes.c_int64),
                ("rows", ctypes.c_uint32), ("heads", ctypes.c_uint32), ("head_dim", ctypes.c_uint32),
                ("dtype", ctypes.c_int), ("scale", ctypes.c_float)]


class KVCacheDesc(ctypes.Structure):
    _fields_ = [("K", ctypes.c_void_p), ("V", ctypes.c_void_p), ("layer_stride", ctypes.c_int64),
                ("page_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64), ("token_stride", ctypes.c_int64),
                ("layers", ctypes.c_uint32), ("pages", ctypes.c_uint32), ("kv_heads", ctypes.c_uint32),
                ("page_tokens", ctypes.c_uint32), ("head_dim", ctypes.c_uint32), ("dtype", ctypes.c_int),
                ("table", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("rows", ctypes.c_uint32),
                ("max_pages", ctypes.c_uint32), ("lens", ctypes.c_void_p), ("refs", ctypes.c_void_p),
                ("status", ctypes.c_void_p), ("refused", ctypes.c_void_p)]


# hq_attn_io as bytes, packed by every call.
_IO = struct.Struct("@PPPqqqqIIIif4x")
assert _IO.size == ctypes.sizeof(AttnIO)

_bound: Optional[ctypes.CDLL] = None


def _lib() -> ctypes.CDLL:
    global _bound
    if _bound is not None:
        return _bound
    L = hq.lib()
    u32, i64, sz, vp, i32 = ctypes.c_uint32, ctypes.c_int64, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_int
    io, cache, szp, text = ctypes.c_char_p, ctypes.POINTER(KVCacheDesc), ctypes.POINTER(ctypes.c_size_t), ctypes.c_char_p
    args = {
        "hq_attn_workspace_bytes": [i32, u32, u32, u32, u32, u32, u32, u32, u32, szp],
        "hq_describe_attn": [i32, u32, u32, u32, u32, u32, u32, u32, u32, text, sz],
        "hq_attn_prompt": [io, vp, i64, i64, vp, i64, i64, u32, u32, vp, vp, u32, i32, u32, vp, sz, vp],
        "hq_attn_paged": [io, cache, u32, vp, vp, u32, u32, vp, sz, vp],
        "hq_attn_shared_prefix": [io, cache, u32, vp, u32, vp, vp, u32, u32, u32, vp, sz, vp],
        "hq_cache_workspace_bytes": [cache, szp],
        "hq_cache_reserve": [cache, vp, vp, u32, vp],
        "hq_cache_append": [cache, u32, vp, i64, i64, vp, i64, i64, u32, vp, vp, u32, vp],
        "hq_cache_fork": [cache, vp, vp, u32, vp, sz, vp],
        "hq_cache_free": [cache, vp, u32, vp],
        "hq_cache_copy_pages": [cache, vp, vp, u32, vp],
        "hq_cache_compact": [cache, vp, i64, vp, vp, sz, vp],
    }
    for name, types in args.items():
        f = getattr(L, name)
        f.restype, f.argtypes = i32, types
    _bound = L
    return L


# ---------------------------------------------------------------- checks
def _check_heads(name: str, t, like=None, dtype=None) -> None:
    """t must be [tokens, heads, dim] on a GPU, unit stride in dim, 8-element aligned strides."""
    dev = t.get_device()
    if dev >= 0 and t.dim() == 3 and t.stride(2) == 1 and (dtype is None or t.dtype == dtype) and (like is None or dev == like.get_device()):
        return
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got shape {tuple(t.shape)}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.stride(2) != 1:
        raise ValueError(f"{name} must have unit stride along its last dimension, got strides {t.stride()}")
    raise ValueError(f"{name} is on {t.device}, expected {like.device}")


def _ints(name: str, t, n: Optional[int], dev: int) -> int:
    """Address of a contiguous int32 tensor of n entries on GPU dev (None: 0)."""
    if t is None:
        return 0
    if not (t.get_device() == dev and t.dtype == (_i32t or _int32()) and t.is_contiguous()) or (n is not None and t.numel() != n):
        raise ValueError(f"{name} must be a contiguous int32 tensor{'' if n is None else f' of {n} entries'} on the call's device, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


_i32t = _empty_like = _dense = None


def _int32():
    global _i32t, _empty_like, _dense
    if _i32t is None:
        import torch

        _empty_like, _dense, _i32t = torch.empty_like, torch.contiguous_format, torch.int32
    return _i32t


def _strides(t):
    """Row and head stride of [tokens, heads, dim]; an axis of one entry may have any stride: 0 stands for it."""
    (r, h, _), (sr, sh, _) = t.shape, t.stride()
    return (sr if r > 1 else 0), (sh if h > 1 else 0)


def _io(q, out, lse, scale: float) -> bytes:
    T, H, D = q.shape
    qr, qh = _strides(q)
    orow, oh = _strides(out)
    return _IO.pack(q.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else 0, qr, qh, orow, oh, T, H, D, hq._dt(q), scale)


def _outputs(q, out, lse, with_lse: bool):
    """The output tensors of a call over q, checked or made."""
    if out is None:
        if _i32t is None:
            _int32()
        out = _empty_like(q, memory_format=_dense)  # 0.6 us less than new_empty
    else:
        _check_heads("out", out, q, q.dtype)
        if out.shape != q.shape:
            raise ValueError(f"out has shape {tuple(out.shape)}, expected {tuple(q.shape)}")
    if lse is not None:
        if not (lse.is_cuda and lse.device == q.device and lse.is_contiguous() and lse.dtype == hq._load().float32 and
                tuple(lse.shape) == tuple(q.shape[:2])):
            raise ValueError(f"lse must be a contiguous float32 tensor of shape {tuple(q.shape[:2])} on q's device")
    elif with_lse:
        lse = q.new_empty(q.shape[:2], dtype=hq._load().float32)
    return out, lse


def _scale(scale: Optional[float], D: int) -> float:
    return 1.0 / math.sqrt(D) if scale is None else float(scale)


# ---------------------------------------------------------------- the cache
_rotary_module = None


def _rotary():
    global _rotary_module
    if _rotary_module is None:
        from . import rotary

        _rotary_module = rotary
    return _rotary_module


class KVCache:
    """A paged key/value cache over the caller's tensors.

    k, v: [layers, pages, kv_heads, page_tokens, head_dim] float16 or bfloat16 (or a view of it whose
    pages hold tokens before heads, k.transpose(2, 3) of a [.., page_tokens, kv_heads, ..] tensor).
    table: int32 [rows, max_pages], -1 past a row's tokens; lens: int32 [rows]; refs: int32 [pages],
    holders of each page, 0: free; status: int32 [1] and refused: int32 [rows], zero, made if not given.

    Where reserve() is refused (check() will raise), nothing has changed, and append() to its rows changes
    nothing either until a later reserve() of them goes through: a step can be enqueued whole."""

    def __init__(self, k, v, table, lens, refs, status=None, refused=None):
        import torch

        if k.dim() != 5 or v.shape != k.shape or v.stride() != k.stride() or v.dtype != k.dtype or v.device != k.device:
            raise ValueError("k and v must be alike: [layers, pages, kv_heads, page_tokens, head_dim], the same strides, dtype and device")
        if not k.is_cuda or k.stride(4) != 1:
            raise ValueError("k and v must be device tensors with unit stride along head_dim")
        dt = hq._dt(k)
        layers, pages, heads, tokens, dim = k.shape
        dev = k.get_device()
        if not (table.is_cuda and table.get_device() == dev and table.dtype == torch.int32 and table.dim() == 2 and
                (table.stride(1) == 1 or table.shape[1] == 1) and (table.stride(0) >= table.shape[1] or table.shape[0] == 1)):
            raise ValueError("table must be an int32 [rows, max_pages] tensor on k's device with unit stride along its rows")
        if status is None or refused is None:
            words = torch.zeros(1 + table.shape[0], dtype=torch.int32, device=k.device)
            status, refused = words[:1] if status is None else status, words[1:] if refused is None else refused
        _ints("lens", lens, table.shape[0], dev)
        _ints("refs", refs, pages, dev)
        _ints("status", status, 1, dev)
        _ints("refused", refused, table.shape[0], dev)
        self.k, self.v, self.table, self.lens, self.refs, self.status, self.refused = k, v, table, lens, refs, status, refused
        self.layers, self.pages, self.kv_heads, self.page_tokens, self.head_dim = k.shape
        self.rows, self.max_pages = table.shape
        self.device_index = dev
        sl, sp, sh, st, _ = k.stride()
        if heads == 1 or tokens == 1:  # an axis of one entry: the order of the others stands
            sh, st = (tokens * dim, dim) if heads == 1 else (dim, heads * dim)
            if (heads == 1 and tokens > 1 and k.stride(3) != dim) or (tokens == 1 and heads > 1 and k.stride(2) != dim):
                raise ValueError(f"a page must be dense, got strides {k.stride()}")
        dense = heads * tokens * dim
        self._desc = KVCacheDesc(k.data_ptr(), v.data_ptr(), sl if layers > 1 else dense * pages, sp if pages > 1 else dense, sh, st,
                                 layers, pages, heads, tokens, dim, dt, table.data_ptr(),
                                 table.stride(0) if table.shape[0] > 1 else table.shape[1], self.rows, self.max_pages,
                                 lens.data_ptr(), refs.data_ptr(), status.data_ptr(), refused.data_ptr())
        self._ref = ctypes.byref(self._desc)

    @classmethod
    def create(cls, layers: int, pages: int, page_tokens: int, kv_heads: int, head_dim: int, rows: int, max_pages: int, dtype=None,
               device="cuda") -> "KVCache":
        """An empty cache of `pages` pages for `rows` sequences of up to max_pages pages each."""
        import torch

        shape = (layers, pages, kv_heads, page_tokens, head_dim)
        dtype = dtype or torch.bfloat16
        k, v = torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)
        i32 = dict(dtype=torch.int32, device=device)
        return cls(k, v, torch.full((rows, max_pages), -1, **i32), torch.zeros(rows, **i32), torch.zeros(pages, **i32))

    def _list(self, name, t, n=None):
        p = _ints(name, t, n, self.device_index)
        if not p:
            raise ValueError(f"{name} must be a non-empty int32 device tensor")
        return p

    def _new(self, name, t, tokens=None):
        _check_heads(name, t, self.k, self.k.dtype)
        n, heads, dim = t.shape
        if heads != self.kv_heads or dim != self.head_dim or (tokens is not None and n != tokens):
            raise ValueError(f"{name} must be [tokens, {self.kv_heads}, {self.head_dim}], got {tuple(t.shape)}")

    def reserve(self, rows, counts, stream=None) -> None:
        """Room for counts[i] more tokens of rows[i]: pages for them, and lens grows by as many. All rows or none."""
        n = rows.numel()
        hq.check((_bound or _lib()).hq_cache_reserve(self._ref, self._list("rows", rows), self._list("counts", counts, n), n,
                                                     hq._stream_ptr(stream)))

    def append(self, layer: int, k, v, rows, cu_seqlens=None, stream=None) -> None:
        """Writes k and v [tokens, kv_heads, head_dim] as the last tokens of each row: tokens
        [cu_seqlens[i], cu_seqlens[i + 1]) are rows[i]'s (None: one token a row). Rows whose reserve() was
        refused, and pages that several rows hold, are left as they are."""
        self._new("k", k)
        self._new("v", v, k.shape[0])
        n = rows.numel()
        (kr, kh), (vr, vh) = _strides(k), _strides(v)
        st = (_bound or _lib()).hq_cache_append(self._ref, layer, k.data_ptr(), kr, kh, v.data_ptr(), vr, vh, k.shape[0],
                                                self._list("rows", rows), _ints("cu_seqlens", cu_seqlens, n + 1, self.device_index) or None, n,
                                                hq._stream_ptr(stream))
        if st:
            hq.check(st)

    def append_rotated(self, layer: int, rotary, q, k, v, rows, cu_seqlens=None, q_weight=None, k_weight=None, eps: float = 1e-6,
                       out=None, stream=None):
        """append() with k normed and rotated (nebula_amd.rotary) on its way into the pages by its tokens' places in their
        rows, and q [tokens, heads, head_dim] (None: none) likewise to out: one launch. Returns q's output, which may be q.
        Where append() skips a token, its q is written all the same."""
        return _rotary().append(self, layer, rotary, q, k, v, rows, cu_seqlens, q_weight, k_weight, eps, out, stream)

    def fork(self, parents, children, stream=None, workspace=None) -> None:
        """children[i], an empty row, becomes a copy of parents[i]: full pages shared, a part-filled one copied."""
        n = parents.numel()
        wp, wb = hq._ws(workspace)
        hq.check((_bound or _lib()).hq_cache_fork(self._ref, self._list("parents", parents), self._list("children", children, n), n, wp, wb,
                                                  hq._stream_ptr(stream)))

    def free(self, rows, stream=None) -> None:
        """Empties rows; pages that no row holds any more are free."""
        hq.check((_bound or _lib()).hq_cache_free(self._ref, self._list("rows", rows), rows.numel(), hq._stream_ptr(stream)))

    def copy_pages(self, src, dst, stream=None) -> None:
        """Copies page src[i] to dst[i] in every layer."""
        n = src.numel()
        hq.check((_bound or _lib()).hq_cache_copy_pages(self._ref, self._list("src", src), self._list("dst", dst, n), n, hq._stream_ptr(stream)))

    def compact(self, out_table=None, out_refs=None, stream=None, workspace=None):
        """Moves the live pages to the front of the pool. The table and counts afterwards go to out_table
        [rows, max_pages] and out_refs [pages] (the cache's own by default); returns them."""
        import torch

        table = self.table if out_table is None else out_table
        refs = self.refs if out_refs is None else out_refs
        if out_table is not None and not (table.is_cuda and table.get_device() == self.device_index and table.dtype == torch.int32 and
                                          table.shape == self.table.shape and (table.stride(1) == 1 or table.shape[1] == 1)):
            raise ValueError(f"out_table must be an int32 tensor of shape {tuple(self.table.shape)} on the cache's device")
        stride = table.stride(0) if table.shape[0] > 1 else table.shape[1]
        wp, wb = hq._ws(workspace)
        hq.check((_bound or _lib()).hq_cache_compact(self._ref, table.data_ptr(), stride, self._list("out_refs", refs, self.pages), wp, wb,
                                                     hq._stream_ptr(stream)))
        return table, refs

    def workspace_bytes(self) -> int:
        """What fork and compact need."""
        b = ctypes.c_size_t(0)
        hq.check(_lib().hq_cache_workspace_bytes(self._ref, ctypes.byref(b)))
        return int(b.value)

    def check(self) -> None:
        """Waits for the device, all its streams, and raises HQError if a call met a fault there since the last check."""
        import torch

        torch.cuda.synchronize(self.device_index)
        got = int(self.status.item())
        if got:
            self.status.zero_()
            torch.cuda.synchronize(self.device_index)  # not after what a call on another stream reports next
            raise hq.HQError(hq.HQ_ERR_DEVICE, "cache: " + "; ".join(text for bit, text in FAULTS.items() if got & bit))


# ---------------------------------------------------------------- attention
def workspace_bytes(kind: int, rows: int, seqs: int, heads: int, kv_heads: int, head_dim: int, max_keys: int, groups: int = 1,
                    max_prefix: int = 0) -> int:
    """Workspace of one call (KIND_*) on the current device, and of every call of as many rows and sequences on
    fewer keys (and a shorter prefix): it does not fall as max_keys and max_prefix grow. max_keys is a bound, 0 is refused."""
    b = ctypes.c_size_t(0)
    hq.check(_lib().hq_attn_workspace_bytes(kind, rows, seqs, groups, heads, kv_heads, head_dim, max_keys, max_prefix, ctypes.byref(b)))
    return int(b.value)


def describe(kind: int, rows: int, seqs: int, heads: int, kv_heads: int, head_dim: int, max_keys: int, groups: int = 1,
             max_prefix: int = 0) -> str:
    """The kernels and splits such a call runs."""
    buf = ctypes.create_string_buffer(512)
    hq.check(_lib().hq_describe_attn(kind, rows, seqs, groups, heads, kv_heads, head_dim, max_keys, max_prefix, buf, len(buf)))
    return buf.value.decode()


def prompt(q, k, v, cu_seqlens, cu_seqlens_k=None, causal: bool = True, scale: Optional[float] = None, max_k: int = 0, out=None, lse=None,
           with_lse: bool = False, stream=None, workspace=None):
    """Attention of packed prompts: sequence b's new tokens are rows [cu_seqlens[b], cu_seqlens[b + 1])
    of q, its keys and values rows [cu_seqlens_k[b], cu_seqlens_k[b + 1]) of k and v (None: the same
    rows); causal: the new tokens are the sequence's last ones. cu_*: int32 [sequences + 1] on the
    device. max_k: no sequence has more keys (a hint for the split). Returns out, or (out, lse) with
    lse or with_lse: float32 [tokens, heads]."""
    _check_heads("q", q)
    for name, t in (("k", k), ("v", v)):
        _check_heads(name, t, q, q.dtype)
        if t.shape != k.shape or t.size(2) != q.size(2):
            raise ValueError(f"{name} has shape {tuple(t.shape)}: k and v must be alike, with q's head_dim {q.shape[2]}")
    dev = q.get_device()
    n = cu_seqlens.numel()
    cu, ck = _ints("cu_seqlens", cu_seqlens, n, dev), _ints("cu_seqlens_k", cu_seqlens_k, n, dev)
    out, lse = _outputs(q, out, lse, with_lse)
    wp, wb = hq._ws(workspace)
    (kr, kh), (vr, vh) = _strides(k), _strides(v)
    st = (_bound or _lib()).hq_attn_prompt(_io(q, out, lse, _scale(scale, q.shape[2])), k.data_ptr(), kr, kh, v.data_ptr(), vr, vh, k.shape[1],
                                           k.shape[0], cu, ck or None, max(n - 1, 0), int(causal), max_k, wp, wb, hq._stream_ptr(stream))
    if st:
        hq.check(st)
    return out if lse is None else (out, lse)


def _check_cached(q, cache: KVCache) -> None:
    _check_heads("q", q, cache.k, cache.k.dtype)
    if q.shape[2] != cache.head_dim:
        raise ValueError(f"q has head_dim {q.shape[2]}, the cache {cache.head_dim}")


def paged(q, cache: KVCache, layer: int, rows=None, cu_seqlens=None, max_len: int = 0, scale: Optional[float] = None, out=None, lse=None,
          with_lse: bool = False, stream=None, workspace=None):
    """Causal attention of new tokens over a layer of the cache, theirs among it: tokens
    [cu_seqlens[b], cu_seqlens[b + 1]) of q are the last ones of cache row rows[b] (cu_seqlens None: one
    token a row; rows None: row b). max_len: no row is longer (a hint for the split). Single tokens and a long
    chunk are faster as two calls: the mean number of new tokens chooses the kernel."""
    _check_cached(q, cache)
    dev = cache.device_index
    seqs = q.shape[0] if cu_seqlens is None else max(cu_seqlens.numel() - 1, 0)
    rp, cu = _ints("rows", rows, seqs, dev), _ints("cu_seqlens", cu_seqlens, seqs + 1, dev)
    out, lse = _outputs(q, out, lse, with_lse)
    wp, wb = hq._ws(workspace)
    st = (_bound or _lib()).hq_attn_paged(_io(q, out, lse, _scale(scale, q.shape[2])), cache._ref, layer, rp or None, cu or None, seqs, max_len,
                                          wp, wb, hq._stream_ptr(stream))
    if st:
        hq.check(st)
    return out if lse is None else (out, lse)


def shared_prefix(q, cache: KVCache, layer: int, rows, starts, prefix_lens, max_prefix: int = 0, max_len: int = 0,
                  scale: Optional[float] = None, out=None, lse=None, with_lse: bool = False, stream=None, workspace=None):
    """paged() with one token a row, for a batch in which sequences [starts[g], starts[g + 1]) share their
    first prefix_lens[g] tokens (as cache.fork leaves them): the whole pages of a prefix are read once
    for its group. starts: int32 [groups + 1], prefix_lens: int32 [groups]. max_prefix: no prefix is longer (a
    hint as max_len; 0: not known)."""
    _check_cached(q, cache)
    dev = cache.device_index
    seqs, groups = q.shape[0], prefix_lens.numel()
    rp = _ints("rows", rows, seqs, dev)
    sp, pp = _ints("starts", starts, groups + 1, dev), _ints("prefix_lens", prefix_lens, groups, dev)
    out, lse = _outputs(q, out, lse, with_lse)
    wp, wb = hq._ws(workspace)
    st = (_bound or _lib()).hq_attn_shared_prefix(_io(q, out, lse, _scale(scale, q.shape[2])), cache._ref, layer, rp or None, seqs, sp, pp,
                                                  groups, max_prefix, max_len, wp, wb, hq._stream_ptr(stream))
    if st:
        hq.check(st)
    return out if lse is None else (out, lse)
