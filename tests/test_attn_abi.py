"""CPU tests of the attention and cache entry points (include/hq_attn.h): exports, struct layouts, and
that bad arguments are refused before anything touches a device."""
import ctypes
import re
from pathlib import Path

import pytest

from nebula_amd import attn, hq

ROOT = Path(__file__).resolve().parent.parent
HEADER = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "hq_attn.h").read_text(), flags=re.S)

P = 1 << 20  # an address that is aligned and never followed


def io(**kw):
    d = dict(Q=P, O=P, lse=0, q_row=6144, q_head=128, o_row=6144, o_head=128, rows=4, heads=48, head_dim=128, dtype=1, scale=0.1)
    d.update(kw)
    return bytes(attn.AttnIO(**d))


def cache(**kw):
    d = dict(K=P, V=P, layer_stride=64 * 65536, page_stride=65536, head_stride=8192, token_stride=128, layers=2, pages=64, kv_heads=8,
             page_tokens=64, head_dim=128, dtype=1, table=P, table_stride=32, rows=16, max_pages=32, lens=P, refs=P, status=P)
    d.update(kw)
    return ctypes.byref(attn.KVCacheDesc(**d))


def test_library_exports_every_declared_symbol():
    declared = sorted(set(re.findall(r"\b(hq_[a-z0-9_]+)\s*\(", HEADER)))
    assert declared == sorted(attn.EXPORTS)
    for name in declared:
        assert hasattr(hq.lib(), name), name


def test_structs_mirror_the_header():
    for cname, cls in (("hq_attn_io", attn.AttnIO), ("hq_kv_cache", attn.KVCacheDesc)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), HEADER, flags=re.S).group(1)
        names = [n.strip().lstrip("*").split()[-1].lstrip("*") for line in body.split(";") if line.strip()
                 for n in line.split(",")]
        assert names == [f[0] for f in cls._fields_]
    assert attn._IO.size == ctypes.sizeof(attn.AttnIO)
    assert dict(re.findall(r"#define HQ_CACHE_(\w+) (\d+)u", HEADER)) == {
        "BAD_ROW": str(attn.BAD_ROW), "NO_PAGES": str(attn.NO_PAGES), "ROW_FULL": str(attn.ROW_FULL), "BAD_PAGE": str(attn.BAD_PAGE),
        "MAX_BATCH": str(attn.MAX_BATCH)}


def call_prompt(i, K=P, k_row=1024, k_head=128, V=P, v_row=1024, v_head=128, kv_heads=8, total_k=4, cu_q=P, cu_k=0, seqs=1, ws=0, wsb=0):
    return attn._lib().hq_attn_prompt(i, K or None, k_row, k_head, V or None, v_row, v_head, kv_heads, total_k, cu_q or None, cu_k or None,
                                      seqs, 1, 0, ws or None, wsb, None)


BAD_IO = [
    (dict(Q=0), hq.HQ_ERR_INVALID_ARG), (dict(O=0), hq.HQ_ERR_INVALID_ARG), (dict(dtype=3), hq.HQ_ERR_INVALID_ARG),
    (dict(head_dim=96), hq.HQ_ERR_UNSUPPORTED), (dict(head_dim=0), hq.HQ_ERR_UNSUPPORTED), (dict(rows=0), hq.HQ_ERR_SHAPE),
    (dict(heads=0), hq.HQ_ERR_SHAPE), (dict(heads=44), hq.HQ_ERR_SHAPE), (dict(rows=1 << 25), hq.HQ_ERR_SHAPE),
    (dict(scale=0.0), hq.HQ_ERR_INVALID_ARG), (dict(scale=-1.0), hq.HQ_ERR_INVALID_ARG), (dict(scale=float("nan")), hq.HQ_ERR_INVALID_ARG),
    (dict(scale=float("inf")), hq.HQ_ERR_INVALID_ARG), (dict(Q=P + 8), hq.HQ_ERR_ALIGNMENT), (dict(O=P + 2), hq.HQ_ERR_ALIGNMENT),
    (dict(lse=P + 2), hq.HQ_ERR_ALIGNMENT), (dict(q_row=6148), hq.HQ_ERR_ALIGNMENT), (dict(o_head=132), hq.HQ_ERR_ALIGNMENT),
    (dict(q_head=64), hq.HQ_ERR_SHAPE), (dict(q_row=-8), hq.HQ_ERR_SHAPE), (dict(o_row=64), hq.HQ_ERR_SHAPE),
    (dict(q_row=1 << 60), hq.HQ_ERR_SHAPE),
]


@pytest.mark.parametrize("kw,status", BAD_IO)
def test_attention_refuses_bad_queries(kw, status):
    L = attn._lib()
    for got in (call_prompt(io(**kw)), L.hq_attn_paged(io(**kw), cache(), 0, None, P, 4, 0, None, 0, None),
                L.hq_attn_shared_prefix(io(**{"rows": 4, **kw}), cache(), 0, None, 4, P, P, 1, 0, 0, None, 0, None)):
        if kw.get("rows") == 1 << 25 and got == hq.HQ_ERR_SHAPE:
            continue
        assert got == status, (kw, got, L.hq_last_error())
    assert L.hq_last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(K=0), hq.HQ_ERR_INVALID_ARG), (dict(V=0), hq.HQ_ERR_INVALID_ARG), (dict(K=P + 8), hq.HQ_ERR_ALIGNMENT),
    (dict(k_row=1028), hq.HQ_ERR_ALIGNMENT), (dict(v_head=64), hq.HQ_ERR_SHAPE), (dict(kv_heads=0), hq.HQ_ERR_SHAPE),
    (dict(kv_heads=7), hq.HQ_ERR_SHAPE), (dict(cu_q=0), hq.HQ_ERR_INVALID_ARG), (dict(cu_q=P + 1), hq.HQ_ERR_ALIGNMENT),
    (dict(cu_k=P + 2), hq.HQ_ERR_ALIGNMENT), (dict(seqs=0), hq.HQ_ERR_SHAPE), (dict(total_k=3), hq.HQ_ERR_SHAPE),
    (dict(total_k=(1 << 30) + 1), hq.HQ_ERR_SHAPE)])
def test_prompt_refuses_bad_keys(kw, status):
    assert call_prompt(io(), **kw) == status, hq.lib().hq_last_error()


BAD_CACHE = [
    (dict(K=0), hq.HQ_ERR_INVALID_ARG), (dict(table=0), hq.HQ_ERR_INVALID_ARG), (dict(status=0), hq.HQ_ERR_INVALID_ARG),
    (dict(dtype=0), hq.HQ_ERR_INVALID_ARG), (dict(head_dim=80), hq.HQ_ERR_UNSUPPORTED), (dict(pages=0), hq.HQ_ERR_SHAPE),
    (dict(page_tokens=0), hq.HQ_ERR_SHAPE), (dict(page_tokens=48), hq.HQ_ERR_SHAPE), (dict(page_tokens=8), hq.HQ_ERR_SHAPE), (dict(page_tokens=1 << 17), hq.HQ_ERR_SHAPE),
    (dict(table_stride=31), hq.HQ_ERR_SHAPE), (dict(token_stride=256), hq.HQ_ERR_SHAPE), (dict(page_stride=65528), hq.HQ_ERR_SHAPE),
    (dict(page_stride=65540), hq.HQ_ERR_SHAPE), (dict(layer_stride=8), hq.HQ_ERR_SHAPE), (dict(V=P + 8), hq.HQ_ERR_ALIGNMENT),
    (dict(lens=P + 2), hq.HQ_ERR_ALIGNMENT), (dict(max_pages=1 << 25, table_stride=1 << 25), hq.HQ_ERR_SHAPE),
]


@pytest.mark.parametrize("kw,status", BAD_CACHE)
def test_cache_calls_refuse_a_bad_cache(kw, status):
    L = attn._lib()
    b = ctypes.c_size_t(0)
    c = cache(**kw)
    for got in (L.hq_attn_paged(io(), c, 0, None, None, 4, 0, None, 0, None),
                L.hq_attn_shared_prefix(io(), c, 0, None, 4, P, P, 1, 0, 0, None, 0, None), L.hq_cache_reserve(c, P, P, 1, None),
                L.hq_cache_append(c, 0, P, 1024, 128, P, 1024, 128, 1, P, None, 1, None), L.hq_cache_fork(c, P, P, 1, None, 0, None),
                L.hq_cache_free(c, P, 1, None), L.hq_cache_copy_pages(c, P, P, 1, None),
                L.hq_cache_compact(c, P, 1 << 25, P, None, 0, None), L.hq_cache_workspace_bytes(c, ctypes.byref(b))):
        assert got == status, (kw, got, L.hq_last_error())


def test_cache_calls_refuse_bad_arguments():
    L = attn._lib()
    E = hq
    assert L.hq_attn_paged(io(), cache(), 2, None, None, 4, 0, None, 0, None) == E.HQ_ERR_SHAPE  # layer
    assert L.hq_attn_paged(io(rows=5), cache(), 0, None, None, 4, 0, None, 0, None) == E.HQ_ERR_SHAPE
    assert L.hq_attn_paged(io(rows=17), cache(), 0, None, None, 17, 0, None, 0, None) == E.HQ_ERR_SHAPE  # more than the cache's rows
    assert L.hq_attn_paged(io(dtype=2), cache(), 0, None, None, 4, 0, None, 0, None) == E.HQ_ERR_SHAPE
    assert L.hq_attn_paged(io(head_dim=64), cache(), 0, None, None, 4, 0, None, 0, None) == E.HQ_ERR_SHAPE
    assert L.hq_attn_paged(io(), None, 0, None, None, 4, 0, None, 0, None) == E.HQ_ERR_INVALID_ARG
    for groups in (0, 5):
        assert L.hq_attn_shared_prefix(io(), cache(), 0, None, 4, P, P, groups, 0, 0, None, 0, None) == E.HQ_ERR_SHAPE
    assert L.hq_attn_shared_prefix(io(), cache(), 0, None, 4, None, P, 1, 0, 0, None, 0, None) == E.HQ_ERR_INVALID_ARG
    assert L.hq_attn_shared_prefix(io(rows=3), cache(), 0, None, 4, P, P, 1, 0, 0, None, 0, None) == E.HQ_ERR_SHAPE
    for n in (0, attn.MAX_BATCH + 1):
        for got in (L.hq_cache_reserve(cache(), P, P, n, None), L.hq_cache_fork(cache(), P, P, n, None, 0, None),
                    L.hq_cache_free(cache(), P, n, None), L.hq_cache_copy_pages(cache(), P, P, n, None),
                    L.hq_cache_append(cache(), 0, P, 1024, 128, P, 1024, 128, n, P, None, n, None)):
            assert got == E.HQ_ERR_SHAPE
    for got in (L.hq_cache_reserve(cache(), None, P, 1, None), L.hq_cache_reserve(cache(), P, None, 1, None),
                L.hq_cache_fork(cache(), P, None, 1, None, 0, None), L.hq_cache_free(cache(), None, 1, None),
                L.hq_cache_copy_pages(cache(), None, P, 1, None), L.hq_cache_compact(cache(), None, 32, P, None, 0, None),
                L.hq_cache_compact(cache(), P, 32, None, None, 0, None)):
        assert got == E.HQ_ERR_INVALID_ARG
    assert L.hq_cache_reserve(cache(), P + 2, P, 1, None) == E.HQ_ERR_ALIGNMENT
    assert L.hq_cache_append(cache(), 0, P, 1024, 128, P, 1024, 128, 3, P, None, 2, None) == E.HQ_ERR_SHAPE
    assert L.hq_cache_append(cache(), 7, P, 1024, 128, P, 1024, 128, 2, P, None, 2, None) == E.HQ_ERR_SHAPE
    assert L.hq_cache_append(cache(), 0, P + 8, 1024, 128, P, 1024, 128, 2, P, None, 2, None) == E.HQ_ERR_ALIGNMENT
    assert L.hq_cache_compact(cache(), P, 31, P, None, 0, None) == E.HQ_ERR_SHAPE
    assert L.hq_cache_compact(cache(), P, 64, P, None, 0, None) == E.HQ_ERR_SHAPE  # the cache's own table, another stride
    # A workspace too small, or not aligned.
    assert L.hq_cache_fork(cache(), P, P, 1, P, 64, None) == E.HQ_ERR_WORKSPACE
    assert L.hq_cache_compact(cache(), P + 4096, 32, P, P + 64, 1 << 20, None) == E.HQ_ERR_ALIGNMENT


def test_queries_refuse_bad_shapes():
    for bad in (dict(kind=0), dict(kind=4), dict(rows=0), dict(seqs=0), dict(heads=47), dict(head_dim=32)):
        a = dict(kind=attn.KIND_PAGED, rows=4, seqs=4, heads=48, kv_heads=8, head_dim=128, max_keys=100) | bad
        with pytest.raises(hq.HQError):
            attn.workspace_bytes(**a)
        with pytest.raises(hq.HQError):
            attn.describe(**a)
    with pytest.raises(hq.HQError):
        attn.workspace_bytes(attn.KIND_SHARED, 4, 4, 48, 8, 128, 100, groups=5)
    assert "hq_attn" in attn.describe(attn.KIND_PROMPT, 4, 1, 48, 8, 128, 4)


def test_wrappers_refuse_host_tensors():
    import torch

    q = torch.zeros(4, 8, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        attn.prompt(q, q, q, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        attn.KVCache(torch.zeros(1, 2, 2, 16, 64), torch.zeros(1, 2, 2, 16, 64), None, None, None)
