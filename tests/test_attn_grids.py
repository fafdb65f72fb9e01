"""CPU tests: calls whose launches would have 2^32 threads or more in a grid's dimension are refused by their
shapes, before anything is enqueued."""
import pytest

from nebula_amd import attn, hq
from test_attn_abi import P, cache, io

M = 1 << 20


@pytest.mark.parametrize("kind,rows,seqs,heads,kv_heads", [
    (attn.KIND_PAGED, M, M, 1024, 1024), (attn.KIND_PROMPT, M, M, 64, 64), (attn.KIND_SHARED, M, M, 512, 8), (attn.KIND_SHARED, M, M, 64, 1),
    (attn.KIND_PROMPT, M, M, 16, 16)])
def test_queries_refuse_too_many_workgroups(kind, rows, seqs, heads, kv_heads):
    for f in (attn.workspace_bytes, attn.describe):
        with pytest.raises(hq.HQError) as e:
            f(kind, rows, seqs, heads, kv_heads, 128, 4096, 1, 64)
        assert e.value.status == hq.HQ_ERR_SHAPE


@pytest.mark.parametrize("kind,rows,seqs,heads,kv_heads", [
    (attn.KIND_PAGED, M, M, 8, 8), (attn.KIND_PROMPT, 1 << 24, 1, 64, 8), (attn.KIND_PROMPT, 1 << 20, 1, 1024, 1024), (attn.KIND_SHARED, 1 << 18, 1 << 18, 64, 8)])
def test_the_largest_pass(kind, rows, seqs, heads, kv_heads):
    assert "hq_attn" in attn.describe(kind, rows, seqs, heads, kv_heads, 128, 4096, 1, 64)


def test_calls_refuse_them():
    L = attn._lib()
    c = cache(rows=M)
    big = io(rows=M, heads=512, o_row=512 * 128, q_row=512 * 128)
    assert L.hq_attn_shared_prefix(big, c, 0, None, M, P, P, 1, 64, 0, None, 0, None) == hq.HQ_ERR_SHAPE
    wide = dict(kv_heads=1024, head_stride=64 * 128, token_stride=128, page_stride=1024 * 64 * 128, layer_stride=64 * 1024 * 64 * 128)
    assert L.hq_attn_paged(io(rows=M, heads=1024, o_row=1 << 17, q_row=1 << 17), cache(rows=M, **wide), 0, None, None, M, 0, None, 0, None) == hq.HQ_ERR_SHAPE
    assert L.hq_cache_append(cache(**wide), 0, P, 1 << 17, 128, P, 1 << 17, 128, 1 << 19, P, P, 1, None) == hq.HQ_ERR_SHAPE
    # A page of 160 GiB over all layers.
    huge = dict(kv_heads=1024, page_tokens=65536, head_stride=65536 * 128, token_stride=128, page_stride=1 << 33, layer_stride=1 << 33, layers=5, pages=1,
                max_pages=1, table_stride=1)
    for got in (L.hq_cache_fork(cache(**huge), P, P, 1, None, 0, None), L.hq_cache_copy_pages(cache(**huge), P, P, 1, None)):
        assert got == hq.HQ_ERR_SHAPE
