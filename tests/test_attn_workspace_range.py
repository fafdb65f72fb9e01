"""CPU tests of the workspace that attention calls ask for over lengths: a buffer taken at the longest keys (and
prefix) serves every shorter call, and a query needs a bound."""
import ctypes
import re

import pytest

from nebula_amd import attn, hq
from test_attn_abi import P, cache, io

LENGTHS = [1, 15, 64, 65, 200, 511, 777, 1024, 2000, 3071, 4096, 6000, 6064, 7999, 8000, 8063, 8064, 8065, 8192, 12288, 20000, 32768, 65536, 131072]
SHAPES = [(64, 1, 48, 8, 128), (64, 1, 24, 4, 256), (16, 16, 24, 4, 256), (64, 64, 48, 8, 128), (512, 1, 32, 4, 64), (2048, 2, 24, 4, 256),
          (1, 1, 48, 8, 128), (4, 4, 12, 2, 128), (80, 17, 48, 8, 128), (333, 3, 12, 12, 64), (17, 1, 40, 1, 128)]


def used(**kw):
    return int(re.search(r"ws=(\d+)", attn.describe(**kw))[1])


@pytest.mark.parametrize("kind", [attn.KIND_PROMPT, attn.KIND_PAGED])
@pytest.mark.parametrize("rows,seqs,heads,kv_heads,dim", SHAPES)
def test_need_does_not_fall_with_the_keys(kind, rows, seqs, heads, kv_heads, dim):
    shape = dict(kind=kind, rows=rows, seqs=seqs, heads=heads, kv_heads=kv_heads, head_dim=dim)
    need = [attn.workspace_bytes(**shape, max_keys=n) for n in LENGTHS]
    assert need == sorted(need), list(zip(LENGTHS, need))
    for n in list(range(1, 700)) + list(range(700, 131073, 61)):
        assert used(**shape, max_keys=n) <= attn.workspace_bytes(**shape, max_keys=n) <= need[-1], n


@pytest.mark.parametrize("groups", [1, 4])
@pytest.mark.parametrize("seqs,heads,kv_heads,dim", [(64, 48, 8, 128), (16, 24, 4, 256), (4, 48, 8, 128), (128, 48, 8, 128), (33, 8, 8, 64)])
def test_need_of_shared_prefixes_does_not_fall(groups, seqs, heads, kv_heads, dim):
    shape = dict(kind=attn.KIND_SHARED, rows=seqs, seqs=seqs, groups=groups, heads=heads, kv_heads=kv_heads, head_dim=dim)
    for n in (100, 4096, 8065, 40000):
        need = [attn.workspace_bytes(**shape, max_keys=n, max_prefix=p) for p in LENGTHS if p <= n]
        assert need == sorted(need)
    for p in (16, 4011, 8192):
        need = [attn.workspace_bytes(**shape, max_keys=n, max_prefix=p) for n in LENGTHS if n >= p]
        assert need == sorted(need)
    most = attn.workspace_bytes(**shape, max_keys=40000, max_prefix=40000)
    for n in range(1, 40000, 97):
        for p in {max(1, n // 7), max(1, n - 500), n}:
            assert used(**shape, max_keys=n, max_prefix=p) <= most, (n, p)


def test_a_buffer_for_the_longest_serves_shorter_calls():
    # Refused by its alignment and not its size, before anything touches a device.
    c = cache(max_pages=256, table_stride=256)
    need = attn.workspace_bytes(attn.KIND_PAGED, 64, 1, 48, 8, 128, 256 * 64)
    for max_len in LENGTHS + [0]:
        st = attn._lib().hq_attn_paged(io(rows=64), c, 0, P, P, 1, max_len, ctypes.c_void_p(P + 64), need, None)
        assert st == hq.HQ_ERR_ALIGNMENT or used(kind=attn.KIND_PAGED, rows=64, seqs=1, heads=48, kv_heads=8, head_dim=128, max_keys=max_len) == 0, max_len
    st = attn._lib().hq_attn_paged(io(rows=64), c, 0, P, P, 1, 8192, ctypes.c_void_p(P), 1 << 20, None)
    assert st == hq.HQ_ERR_WORKSPACE


def test_queries_need_a_bound():
    for kind in (attn.KIND_PROMPT, attn.KIND_PAGED, attn.KIND_SHARED):
        for f in (attn.workspace_bytes, attn.describe):
            with pytest.raises(hq.HQError, match="max_keys=0"):
                f(kind, 4, 4, 48, 8, 128, 0)


@pytest.mark.parametrize("kind,rows,seqs,heads,kv_heads,dim,keys,groups,prefix,splits", [
    (attn.KIND_PAGED, 64, 1, 48, 8, 128, 6064, 1, 0, 10), (attn.KIND_PAGED, 512, 1, 48, 8, 128, 8000, 1, 0, 5),
    (attn.KIND_PROMPT, 512, 1, 48, 8, 128, 512, 1, 0, 1), (attn.KIND_SHARED, 100, 100, 48, 8, 128, 2500, 5, 2000, 4)])
def test_splits_that_were_measured(kind, rows, seqs, heads, kv_heads, dim, keys, groups, prefix, splits):
    assert f"splits={splits}" in attn.describe(kind, rows, seqs, heads, kv_heads, dim, keys, groups, prefix)
