"""GPU tests of the cache's page keeping (KVCache.reserve, append, fork, free, copy_pages, compact) against its
rules on the host (tests/attn_oracle.py): every table entry, length, count and pool value is equal."""
import numpy as np
import pytest
import torch

import attn_oracle as A
from nebula_amd import attn, hq

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.as_tensor(np.asarray(x, dtype=np.int32)).cuda()


def fresh(page=16, pages=40, rows=12, max_pages=8, layers=2, Hkv=2, D=64, dtype=torch.bfloat16, order="heads", gap=0):
    """A cache whose pools hold random values everywhere, and its host twin. gap: unused pages between layers."""
    shape = (layers, pages + gap, Hkv, page, D) if order == "heads" else (layers, pages + gap, page, Hkv, D)
    gen = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(shape, generator=gen, device="cuda").to(dtype) for _ in range(2))
    if order != "heads":
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    k, v = k[:, :pages], v[:, :pages]
    z = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")
    c = attn.KVCache(k, v, torch.full((rows, max_pages), -1, dtype=torch.int32, device="cuda"), z(rows), z(pages))
    return c, A.Cache(k.cpu(), v.cpu(), np.full((rows, max_pages), -1), np.zeros(rows), np.zeros(pages))


def same(c, h, label=""):
    assert np.array_equal(c.table.cpu().numpy(), h.table), label
    assert np.array_equal(c.lens.cpu().numpy(), h.lens), label
    assert np.array_equal(c.refs.cpu().numpy(), h.refs), label
    assert torch.equal(c.k.cpu(), h.k) and torch.equal(c.v.cpu(), h.v), label


def grow(c, h, rows, counts, rng, check=True):
    c.reserve(i32(rows), i32(counts))
    h.reserve(rows, counts)
    cu = np.concatenate([[0], np.cumsum(counts)])
    Hkv, D = c.kv_heads, c.head_dim
    for layer in range(c.layers):
        k, v = (torch.from_numpy(rng.standard_normal((cu[-1], Hkv, D)).astype(np.float32)).to(c.k.dtype) for _ in range(2))
        if cu[-1]:
            c.append(layer, k.cuda(), v.cuda(), i32(rows), cu_seqlens=i32(cu))
            h.append(layer, k, v, rows, cu)
    if check:
        c.check()


@pytest.mark.parametrize("kw", [dict(), dict(page=16, pages=300, max_pages=90, Hkv=1), dict(page=64, D=128, dtype=torch.float16),
                                dict(order="tokens", Hkv=3, gap=2), dict(Hkv=1, D=256, page=32), dict(page=16, Hkv=1, layers=1, order="tokens"),
                                dict(pages=9000, page=16, Hkv=1, max_pages=30, layers=1)],
                         ids=lambda kw: "-".join(f"{a}{b}" for a, b in kw.items()) or "plain")
def test_a_life_of_sequences(cuda, kw):
    """Sequences that grow, fork, end and are compacted, in an order of their own."""
    c, h = fresh(**kw)
    rng = np.random.default_rng(3)
    grow(c, h, [3, 0, 7], [17, 1, 40], rng)
    same(c, h, "first")
    grow(c, h, [7, 3, 5], [1, 15, 0], rng)  # ends a page, fills one, adds nothing
    same(c, h, "grown")
    c.fork(i32([7, 3, 7, 0]), i32([1, 2, 4, 6]))
    h.fork([7, 3, 7, 0], [1, 2, 4, 6])
    c.check()
    same(c, h, "forked")
    grow(c, h, [1, 4, 2], [9, 2, 3], rng)
    c.free(i32([7, 0, 11]))  # 11 is empty already
    h.free([7, 0, 11])
    c.check()
    same(c, h, "freed")
    old_k, old_t = c.k.clone(), c.table.clone()
    t, r = torch.full_like(c.table, 77), torch.full_like(c.refs, 77)
    before = h.table.copy(), h.lens.copy(), h.refs.copy()
    got = c.compact(out_table=t, out_refs=r)
    assert got[0] is t and got[1] is r
    h.compact()
    c.check()
    assert torch.equal(c.k.cpu(), h.k) and torch.equal(c.v.cpu(), h.v)
    assert np.array_equal(t.cpu().numpy(), h.table) and np.array_equal(r.cpu().numpy(), h.refs)
    # The old table still reads the old tokens.
    assert torch.equal(c.table, old_t) and np.array_equal(c.refs.cpu().numpy(), before[2])
    held = np.unique(before[0][before[0] >= 0])
    assert torch.equal(c.k[:, torch.from_numpy(held).cuda()], old_k[:, torch.from_numpy(held).cuda()])
    c.compact()  # in place
    same(c, h, "compacted")
    c.compact()  # nothing left to move
    same(c, h, "compacted again")
    live = int((h.refs > 0).sum())
    assert (h.refs[:live] > 0).all() and not h.refs[live:].any()
    grow(c, h, [0, 9], [20, 2], rng)
    c.free(i32(list(range(12))))
    h.free(range(12))
    same(c, h, "all freed")
    assert not h.refs.any()


@pytest.mark.parametrize("live", [0, 1, 4095, 4096, 4097, 9000])
def test_compaction_of_large_pools(cuda, live):
    """Counts past one pass of the planning workgroup, none and all of the pages live."""
    P, rng = 9000, np.random.default_rng(live)
    refs = np.zeros(P, dtype=np.int64)
    refs[rng.permutation(P)[:live]] = rng.integers(1, 5, live)
    table = np.full((3, 64), -1)
    held = np.flatnonzero(refs)
    for i in range(3):
        table[i, :min(64, live)] = rng.permutation(held)[:64]
    k = torch.arange(P, device="cuda").view(1, P, 1, 1, 1).expand(1, P, 1, 16, 64).to(torch.float16).contiguous()
    v = (k + 0.5).contiguous()
    h = A.Cache(k.cpu(), v.cpu(), table, [1024] * 3, refs)
    c = attn.KVCache(k, v, i32(table), i32([1024] * 3), i32(refs))
    c.compact()
    h.compact()
    same(c, h)


def test_reserve_refuses_whole_calls(cuda):
    c, h = fresh(pages=6)
    rng = np.random.default_rng(4)
    grow(c, h, [0, 1], [30, 20], rng)  # 2 + 2 pages
    for rows, counts, why in (([2, 3], [17, 17], "free pages"), ([2, 0], [1, 1000], "row of the table"), ([2, 12], [1, 1], "row number"),
                              ([2, -1], [1, 1], "row number"), ([2, 2], [1, 1], "row number"), ([2, 3], [1, -1], "row number"),
                              ([2], [2 ** 31 - 1], "row of the table")):
        c.reserve(i32(rows), i32(counts))
        with pytest.raises(hq.HQError, match=why):
            c.check()
        same(c, h, f"{rows} {counts}")
    grow(c, h, [2, 3], [16, 16], rng)  # exactly what is left
    same(c, h)


def test_fork_refuses_whole_calls(cuda):
    c, h = fresh(pages=5)
    rng = np.random.default_rng(5)
    grow(c, h, [0, 1], [30, 20], rng)
    for parents, children, why in (([0, 0], [2, 3], "free pages"), ([0], [1], "row number"), ([0, 0], [2, 2], "row number"),
                                   ([0], [12], "row number"), ([-1], [2], "row number"), ([0, 2], [2, 3], "row number"), ([0], [0], "row number")):
        c.fork(i32(parents), i32(children))
        with pytest.raises(hq.HQError, match=why):
            c.check()
        same(c, h, f"{parents} {children}")
    c.fork(i32([0, 5]), i32([2, 3]))  # an empty parent gives an empty child
    h.fork([0, 5], [2, 3])
    c.check()
    same(c, h)


def test_free_and_copy_report_and_skip(cuda):
    c, h = fresh()
    rng = np.random.default_rng(6)
    grow(c, h, [0, 1], [30, 20], rng)
    c.free(i32([1, 1, 99]))
    with pytest.raises(hq.HQError, match="row number"):
        c.check()
    h.free([1])
    same(c, h)
    src, dst = [0, 1, 50, 2], [20, 21, 22, -3]
    c.copy_pages(i32(src), i32(dst))
    with pytest.raises(hq.HQError, match="page number"):
        c.check()
    for pool in (h.k, h.v):
        pool[:, [20, 21]] = pool[:, [0, 1]]
    same(c, h)
    c.append(0, torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda"), i32([5]))
    with pytest.raises(hq.HQError, match="row number"):  # an empty row has no last token
        c.check()
    same(c, h)


def test_many_sequences_at_once(cuda):
    n = attn.MAX_BATCH
    c, h = fresh(page=16, pages=3 * n, rows=2 * n, max_pages=3, layers=1, Hkv=1)
    rng = np.random.default_rng(7)
    rows, counts = rng.permutation(2 * n)[:n], rng.integers(0, 40, n)
    grow(c, h, list(rows), list(counts), rng)
    kids = np.setdiff1d(np.arange(2 * n), rows)
    c.fork(i32(rows), i32(kids))
    h.fork(rows, kids)
    c.check()
    same(c, h)
    c.free(i32(rows))
    h.free(rows)
    c.check()
    same(c, h)


def test_strided_sources_and_single_tokens(cuda):
    c, h = fresh(page=16, Hkv=4, D=128, dtype=torch.float16)
    rows = [2, 5, 0]
    c.reserve(i32(rows), i32([1, 1, 1]))
    h.reserve(rows, [1, 1, 1])
    wide = torch.randn(3, 4 * 128 * 2 + 8, device="cuda").to(torch.float16)
    k, v = wide[:, :512].view(3, 4, 128), wide[:, 512:1024].view(3, 4, 128).transpose(0, 1).contiguous().transpose(0, 1)
    c.append(1, k, v, i32(rows))
    h.append(1, k.cpu(), v.cpu(), rows, [0, 1, 2, 3])
    c.check()
    same(c, h)


def test_graph_of_a_step(cuda):
    """reserve and append recorded once and replayed: each replay is one more token."""
    c, h = fresh(layers=1)
    rng = np.random.default_rng(8)
    grow(c, h, [0, 1, 2], [14, 3, 30], rng)
    rows, ones = i32([0, 1, 2]), i32([1, 1, 1])
    k, v = (torch.randn(3, 2, 64, device="cuda").to(torch.bfloat16) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        c.reserve(rows, ones, stream=side)
        c.append(0, k, v, rows, stream=side)
    for _ in range(4):
        k.normal_()
        v.normal_()
        g.replay()
        h.reserve([0, 1, 2], [1, 1, 1])
        h.append(0, k.cpu(), v.cpu(), [0, 1, 2], [0, 1, 2, 3])
        torch.cuda.synchronize()
        same(c, h)
    c.check()
