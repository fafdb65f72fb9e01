"""GPU tests of attn.prompt, attn.paged and attn.shared_prefix against the definition in 64 bits
(tests/attn_oracle.py, whose bounds follow from the roundings that a kernel makes): types, head
layouts, lengths from none to many tiles, strides, empty rows, masked places that hold infinities and
NaN, scattered pages, long pools, streams and graphs."""
import math

import numpy as np
import pytest
import torch

import attn_oracle as A
from nebula_amd import attn, hq

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def randn(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def i32(x):
    return torch.as_tensor(np.asarray(x, dtype=np.int32)).cuda()


def cum(lens):
    return np.concatenate([[0], np.cumsum(lens)])


def check_packed(out, lse, q, k, v, cu_q, cu_k, causal, scale, label, worst_rows=4096):
    """Every row against the oracle, sequence by sequence and head by head."""
    H, Hkv = q.shape[1], k.shape[1]
    q, k, v = q.cpu(), k.cpu(), v.cpu()
    for b in range(len(cu_q) - 1):
        q0, q1, k0, k1 = cu_q[b], cu_q[b + 1], cu_k[b], cu_k[b + 1]
        nq, nk = q1 - q0, k1 - k0
        limits = np.arange(nq) + nk - nq + 1 if causal else np.full(nq, nk)
        if nq == 0:
            continue
        for h in range(H):
            g = h // (H // Hkv)
            want = A.attend(q[q0:q1, h], k[k0:k1, g], v[k0:k1, g], limits, scale, q.dtype)
            A.check(out[q0:q1, h], None if lse is None else lse[q0:q1, h], want, f"{label}: sequence {b} head {h}")


def run_prompt(dtype, D, H, Hkv, q_lens, k_lens=None, causal=True, seed=0, scale=None, spread=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cu_q, cu_k = cum(q_lens), cum(k_lens if k_lens is not None else q_lens)
    q, k, v = randn(gen, dtype, cu_q[-1], H, D) * spread, randn(gen, dtype, cu_k[-1], Hkv, D), randn(gen, dtype, cu_k[-1], Hkv, D)
    out, lse = attn.prompt(q, k, v, i32(cu_q), None if k_lens is None else i32(cu_k), causal=causal, scale=scale, with_lse=True)
    torch.cuda.synchronize()
    check_packed(out, lse, q, k, v, cu_q, cu_k, causal, scale or 1 / math.sqrt(D), f"{dtype} D={D} {H}/{Hkv} {q_lens} {k_lens}")
    return q, k, v, out


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,H,Hkv", [(64, 4, 4), (64, 8, 1), (128, 12, 2), (128, 3, 1), (256, 6, 1), (256, 5, 5), (128, 40, 1)])
@pytest.mark.parametrize("lens", [(1,), (2, 31, 1), (64,), (65, 127), (300, 0, 5), (513,)])
def test_prompts(cuda, dtype, D, H, Hkv, lens):
    run_prompt(dtype, D, H, Hkv, lens, seed=sum(lens) + D)


@pytest.mark.parametrize("dtype,D,H,Hkv", [(F16, 128, 2, 1), (BF16, 64, 2, 2), (BF16, 256, 2, 1)])
def test_a_long_prompt(cuda, dtype, D, H, Hkv):
    run_prompt(dtype, D, H, Hkv, (2111,), seed=5)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,H,Hkv", [(128, 6, 1), (64, 4, 2), (256, 6, 2)])
@pytest.mark.parametrize("q_lens,k_lens", [((64,), (1000,)), ((1, 3, 70), (700, 3, 71)), ((5, 9, 40), (2, 0, 33)), ((4, 0, 2), (0, 7, 130)),
                                           ((1,), (4097,)), ((17, 200), (1900, 333))])
def test_more_or_fewer_keys_than_queries(cuda, dtype, D, H, Hkv, q_lens, k_lens):
    """Chunks over earlier keys; rows that see no key give zeros and -infinity."""
    run_prompt(dtype, D, H, Hkv, q_lens, k_lens, seed=1)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_lens,k_lens", [((33, 128), (257, 0)), ((3,), (1025,)), ((200,), (64,))])
def test_without_the_causal_mask(cuda, dtype, q_lens, k_lens):
    run_prompt(dtype, 128, 6, 2, q_lens, k_lens, causal=False, seed=2)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("spread,scale", [(30.0, None), (1.0, 3.0), (1e-3, 1e-3)])
def test_peaked_and_flat_scores(cuda, dtype, spread, scale):
    """Maxima that move by hundreds along the keys, and weights that are all alike."""
    run_prompt(dtype, 128, 4, 2, (300, 77), seed=3, spread=spread, scale=scale)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rising_scores(cuda, dtype):
    """Every key's score is above all earlier ones by more than the last."""
    n, D = 700, 64
    q = torch.zeros(n, 1, D, dtype=dtype, device="cuda")
    k = torch.zeros_like(q)
    q[:, 0, 0] = 1.0
    k[:, 0, 0] = torch.arange(n, device="cuda").float().mul(0.05).to(dtype)
    v = randn(torch.Generator(device="cuda").manual_seed(1), dtype, n, 1, D)
    out, lse = attn.prompt(q, k, v, i32([0, n]), scale=4.0, with_lse=True)
    check_packed(out, lse, q, k, v, [0, n], [0, n], True, 4.0, "rising")


def test_large_magnitudes(cuda):
    """Scores up to 1e37 in bf16: the largest wins alone, and all of them very negative is no empty row."""
    D = 64
    q = torch.zeros(3, 1, D, dtype=BF16, device="cuda")
    k = torch.zeros(5, 1, D, dtype=BF16, device="cuda")
    q[:, 0, 0] = 1e18
    k[:, 0, 0] = torch.tensor([-1e19, -2e19, -1.5e19, -3e19, -9e18], device="cuda").to(BF16)
    v = torch.arange(5 * D, device="cuda").view(5, 1, D).to(BF16)
    out = attn.prompt(q, k, v, i32([0, 3]), i32([0, 5]), scale=1.0)
    want = torch.stack([v[0, 0], v[0, 0], v[4, 0]])
    assert torch.equal(out[:, 0], want)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), torch.finfo(torch.float16).min])
def test_masked_places_take_no_part(cuda, dtype, bad):
    """Keys and values that only later rows see hold NaN, infinities or the type's lowest value."""
    n, D, H = 150, 128, 3
    gen = torch.Generator(device="cuda").manual_seed(4)
    q, k, v = randn(gen, dtype, n, H, D), randn(gen, dtype, n, 1, D), randn(gen, dtype, n, 1, D)
    for at in (70, 130):
        v[at, 0, 5] = bad
    k2 = k.clone()
    k2[140:] = bad
    v2 = v.clone()
    v2[140:] = bad
    cu = [0, n]
    out, _ = attn.prompt(q, k, v, i32(cu), with_lse=True)
    check_packed(out, None, q, k, v, cu, cu, True, 1 / math.sqrt(D), f"values {bad}")
    out = attn.prompt(q, k2, v2, i32(cu))
    clean = attn.prompt(q, k, v, i32(cu))
    assert torch.equal(torch.nan_to_num(out[:140], 7.0), torch.nan_to_num(clean[:140], 7.0))
    # Rows of another sequence in the same tile.
    out = attn.prompt(q[:90], k2[60:], v2[60:], i32([0, 80, 90]), i32([0, 80, 90]))
    clean = attn.prompt(q[:90], k[60:], v[60:], i32([0, 80, 90]), i32([0, 80, 90]))
    assert torch.equal(torch.nan_to_num(out[:80], 7.0), torch.nan_to_num(clean[:80], 7.0))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_strides(cuda, dtype, D):
    """q a column view with its gate beside it, k and v views of one projection, heads before tokens, out a view."""
    H, Hkv, T = 6, 2, 100
    gen = torch.Generator(device="cuda").manual_seed(6)
    wide = randn(gen, dtype, T, 2 * H * D)
    kv = randn(gen, dtype, T, 2 * Hkv * D + 8)
    cu = [0, 37, 100]
    q = wide[:, H * D:].view(T, H, D)
    k, v = kv[:, :Hkv * D].view(T, Hkv, D), kv[:, Hkv * D:2 * Hkv * D].view(T, Hkv, D)
    ref, lse = attn.prompt(q.contiguous(), k.contiguous(), v.contiguous(), i32(cu), with_lse=True)
    check_packed(ref, lse, q, k, v, cu, cu, True, 1 / math.sqrt(D), "contiguous")
    store = torch.full((H, T + 3, D + 16), 9.0, dtype=dtype, device="cuda")
    out = store[:, 2:T + 2, 8:8 + D].transpose(0, 1)
    got = attn.prompt(q, k, v, i32(cu), out=out)
    assert got is out and torch.equal(out, ref)
    store[:, 2:T + 2, 8:8 + D] = 9.0
    assert bool((store == 9.0).all())
    kt, vt = k.transpose(0, 1).contiguous().transpose(0, 1), v.transpose(0, 1).contiguous().transpose(0, 1)
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(attn.prompt(qt, kt, vt, i32(cu)), ref)


def test_rows_of_no_sequence_are_left_alone(cuda):
    q = randn(torch.Generator(device="cuda").manual_seed(7), F16, 20, 2, 64)
    out = torch.full_like(q, 5.0)
    attn.prompt(q, q, q, i32([3, 10, 18]), out=out)
    assert bool((out[:3] == 5.0).all()) and bool((out[18:] == 5.0).all()) and not bool((out[3:18] == 5.0).any())


# ---------------------------------------------------------------- over the cache
def make_cache(gen, dtype, D, Hkv, page, lens, layers=2, order="heads", spare=3, seed=0):
    rng = np.random.default_rng(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    perm = rng.permutation(pages)
    table = np.full((len(lens) + 1, max(need + [1]) + 1), -1)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = perm[at:at + n]
        at += n
    # What no sequence holds is NaN: free pages, and the places after a last token.
    shape = (layers, pages, Hkv, page, D) if order == "heads" else (layers, pages, page, Hkv, D)
    k, v = (torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    if order != "heads":
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    for r, n in enumerate(lens):
        for j in range(need[r]):
            m = min(page, n - j * page)
            for pool in (k, v):
                pool[:, table[r, j], :, :m] = randn(gen, dtype, layers, Hkv, m, D)
    refs = np.bincount(table[table >= 0], minlength=pages)
    c = attn.KVCache(k, v, i32(table), i32(list(lens) + [0]), i32(refs))
    return c, A.Cache(k.cpu(), v.cpu(), table, list(lens) + [0], refs)


def check_cached(out, lse, q, host, layer, rows, cu, scale, label):
    H, Hkv = q.shape[1], host.k.shape[2]
    for i, r in enumerate(rows):
        a, b = cu[i], cu[i + 1]
        n = int(host.lens[r])
        limits = np.arange(b - a) + n - (b - a) + 1
        for h in range(H):
            g = h // (H // Hkv)
            want = A.attend(q[a:b, h], host.tokens(host.k, layer, r, g), host.tokens(host.v, layer, r, g), limits, scale, q.dtype)
            A.check(out[a:b, h], None if lse is None else lse[a:b, h], want, f"{label}: row {r} head {h}")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,H,Hkv", [(128, 12, 2), (64, 8, 8), (256, 6, 1), (128, 33, 1), (64, 24, 2)])
@pytest.mark.parametrize("page,order", [(16, "heads"), (16, "tokens"), (64, "heads"), (256, "heads")])
def test_single_tokens(cuda, dtype, D, H, Hkv, page, order):
    gen = torch.Generator(device="cuda").manual_seed(page + D)
    lens = [1, 33, 0, 64, 700, 65, 2, 31]
    c, host = make_cache(gen, dtype, D, Hkv, page, lens, order=order)
    rows = [4, 0, 2, 7, 1, 8, 3, 5]  # 2 and 8 hold nothing
    q = randn(gen, dtype, len(rows), H, D)
    for layer, max_len in ((0, 0), (1, 700), (1, 64)):  # the last: a hint that is wrong
        out, lse = attn.paged(q, c, layer, i32(rows), max_len=max_len, with_lse=True)
        check_cached(out, lse, q, host, layer, rows, np.arange(len(rows) + 1), 1 / math.sqrt(D), f"layer {layer}")
    out = attn.paged(q[:3], c, 0)  # rows 0, 1, 2
    check_cached(out, None, q[:3], host, 0, [0, 1, 2], np.arange(4), 1 / math.sqrt(D), "default rows")
    c.check()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,H,Hkv,page", [(128, 12, 2, 16), (64, 4, 4, 64), (256, 6, 1, 32)])
@pytest.mark.parametrize("news", [(64,), (3, 0, 1), (1, 70, 5, 2), (7, 7)])
def test_chunks(cuda, dtype, D, H, Hkv, page, news):
    gen = torch.Generator(device="cuda").manual_seed(sum(news))
    lens = [999, 70, 5, 130]
    c, host = make_cache(gen, dtype, D, Hkv, page, lens)
    rows = list(range(len(news)))
    cu = cum(news)
    q = randn(gen, dtype, cu[-1], H, D)
    out, lse = attn.paged(q, c, 1, i32(rows), cu_seqlens=i32(cu), max_len=999, with_lse=True)
    check_cached(out, lse, q, host, 1, rows, cu, 1 / math.sqrt(D), f"{news}")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,H,Hkv,page", [(128, 12, 2, 64), (64, 8, 8, 16), (256, 6, 1, 32), (128, 20, 1, 16)])
@pytest.mark.parametrize("prefix,groups", [((500,), ((11, 200, 1, 64, 5),)), ((64, 1000, 3), ((1, 2), (100, 1, 30, 7), (90,))),
                                           ((128,), ((0, 0, 3),)), ((0, 70), ((5, 9), (1,)))])
def test_shared_prefixes(cuda, dtype, D, H, Hkv, page, prefix, groups):
    """Sequences forked from one prompt and grown apart; also prefixes of no whole page, and of nothing."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    n = sum(len(g) for g in groups)
    total = sum(prefix) + n * (page + max(max(g) for g in groups) + page)
    c = attn.KVCache.create(1, total // page + 2 * n + 8, page, Hkv, D, n + len(prefix), max(prefix) // page + 4 + 1200 // page, dtype)
    host = A.Cache(c.k.cpu(), c.v.cpu(), c.table.cpu().numpy(), c.lens.cpu().numpy(), c.refs.cpu().numpy())
    batch, starts, at = [], [0], 0

    def grow(row, m):
        if m == 0:
            return
        k, v = randn(gen, dtype, m, Hkv, D), randn(gen, dtype, m, Hkv, D)
        c.reserve(i32([row]), i32([m]))
        c.append(0, k, v, i32([row]), cu_seqlens=i32([0, m]))
        host.reserve([row], [m])
        host.append(0, k.cpu(), v.cpu(), [row], [0, m])

    for g, (p, tails) in enumerate(zip(prefix, groups)):
        parent = n + g
        grow(parent, p)
        kids = list(range(at, at + len(tails)))
        c.fork(i32([parent] * len(kids)), i32(kids))
        host.fork([parent] * len(kids), kids)
        for r, m in zip(kids, tails):
            grow(r, m)
        batch += kids
        at += len(kids)
        starts.append(at)
    c.check()
    assert np.array_equal(c.table.cpu().numpy(), host.table) and np.array_equal(c.refs.cpu().numpy(), host.refs)
    q = randn(gen, dtype, n, H, D)
    for mp, ml in ((0, 0), (max(prefix), int(host.lens.max()))):
        out, lse = attn.shared_prefix(q, c, 0, i32(batch), i32(starts), i32(prefix), max_prefix=mp, max_len=ml, with_lse=True)
        check_cached(out, lse, q, host, 0, batch, np.arange(n + 1), 1 / math.sqrt(D), f"{prefix} {mp}")
    c.check()


def test_a_pool_past_32_bit_offsets(cuda):
    """Pages on both sides of 4 GiB and of 2^32 elements."""
    D, Hkv, page = 128, 2, 64
    size = page * Hkv * D  # elements of a page
    pages = (1 << 32) // size + 40
    k = torch.empty(1, pages, Hkv, page, D, dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    gen = torch.Generator(device="cuda").manual_seed(11)
    used = [pages - 1, 0, (1 << 31) // size, pages - 2, (1 << 31) // size - 1, (1 << 30) // size, 1]
    for p in used:
        k[0, p], v[0, p] = randn(gen, BF16, Hkv, page, D), randn(gen, BF16, Hkv, page, D)
    n = len(used) * page - 9
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[used] = 1
    table = torch.full((2, 8), -1, dtype=torch.int32, device="cuda")
    table[0, :len(used)] = i32(used)
    c = attn.KVCache(k, v, table, i32([n, 0]), refs)
    kk, vv = (torch.cat([p[0, u] for u in used], dim=1).transpose(0, 1)[:n].contiguous() for p in (k, v))
    for m in (1, 3, 64):
        q = randn(gen, BF16, m, 12, D)
        out = attn.paged(q, c, 0, i32([0]), cu_seqlens=i32([0, m]), max_len=n)
        check_packed(out, None, q, kk, vv, [0, m], [0, n], True, 1 / math.sqrt(D), f"{m} tokens")
    out = attn.shared_prefix(q[:1], c, 0, i32([0]), i32([0, 1]), i32([300]), max_prefix=300, max_len=n)
    check_packed(out, None, q[:1], kk, vv, [0, 1], [0, n], True, 1 / math.sqrt(D), "shared")
    src, dst = [pages - 1, 0], [pages - 3, 2]
    c.copy_pages(i32(src), i32(dst))
    for s, d in zip(src, dst):
        assert torch.equal(k[0, s], k[0, d]) and torch.equal(v[0, s], v[0, d])
    c.check()


def test_bad_rows_and_pages_are_reported_and_not_followed(cuda):
    gen = torch.Generator(device="cuda").manual_seed(12)
    for m in (1, 64):
        c, host = make_cache(gen, F16, 64, 1, 16, [200, 100, 90])
        cu = [0, m, 2 * m, 3 * m]
        q = randn(gen, F16, 3 * m, 2, 64)
        attn.paged(q, c, 0, i32([0, 99, 2]), cu_seqlens=i32(cu))
        with pytest.raises(hq.HQError, match="row"):
            c.check()
        out = attn.paged(q, c, 0, i32([0, -1, 2]), cu_seqlens=i32(cu))
        check_cached(out[:m], None, q[:m], host, 0, [0], [0, m], 0.125, "good row beside a bad one")
        assert not bool(out[m:2 * m].any())
        c.status.zero_()
        c.table[0, 3] = 1 << 30
        c.table[2, 1] = -7
        out = attn.paged(q, c, 0, i32([0, 1, 2]), cu_seqlens=i32(cu))
        with pytest.raises(hq.HQError, match="page"):
            c.check()
        check_cached(out[m:2 * m], None, q[m:2 * m], host, 0, [1], [0, m], 0.125, "good table beside bad ones")
        c.check()


# ---------------------------------------------------------------- streams, graphs, determinism
def calls(seed):
    """A call of each kind whose plan meets through a workspace, if one does: [(label, function of out)]."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c, _ = make_cache(gen, BF16, 128, 2, 16, [3000, 40, 900, 0], seed=seed)
    q1, q64 = randn(gen, BF16, 4, 12, 128), randn(gen, BF16, 64, 12, 128)
    k, v = randn(gen, BF16, 2000, 2, 128), randn(gen, BF16, 2000, 2, 128)
    rows, one, cu64, cu_q, cu_k = i32([0, 1, 2, 3]), i32([0]), i32([0, 64]), i32([0, 64]), i32([0, 2000])
    starts, pre = i32([0, 1, 4]), i32([2900, 0])
    return [("decode", q1, lambda out, **kw: attn.paged(q1, c, 0, rows, max_len=3000, out=out, **kw)),
            ("chunk", q64, lambda out, **kw: attn.paged(q64, c, 1, one, cu_seqlens=cu64, max_len=3000, out=out, **kw)),
            ("prompt", q64, lambda out, **kw: attn.prompt(q64, k, v, cu_q, cu_k, out=out, **kw)),
            ("shared", q1, lambda out, **kw: attn.shared_prefix(q1, c, 0, rows, starts, pre, max_prefix=2900, max_len=3000, out=out, **kw))]


def test_repeats_are_the_same_bits(cuda):
    for label, q, f in calls(1):
        ref = f(torch.empty_like(q))
        for _ in range(4):
            assert torch.equal(f(torch.full_like(q, float("nan"))), ref), label


def test_two_streams(cuda):
    torch.cuda.synchronize()
    work = calls(2)
    refs = [f(torch.empty_like(q)) for _, q, f in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[torch.full_like(q, float("nan")) for _, q, _ in work] for _ in streams]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for j in range(len(work)):
            for n, s in enumerate(streams):
                i = j if n == 0 else len(work) - 1 - j
                work[i][2](outs[n][i], stream=s)  # torch's current stream is another
    torch.cuda.synchronize()
    for o in outs:
        for i, r in enumerate(refs):
            assert torch.equal(o[i], r), work[i][0]


def test_graphs(cuda):
    side = torch.cuda.Stream()
    for label, q, f in calls(3):
        ws = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
        ref = f(torch.empty_like(q))
        out = torch.empty_like(q)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f(out, workspace=ws)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            f(out, workspace=ws)
        for r in range(3):
            out.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ref), f"{label}: replay {r}"
            assert torch.equal(f(torch.empty_like(q)), ref), f"{label}: eager after replay {r}"


def test_workspace_queries_are_what_calls_ask_for(cuda):
    c, _ = make_cache(torch.Generator(device="cuda").manual_seed(1), BF16, 128, 2, 16, [3000, 40])
    q = torch.zeros(2, 12, 128, dtype=BF16, device="cuda")
    need = attn.workspace_bytes(attn.KIND_PAGED, 2, 2, 12, 2, 128, 3000)
    if need:
        attn.paged(q, c, 0, max_len=3000, workspace=torch.zeros(need, dtype=torch.uint8, device="cuda"))
        with pytest.raises(hq.HQError) as e:
            attn.paged(q, c, 0, max_len=3000, workspace=torch.zeros(need - 256, dtype=torch.uint8, device="cuda"))
        assert e.value.status == hq.HQ_ERR_WORKSPACE


def test_wrapper_refusals(cuda):
    gen = torch.Generator(device="cuda").manual_seed(1)
    c, _ = make_cache(gen, F16, 64, 1, 16, [20, 5])
    q = randn(gen, F16, 2, 2, 64)
    cu = i32([0, 2])
    for bad in (lambda: attn.prompt(q.float(), q, q, cu), lambda: attn.prompt(q, q.to(BF16), q, cu), lambda: attn.prompt(q, q, q[:1], cu),
                lambda: attn.prompt(q[0], q, q, cu), lambda: attn.prompt(q, q, q, cu.long()), lambda: attn.prompt(q, q, q, cu.cpu()),
                lambda: attn.prompt(q, q, q, cu, out=torch.empty(3, 2, 64, dtype=F16, device="cuda")),
                lambda: attn.prompt(q, q, q, cu, lse=torch.empty(2, 2, dtype=F16, device="cuda")),
                lambda: attn.prompt(q.transpose(1, 2), q, q, cu), lambda: attn.paged(q, c, 0, i32([0])),
                lambda: attn.paged(randn(gen, F16, 2, 2, 128), c, 0), lambda: attn.paged(q.to(BF16), c, 0),
                lambda: attn.shared_prefix(q, c, 0, i32([0, 1]), i32([0, 1, 2]), i32([3])),
                lambda: c.append(0, q, q, i32([0, 1])), lambda: c.reserve(i32([0, 1]), i32([1])),
                lambda: attn.KVCache(c.k, c.v.float(), c.table, c.lens, c.refs), lambda: attn.KVCache(c.k, c.v, c.table, c.lens[:1], c.refs)):
        with pytest.raises((ValueError, TypeError)):
            bad()
    with pytest.raises(hq.HQError):
        attn.paged(q, c, 2)
    with pytest.raises(hq.HQError):
        attn.prompt(q, q, q, cu, scale=0.0)
