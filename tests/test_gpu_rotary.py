"""GPU tests of the rotated heads (rotary.rotate, KVCache.append_rotated) against their definition in 64 bits
(tests/mixer_oracle.py), and of the append against rotate and KVCache.append, whose bits it has to have."""
import numpy as np
import pytest
import torch

import mixer_oracle as M
from nebula_amd import attn, hq, rotary

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def randn(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def angles_of(rot):
    return (rot.turns * (2 * np.pi)).cpu()


SHAPES = [  # tokens, heads, kv heads, head_dim, rotated
    (1, 24, 4, 256, 64), (1, 1, 1, 64, 16), (3, 48, 8, 128, 128), (16, 8, 1, 128, 32), (17, 5, 3, 64, 64), (80, 24, 4, 256, 256),
    (257, 32, 4, 64, 48), (333, 7, 1, 128, 112), (1000, 40, 8, 128, 64),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("T,H,Hkv,D,R", SHAPES)
def test_rotate(cuda, dtype, layout, norm, T, H, Hkv, D, R):
    gen = torch.Generator(device="cuda").manual_seed(T)
    q, k = randn(gen, dtype, T, 2 * H * D)[:, :H * D].view(T, H, D), randn(gen, dtype, T, Hkv, D)
    wq, wk = (1 + 0.3 * randn(gen, torch.float32, D) if norm else None for _ in range(2))
    rot = rotary.Rotary(R, base=500000.0, layout=layout, scaling=rotary.Stretch(8.0, 1024))
    pos = torch.randint(0, 1 << 20, (T,), generator=gen, device="cuda", dtype=torch.int32)
    gq, gk = rotary.rotate(q, k, rot, pos, q_weight=wq, k_weight=wk, eps=1e-5)
    for got, x, w, name in ((gq, q, wq, "q"), (gk, k, wk, "k")):
        M.check(got, *M.rotate(x, pos, angles_of(rot), layout, rot.scale, w, 1e-5), name)
    # q alone, in place, on a view whose neighbours stay as they are.
    wide = randn(gen, dtype, T, H + 2, D)
    before = wide.clone()
    mine = wide[:, 1:H + 1]
    mine.copy_(q)
    assert rotary.rotate(mine, None, rot, pos, q_weight=wq, eps=1e-5, out_q=mine) is mine
    assert torch.equal(mine, gq) and torch.equal(wide[:, 0], before[:, 0]) and torch.equal(wide[:, -1], before[:, -1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_positions_and_values_at_their_ends(cuda, dtype):
    """Positions of both signs up to 31 bits, zeros, the type's largest values, infinities and NaN in one head or the part
    that is not rotated, which leave the others alone."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    T, H, D, R = 9, 4, 128, 32
    q = randn(gen, dtype, T, H, D)
    q[0] = 0
    q[1] *= torch.finfo(dtype).max / 8 / q[1].abs().max()
    q[2] *= torch.finfo(dtype).tiny
    pos = i32(0, 1, 2147483647, -2147483648, -1, 131072, 7, 1000003, 0)
    for layout in rotary.LAYOUTS:
        rot = rotary.Rotary(R, layout=layout)
        M.check(rotary.rotate(q, None, rot, pos), *M.rotate(q, pos, angles_of(rot), layout), layout)
        odd = q.clone()
        odd[3, 1, 0], odd[4, 2, R], odd[5, 0, R + 1] = float("nan"), float("inf"), float("nan")
        got, plain = rotary.rotate(odd, None, rot, pos), rotary.rotate(q, None, rot, pos)
        other = R // 2 if layout == "half" else 1
        assert torch.isnan(got[3, 1, [0, other]]).all() and torch.isinf(got[4, 2, R]) and torch.isnan(got[5, 0, R + 1])
        got[3, 1, [0, other]], got[4, 2, R], got[5, 0, R + 1] = plain[3, 1, [0, other]], plain[4, 2, R], plain[5, 0, R + 1]
        assert torch.equal(got, plain)
    w = torch.ones(D, device="cuda")
    got = rotary.rotate(q, None, rot, pos, q_weight=w, eps=0.0 + 1e-6)
    assert torch.equal(got[0], torch.zeros_like(got[0]))  # a head of zeros has the norm eps


def cache_of(dtype, Hkv, D, page, lens, order="heads", layers=2, spare=2):
    rng = np.random.default_rng(3)
    used = [-(-n // page) for n in lens]
    pages = sum(used) + spare
    table = np.full((len(lens) + 1, max(used) + 1), -1)
    perm, at = rng.permutation(pages), 0
    for i, n in enumerate(used):
        table[i, :n] = perm[at:at + n]
        at += n
    refs = np.bincount(table[table >= 0], minlength=pages)
    gen = torch.Generator(device="cuda").manual_seed(4)
    shape = (layers, pages, Hkv, page, D) if order == "heads" else (layers, pages, page, Hkv, D)
    k, v = randn(gen, dtype, *shape), randn(gen, dtype, *shape)
    if order != "heads":
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    dev = lambda x: torch.from_numpy(np.asarray(x, dtype=np.int32)).cuda()  # noqa: E731
    return attn.KVCache(k, v, dev(table), dev(list(lens) + [0]), dev(refs))


def both(cache, layer, rot, q, k, v, rows, cu, pos, **kw):
    """append_rotated on the cache, and what rotate and append of a copy give."""
    twin = attn.KVCache(cache.k.clone(memory_format=torch.preserve_format), cache.v.clone(memory_format=torch.preserve_format), cache.table.clone(),
                        cache.lens.clone(), cache.refs.clone(), refused=cache.refused.clone())
    want_q, want_k = rotary.rotate(q, k, rot, pos, **kw)
    twin.append(layer, want_k, v, rows, cu)
    got = cache.append_rotated(layer, rot, q, k, v, rows, cu, **kw)
    return got, want_q, twin


CASES = [  # dtype, heads, kv heads, D, R, layout, page, lens, new tokens, order
    (torch.bfloat16, 24, 4, 256, 64, "half", 64, [80, 1, 4096, 333], [1, 1, 1, 1], "heads"),
    (torch.float16, 48, 8, 128, 128, "interleaved", 16, [100, 17], [100, 16], "heads"),
    (torch.bfloat16, 8, 1, 128, 32, "half", 32, [500, 3, 40, 77, 1], [129, 0, 1, 64, 1], "tokens"),
    (torch.float16, 5, 3, 64, 64, "half", 16, [1000], [1000], "tokens"),
    (torch.bfloat16, 16, 2, 256, 256, "interleaved", 128, [1500, 9], [1400, 5], "heads"),
]


@pytest.mark.parametrize("dtype,H,Hkv,D,R,layout,page,lens,new,order", CASES)
@pytest.mark.parametrize("norm", [False, True])
def test_append_rotated_is_rotate_and_append(cuda, dtype, H, Hkv, D, R, layout, page, lens, new, order, norm):
    cache = cache_of(dtype, Hkv, D, page, lens, order)
    gen = torch.Generator(device="cuda").manual_seed(5)
    T = sum(new)
    q, k, v = randn(gen, dtype, T, 2 * H, D)[:, :H], randn(gen, dtype, T, Hkv, D), randn(gen, dtype, T, Hkv, D)
    rows = list(range(len(lens)))[::-1]
    new = new[::-1]
    pos = i32(*[lens[r] - n + t for r, n in zip(rows, new) for t in range(n)])
    cu = None if all(n == 1 for n in new) else i32(*np.concatenate([[0], np.cumsum(new)]).tolist())
    w = dict(q_weight=1 + 0.1 * randn(gen, torch.float32, D), k_weight=1 + 0.1 * randn(gen, torch.float32, D)) if norm else {}
    rot = rotary.Rotary(R, layout=layout)
    got, want, twin = both(cache, 1, rot, q, k, v, i32(*rows), cu, pos, **w)
    cache.check()
    assert torch.equal(got, want) and torch.equal(cache.k, twin.k) and torch.equal(cache.v, twin.v)
    # Keys alone, and q in place.
    cache = cache_of(dtype, Hkv, D, page, lens, order)
    assert cache.append_rotated(1, rot, None, k, v, i32(*rows), cu, **w) is None
    assert torch.equal(cache.k, twin.k) and torch.equal(cache.v, twin.v)
    assert torch.equal(cache.append_rotated(1, rot, q, k, v, i32(*rows), cu, out=q, **w), want)


def test_append_rotated_leaves_alone_what_append_does(cuda):
    """Refused rows, a row out of range, a page of several rows, a bad page, tokens of no sequence."""
    dtype, H, Hkv, D = torch.float16, 6, 2, 64
    cache = cache_of(dtype, Hkv, D, 16, [20, 33, 48, 5, 40])
    cache.refused[1] = 1
    cache.refs[cache.table[2, 2]] = 2
    cache.table[3, 0] = 9999
    gen = torch.Generator(device="cuda").manual_seed(6)
    T = 9
    q, k, v = randn(gen, dtype, T, H, D), randn(gen, dtype, T, Hkv, D), randn(gen, dtype, T, Hkv, D)
    rows, cu = i32(0, 1, 2, 3, 99, 4), i32(1, 2, 4, 5, 6, 7, 8)  # tokens 0 and 8 are no sequence's
    pos = i32(0, 19, 31, 32, 47, 4, 0, 39, 0)
    rot = rotary.Rotary(64)
    out = torch.full_like(q, 7.0)
    want_q, want_k = rotary.rotate(q, k, rot, pos)
    twin = attn.KVCache(cache.k.clone(), cache.v.clone(), cache.table, cache.lens, cache.refs, refused=cache.refused)
    twin.append(0, want_k, v, rows, cu)
    with pytest.raises(hq.HQError):
        twin.check()
    cache.append_rotated(0, rot, q, k, v, rows, cu, out=out)
    with pytest.raises(hq.HQError, match="row number.*page number"):
        cache.check()
    assert torch.equal(cache.k, twin.k) and torch.equal(cache.v, twin.v)
    assert torch.equal(out[1:8], want_q[1:8])
    assert (out[0] == 7).all() and (out[8] == 7).all()
    cache.check()


def test_refusals(cuda):
    rot = rotary.Rotary(64)
    q = torch.zeros(4, 8, 128, dtype=torch.float16, device="cuda")
    pos = i32(0, 1, 2, 3)
    for bad in (lambda: rotary.rotate(q, None, rot, pos[:3]), lambda: rotary.rotate(q, None, rot, pos.long()),
                lambda: rotary.rotate(q.float(), None, rot, pos), lambda: rotary.rotate(q[..., :96], None, rot, pos),
                lambda: rotary.rotate(q, q[:3], rot, pos), lambda: rotary.rotate(q, q.bfloat16(), rot, pos),
                lambda: rotary.rotate(q, None, rotary.Rotary(64, device="cpu"), pos), lambda: rotary.rotate(q, None, rot, pos.cpu()),
                lambda: rotary.rotate(q, None, rot, pos, q_weight=torch.ones(64, device="cuda")),
                lambda: rotary.rotate(q, None, rot, pos, q_weight=torch.ones(128, device="cuda").half()),
                lambda: rotary.rotate(q, None, rot, pos, q_weight=torch.ones(128, device="cuda"), eps=-1.0),
                lambda: rotary.rotate(q, None, rot, pos, out_q=q.transpose(0, 1)), lambda: rotary.rotate(q[..., :64], None, rotary.Rotary(128), pos),
                lambda: rotary.rotate(q[:, :, 1:65], None, rot, pos)):
        with pytest.raises((ValueError, TypeError, hq.HQError)):
            bad()
    cache = cache_of(torch.float16, 2, 128, 16, [20, 30])
    k = torch.zeros(2, 2, 128, dtype=torch.float16, device="cuda")
    for bad in (lambda: cache.append_rotated(0, rot, q, k, k, i32(0, 1)), lambda: cache.append_rotated(0, rot, None, k, k, i32(0)),
                lambda: cache.append_rotated(2, rot, None, k, k, i32(0, 1)), lambda: cache.append_rotated(0, rot, q[:2, :, :64], k, k, i32(0, 1)),
                lambda: cache.append_rotated(0, rot, None, k[:, :1], k, i32(0, 1))):
        with pytest.raises((ValueError, hq.HQError)):
            bad()


def test_streams_and_graphs(cuda):
    """On another stream, and captured: replays follow the lengths that the graph finds, eager work between them."""
    dtype, H, Hkv, D = torch.bfloat16, 8, 2, 128
    cache = cache_of(dtype, Hkv, D, 16, [20, 33])
    gen = torch.Generator(device="cuda").manual_seed(7)
    q, k, v = randn(gen, dtype, 2, H, D), randn(gen, dtype, 2, Hkv, D), randn(gen, dtype, 2, Hkv, D)
    rot, rows, out = rotary.Rotary(32, layout="interleaved"), i32(0, 1), torch.empty(2, H, D, dtype=dtype, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    cache.append_rotated(0, rot, q, k, v, rows, out=out, stream=s)
    s.synchronize()
    assert torch.equal(out, rotary.rotate(q, None, rot, i32(19, 32)))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.append_rotated(0, rot, q, k, v, rows, out=out)
    for step in range(1, 4):
        cache.reserve(rows, i32(1, 1))
        q.copy_(randn(gen, dtype, 2, H, D))
        k.copy_(randn(gen, dtype, 2, Hkv, D))
        g.replay()
        wq, wk = rotary.rotate(q, k, rot, i32(19 + step, 32 + step))
        cache.check()
        assert torch.equal(out, wq)
        for r, at in ((0, 19 + step), (1, 32 + step)):
            page = int(cache.table[r, at // 16])
            assert torch.equal(cache.k[0, page, :, at % 16], wk[r]) and torch.equal(cache.v[0, page, :, at % 16], v[r])
