"""GPU tests of the state space layer's operators (StateCache.conv, StateCache.scan) against their definitions in 64 bits
(tests/mixer_oracle.py)."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

import mixer_oracle as M
from nebula_amd import hq, ssm

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def randn(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def offsets(lens):
    return [0] + np.cumsum(lens).tolist()


# ---------------------------------------------------------------- the convolution
LENS = [
    None,                      # single tokens
    [1], [2], [3], [4], [15], [16], [17], [100],
    [1, 1, 1, 1, 1], [2, 0, 1, 3, 0, 0, 4, 1], [33, 1, 2, 64, 0, 45], [0, 50, 14, 3, 1, 61], [130, 62, 65],
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("C,W", [(8, 4), (520, 4), (1536, 3), (64, 2)])
def test_conv(cuda, dtype, lens, C, W):
    gen = torch.Generator(device="cuda").manual_seed(C + W)
    n = 5 if lens is None else len(lens)
    cu = None if lens is None else offsets(lens)
    T = n if lens is None else cu[-1]
    rows = torch.randperm(n + 3, generator=gen, device="cuda")[:n].tolist()
    held = [3 * (i % 2) for i in range(n)]
    x = randn(gen, dtype, T, C + 16)[:, 8:C + 8]  # a view of wider rows
    w, b = randn(gen, torch.float32, C, W), randn(gen, torch.float32, C)
    state = randn(gen, dtype, 2, n + 3, W - 1, C)
    for bias, act, hold in ((b, True, held), (None, False, None)):
        c = ssm.StateCache(conv=state.clone())
        out = torch.full((T, C), 7.0, dtype=dtype, device="cuda")
        got = c.conv(1, x, w, i32(*rows), None if cu is None else i32(*cu), bias=bias, silu=act, held=None if hold is None else i32(*hold), out=out)
        assert got is out
        c.check()
        want, bound, kept = M.conv(x, w, bias, state[1], rows, cu, hold, act)
        M.check(got, want, bound, f"{lens} act={act}")
        assert torch.equal(c.conv_state[1].double().cpu(), kept)  # kept inputs are inputs, to the bit
        assert torch.equal(c.conv_state[0], state[0])


@pytest.mark.parametrize("T", [70, 1000])
def test_conv_in_pieces_is_the_whole(cuda, T):
    """A prompt in pieces, some of single tokens: the same bits as at once."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    C, W, dtype = 264, 4, torch.bfloat16
    x, w = randn(gen, dtype, T, C), randn(gen, torch.float32, C, W)
    whole = ssm.StateCache(conv=torch.full((1, 1, W - 1, C), float("nan"), dtype=dtype, device="cuda"))
    want = whole.conv(0, x, w, cu_seqlens=i32(0, T), held=i32(0))
    c = ssm.StateCache(conv=torch.full((1, 1, W - 1, C), float("nan"), dtype=dtype, device="cuda"))
    at, parts = 0, []
    for n in (1, 1, 2, 1, 37, 1, 3, T - 46):
        parts.append(c.conv(0, x[at:at + n], w, cu_seqlens=None if n == 1 else i32(0, n), held=i32(at)))
        at += n
    assert at == T and torch.equal(torch.cat(parts), want) and torch.equal(c.conv_state, whole.conv_state)


@pytest.mark.parametrize("lens", [None, [40, 1, 3, 30, 2, 64]], ids=str)
def test_conv_rows_that_are_not_kept(cuda, lens):
    """Rows out of range and repeated ones are computed from zeros and reported, refused ones as usual; none of them is
    written, nor are tokens of no sequence."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    C, W, dtype, n = 136, 4, torch.float16, 6
    cu = None if lens is None else [x + 2 for x in offsets(lens)]
    T = n if lens is None else cu[-1] + 5
    x, w, state = randn(gen, dtype, T, C), randn(gen, torch.float32, C, W), randn(gen, dtype, 1, 8, W - 1, C)
    refused = torch.zeros(8, dtype=torch.int32, device="cuda")
    refused[5] = 1
    c = ssm.StateCache(conv=state.clone(), refused=refused)
    out = torch.full((T, C), 7.0, dtype=dtype, device="cuda")
    rows = [3, 8, 5, 3, -1, 0]
    c.conv(0, x, w, i32(*rows), None if cu is None else i32(*cu), out=out)
    with pytest.raises(hq.HQError, match="row number"):
        c.check()
    c.check()
    padded = torch.cat([state[0], torch.zeros(3, W - 1, C, dtype=dtype, device="cuda")])  # rows 8..10: zeros
    want, bound, kept = M.conv(x, w, None, padded, [3, 8, 5, 9, 10, 0], cu)
    M.check(out, want, bound)
    assert (out.double().cpu()[torch.isnan(want)] == 7).all()
    kept[5] = state[0, 5].double().cpu()
    assert torch.equal(c.conv_state[0].double().cpu(), kept[:8])


# ---------------------------------------------------------------- the scan
def problem(gen, dtype, T, H, G, P, N, dt_dtype=None, gate=True, wide=True, scale=1.0):
    """Inputs as the convolution leaves them: x, B and C views of one row a token."""
    width = H * P + 2 * G * N
    xbc = (scale * F.silu(torch.randn(T, width + (64 if wide else 0), generator=gen, device="cuda"))).to(dtype)
    x = xbc[:, :H * P].unflatten(1, (H, P))
    B, C = (xbc[:, H * P + j * G * N:][:, :G * N].unflatten(1, (G, N)) for j in (0, 1))
    steps = torch.exp(torch.rand(H, generator=gen, device="cuda") * np.log(100) + np.log(0.001))
    return dict(x=x, dt=randn(gen, dt_dtype or dtype, T, H), A=-(1 + 15 * torch.rand(H, generator=gen, device="cuda")), B=B, C=C,
                D=randn(gen, torch.float32, H), z=randn(gen, dtype, T, H, P) if gate else None, dt_bias=torch.log(torch.expm1(steps)))


def run(c, layer, p, rows=None, cu=None, held=None, **kw):
    lists = {k: None if v is None else i32(*v) for k, v in (("rows", rows), ("cu_seqlens", cu), ("held", held))}
    return c.scan(layer, p["x"], p["dt"], p["A"], p["B"], p["C"], D=p["D"], z=p["z"], dt_bias=p["dt_bias"], **lists, **kw)


def in_chunks(T, n, cu, H, G, P, N):
    return "chunk" in ssm.describe(T, n, H, G, P, N, single=cu is None)


def compare(c, got, p, state, rows, cu, held, label="", **kw):
    T, H, P = p["x"].shape
    G, N = p["B"].shape[1:]
    chunk = in_chunks(T, len(rows), cu, H, G, P, N)
    want, bound, S, off = M.scan(p["x"], p["dt"], p["A"], p["B"], p["C"], state, rows, cu, p["D"], p["z"], p["dt_bias"], held=held, chunk=chunk, **kw)
    a = M.check(got, want, bound, label + " outputs")
    b = M.check(c.ssm_state[-1], S, off, label + " states")
    return a, b


SCANS = [None, [1], [2], [7], [63], [64], [65], [200], [2, 0, 1, 3, 70], [130, 1, 0, 129, 64]]
SIZES = [(4, 2, 128, 128), (3, 1, 64, 64), (2, 2, 64, 256), (2, 1, 128, 64), (3, 3, 64, 128), (2, 1, 128, 256)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", SCANS, ids=str)
@pytest.mark.parametrize("H,G,P,N", SIZES)
def test_scan(cuda, dtype, lens, H, G, P, N):
    gen = torch.Generator(device="cuda").manual_seed(H + P + N)
    n = 5 if lens is None else len(lens)
    cu = None if lens is None else offsets(lens)
    T = n if lens is None else cu[-1]
    rows = torch.randperm(n + 2, generator=gen, device="cuda")[:n].tolist()
    held = [5 * (i % 2) for i in range(n)]
    state = 0.1 * randn(gen, torch.float32, 2, n + 2, H, P, N)
    for hold, dt_dtype, gate in ((held, None, True), (None, torch.float32, False)):
        p = problem(gen, dtype, T, H, G, P, N, dt_dtype, gate)
        c = ssm.StateCache(ssm=state.clone())
        out = torch.full((T, H, P), 7.0, dtype=dtype, device="cuda")
        got = run(c, 1, p, rows, cu, hold, out=out)
        assert got is out
        c.check()
        compare(c, got, p, state[1], rows, cu, hold, f"{lens}")
        assert torch.equal(c.ssm_state[0], state[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,G,P,N,lens", [(8, 4, 128, 128, [700]), (8, 4, 128, 128, [3, 1, 1000, 500]), (3, 1, 64, 64, [1029]), (4, 4, 64, 256, [600, 40]),
                                          (2, 1, 128, 256, [513])])
def test_scan_of_sequences_in_runs(cuda, dtype, H, G, P, N, lens):
    """Long sequences whose tokens are dealt to several workgroups, some that continue and some that begin."""
    gen = torch.Generator(device="cuda").manual_seed(12)
    cu, T, n = offsets(lens), sum(lens), len(lens)
    assert "twice" in ssm.describe(T, n, H, G, P, N)
    p = problem(gen, dtype, T, H, G, P, N)
    p["A"] /= 30  # states that last from run to run
    state = 0.1 * randn(gen, torch.float32, 1, n + 1, H, P, N)
    for held in (None, [i % 2 for i in range(n)]):
        c = ssm.StateCache(ssm=state.clone())
        rows = list(range(n))[::-1]
        got = run(c, 0, p, rows, cu, held)
        compare(c, got, p, state[0], rows, cu, held)
        d = ssm.StateCache(ssm=state.clone())  # a workspace of the caller's
        ws = torch.zeros(ssm.workspace_bytes(T, n, H, G, P, N), dtype=torch.uint8, device="cuda")
        assert torch.equal(run(d, 0, p, rows, cu, held, workspace=ws), got) and torch.equal(c.ssm_state, d.ssm_state)
        d = ssm.StateCache(ssm=state.clone())  # (another split, other roundings)
        compare(d, run(d, 0, p, rows, cu, held, workspace=ws, max_len=max(lens)), p, state[0], rows, cu, held)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 5, 150])
def test_scan_without_its_options(cuda, dtype, T):
    """Steps as they are, no skip, gate or bias; out in place of the gate; strong and no decay, zero steps."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    H, P, N = 4, 64, 128
    p = problem(gen, dtype, T, H, 2, P, N, torch.float32)
    p["dt"] = p["dt"].abs()
    p["dt"][T // 2] = 0
    p["A"] = torch.tensor([-1.0, -100.0, 0.0, -1e-4], device="cuda")
    state = randn(gen, torch.float32, 1, 1, H, P, N)
    cu = [0, T]
    c = ssm.StateCache(ssm=state.clone())
    got = c.scan(0, p["x"], p["dt"], p["A"], p["B"], p["C"], cu_seqlens=i32(*cu), softplus=False)
    compare(c, got, {**p, "D": None, "z": None, "dt_bias": None}, state[0], [0], cu, None, softplus=False)
    c = ssm.StateCache(ssm=state.clone())
    z = p["z"].clone()
    other = ssm.StateCache(ssm=state.clone())
    want = run(other, 0, p, cu=cu)
    assert run(c, 0, {**p, "z": z}, cu=cu, out=z) is z
    assert torch.equal(z, want) and torch.equal(c.ssm_state, other.ssm_state)


@pytest.mark.parametrize("scale", [1e-3, 30.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scan_of_small_and_large_inputs(cuda, dtype, scale):
    gen = torch.Generator(device="cuda").manual_seed(4)
    T, H, P, N = 150, 2, 64, 64
    p = problem(gen, dtype, T, H, 1, P, N, scale=scale)
    state = scale ** 2 * randn(gen, torch.float32, 1, 1, H, P, N)
    p["D"], p["z"] = None, None
    c = ssm.StateCache(ssm=state.clone())
    compare(c, run(c, 0, p, cu=[0, T]), p, state[0], [0], [0, T], None)


@pytest.mark.parametrize("lens", [None, [1, 2, 1, 3, 1, 2], [70, 1, 3, 130, 2, 64]], ids=str)
def test_scan_rows_that_are_not_kept(cuda, lens):
    """As test_conv_rows_that_are_not_kept; states that are not read may hold anything, and so may the tokens between sequences."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    H, P, N, dtype, n = 2, 64, 64, torch.bfloat16, 6
    cu = None if lens is None else [x + 2 for x in offsets(lens)]
    T = n if lens is None else cu[-1] + 5
    p = problem(gen, dtype, T, H, 1, P, N)
    if cu:
        for t in list(range(2)) + list(range(cu[-1], T)):
            p["x"][t], p["B"][t], p["C"][t], p["dt"][t], p["z"][t] = (float("nan"),) * 5
    state = 0.1 * randn(gen, torch.float32, 1, 8, H, P, N)
    refused = torch.zeros(8, dtype=torch.int32, device="cuda")
    refused[5] = 1
    rows, held = [3, 8, 5, 3, -1, 0], [1, 1, 1, 1, 1, 0]
    state[0, 0] = float("nan")
    c = ssm.StateCache(ssm=state.clone(), refused=refused)
    out = torch.full((T, H, P), 7.0, dtype=dtype, device="cuda")
    run(c, 0, p, rows, cu, held, out=out)
    with pytest.raises(hq.HQError, match="row number"):
        c.check()
    c.check()
    padded = torch.cat([state[0], torch.zeros(3, H, P, N, device="cuda")])
    padded[0] = 0
    chunk = in_chunks(T, n, cu, H, 1, P, N)
    want, bound, S, off = M.scan(p["x"], p["dt"], p["A"], p["B"], p["C"], padded, [3, 8, 5, 9, 10, 0], cu, p["D"], p["z"], p["dt_bias"], held=held,
                                 chunk=chunk)
    M.check(out, want, bound)
    assert (out.double().cpu()[torch.isnan(want)] == 7).all()
    got = c.ssm_state[0]
    M.check(got[[0, 3]], S[[0, 3]], off[[0, 3]], "states")
    assert torch.equal(got[[1, 2, 4, 5, 6, 7]], state[0, [1, 2, 4, 5, 6, 7]])


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_neighbours_odd_values_stay_its_own(cuda, dtype):
    """Infinities and NaN in one sequence, in its state and its tokens, leave the packed ones beside it alone."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    H, P, N, lens = 2, 64, 128, [70, 40, 100]
    cu, T = offsets(lens), sum(lens)
    p = problem(gen, dtype, T, H, 1, P, N)
    state = 0.1 * randn(gen, torch.float32, 1, 3, H, P, N)
    c = ssm.StateCache(ssm=state.clone())
    want = run(c, 0, p, cu=cu)
    odd = {k: v if v is None else v.clone() for k, v in p.items()}
    odd["x"][75], odd["B"][80], odd["C"][90], odd["dt"][100], odd["z"][71] = float("inf"), float("nan"), float("inf"), float("nan"), float("nan")
    bad = state.clone()
    bad[0, 1] = float("nan")
    d = ssm.StateCache(ssm=bad)
    got = run(d, 0, odd, cu=cu)
    for a, b, r in ((0, 70, 0), (110, 210, 2)):
        assert torch.equal(got[a:b], want[a:b]) and torch.equal(d.ssm_state[0, r], c.ssm_state[0, r])
    assert torch.isnan(got[109]).all() and torch.isnan(d.ssm_state[0, 1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_scan_in_pieces(cuda, dtype):
    """A prompt in pieces (chunks, then single tokens): each against 64 bits from the state before it."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    H, G, P, N, T = 6, 2, 128, 128, 300
    p = problem(gen, dtype, T, H, G, P, N)
    c = ssm.StateCache(ssm=torch.full((1, 2, H, P, N), float("nan"), device="cuda"))
    at = 0
    for n in (64, 150, 1, 1, 84):
        part = {k: v[at:at + n] if v is not None and v.shape[0] == T else v for k, v in p.items()}
        before = torch.nan_to_num(c.ssm_state[0].clone())
        cu = None if n == 1 else [0, n]
        got = run(c, 0, part, [1], cu, [at])
        want, bound, S, off = M.scan(part["x"], part["dt"], part["A"], part["B"], part["C"], before, [1], cu, part["D"], part["z"], part["dt_bias"],
                                     held=[at], chunk=in_chunks(n, 1, cu, H, G, P, N))
        M.check(got, want, bound, f"{at}")
        M.check(c.ssm_state[0, 1], S[1], off[1], f"{at} states")
        at += n
    assert torch.isnan(c.ssm_state[0, 0]).all()


def test_streams_and_graphs(cuda):
    """A convolution and the scan behind it on another stream, and captured: replays go on from the states they find."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    H, G, P, N, dtype = 4, 2, 64, 64, torch.bfloat16
    C = H * P + 2 * G * N
    for lens in (None, [3, 150]):
        n = 2
        cu = None if lens is None else i32(*offsets(lens))
        T = n if lens is None else sum(lens)
        w, rows = randn(gen, torch.float32, C, 4), i32(2, 0)
        p = problem(gen, dtype, T, H, G, P, N)
        xbc, y = randn(gen, dtype, T, C), torch.empty(T, H, P, dtype=dtype, device="cuda")
        mid = torch.empty_like(xbc)

        def step(c, stream=None):
            c.conv(0, xbc, w, rows, cu, out=mid, stream=stream)
            x, B, Cm = mid[:, :H * P].unflatten(1, (H, P)), mid[:, H * P:][:, :G * N].unflatten(1, (G, N)), mid[:, H * P + G * N:].unflatten(1, (G, N))
            return c.scan(0, x, p["dt"], p["A"], B, Cm, rows, cu, D=p["D"], z=p["z"], dt_bias=p["dt_bias"], out=y, stream=stream)

        make = lambda: ssm.StateCache.create(1, 3, C, 4, H, P, N, dtype)  # noqa: E731
        a, b = make(), make()
        want = step(a).clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        step(b, s)
        s.synchronize()
        assert torch.equal(y, want) and torch.equal(a.ssm_state, b.ssm_state) and torch.equal(a.conv_state, b.conv_state)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(b)
        for _ in range(3):
            xbc.copy_(randn(gen, dtype, T, C))
            want = step(a).clone()
            y.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want) and torch.equal(a.ssm_state, b.ssm_state) and torch.equal(a.conv_state, b.conv_state)
        b.check()


def test_offsets_that_fall(cuda):
    """Offsets that are not what they should be are clamped: whatever comes out, nothing is touched but the call's own."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    H, P, N, T, dtype = 2, 64, 64, 900, torch.float16
    p = problem(gen, dtype, T, H, 1, P, N)
    for cu in ([0, T, 0, T, -5, 10 * T, 3], [T, T, T, T, T, T, T], [-9, -8, -7, 100, 50, 60, T + 1]):
        c = ssm.StateCache.create(1, 8, 64, 4, H, P, N, dtype)
        out = torch.full((T + 64, H, P), 7.0, dtype=dtype, device="cuda")
        run(c, 0, p, list(range(6)), cu, out=out[:T])
        c.conv(0, p["x"][:, 0].contiguous(), randn(gen, torch.float32, P, 4), i32(*range(6)), i32(*cu))
        torch.cuda.synchronize()
        assert (out[T:] == 7).all() and not c.ssm_state[0, 6:].any() and not c.conv_state[0, 6:].any()


def test_results_are_the_same_every_time(cuda):
    gen = torch.Generator(device="cuda").manual_seed(9)
    H, G, P, N, T = 8, 4, 128, 128, 700
    p = problem(gen, torch.bfloat16, T, H, G, P, N)
    got = []
    for _ in range(3):
        c = ssm.StateCache(ssm=torch.ones(1, 1, H, P, N, device="cuda"))
        got.append((run(c, 0, p, cu=[0, T]), c.ssm_state))
    assert all(torch.equal(a, got[0][0]) and torch.equal(b, got[0][1]) for a, b in got[1:])


def test_refusals(cuda):
    H, G, P, N, T, dtype = 4, 2, 64, 64, 6, torch.float16
    gen = torch.Generator(device="cuda").manual_seed(10)
    C = H * P + 2 * G * N
    c = ssm.StateCache.create(1, 3, C, 4, H, P, N, dtype)
    x, w = randn(gen, dtype, T, C), randn(gen, torch.float32, C, 4)
    p = problem(gen, dtype, T, H, G, P, N)
    cu = i32(0, T)
    scan = lambda layer=0, cu=cu, **kw: (lambda q: c.scan(layer, q["x"], q["dt"], q["A"], q["B"], q["C"], i32(0), cu, D=q["D"], z=q["z"], dt_bias=q["dt_bias"],  # noqa: E731
                                                          **{k: v for k, v in kw.items() if k not in p}))({**p, **kw})
    for bad in (lambda: c.conv(1, x, w, i32(0), cu), lambda: c.conv(0, x, w, i32(0)), lambda: c.conv(0, x, w, i32(0, 1), cu),
                lambda: c.conv(0, x.bfloat16(), w, i32(0), cu), lambda: c.conv(0, x[:, :C - 8], w, i32(0), cu), lambda: c.conv(0, x, w.half(), i32(0), cu),
                lambda: c.conv(0, x, w[:, :3], i32(0), cu), lambda: c.conv(0, x, w, i32(0), cu, out=x), lambda: c.conv(0, x, w, i32(0), cu.long()),
                lambda: c.conv(0, x.cpu(), w, i32(0), cu), lambda: c.conv(0, x, w, i32(0), cu, held=i32(0, 1)), lambda: c.conv(0, x, w, i32(0), cu, bias=w[:8, 0]),
                lambda: c.conv(0, x, w, i32(0), i32()), lambda: c.conv(0, x, w),
                lambda: scan(layer=1), lambda: scan(x=p["x"].bfloat16()), lambda: scan(x=p["x"][:, :3]), lambda: scan(B=p["B"][..., :32]),
                lambda: scan(B=p["B"][:, :1]), lambda: scan(dt=p["dt"][:, :3]), lambda: scan(dt=p["dt"].double()), lambda: scan(A=p["A"].half()),
                lambda: scan(D=p["D"][:3]), lambda: scan(z=p["z"][:3]), lambda: scan(out=p["x"]), lambda: scan(out=p["z"].transpose(0, 1)),
                lambda: scan(cu=None), lambda: scan(B=p["B"][:, [0, 0, 0]], C=p["C"][:, [0, 0, 0]]),
                lambda: ssm.StateCache(), lambda: ssm.StateCache(ssm=c.ssm_state.half()), lambda: ssm.StateCache(conv=c.conv_state, ssm=c.ssm_state[:, :2]),
                lambda: ssm.StateCache(ssm=c.ssm_state.transpose(3, 4)), lambda: ssm.StateCache(conv=c.conv_state, refused=i32(0))):
        with pytest.raises((ValueError, TypeError, hq.HQError)):
            bad()
    c.check()
