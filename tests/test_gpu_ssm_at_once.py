"""Scans dealt to several workgroups, whose runs meet in a workspace: two streams at once, and replayed graphs beside eager calls."""
import pytest
import torch

from nebula_amd import ssm
from test_gpu_ssm import i32, offsets, problem, randn

pytestmark = pytest.mark.gpu

H, G, P, N, LENS = 4, 2, 128, 128, [700, 1, 400]


def setup(dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T = sum(LENS)
    assert "twice" in ssm.describe(T, len(LENS), H, G, P, N, max_len=max(LENS))
    p = problem(gen, dtype, T, H, G, P, N)
    return p, randn(gen, torch.float32, 1, 4, H, P, N), i32(*offsets(LENS)), i32(2, 0, 3)


def call(c, p, cu, rows, **kw):
    return c.scan(0, p["x"], p["dt"], p["A"], p["B"], p["C"], rows, cu, D=p["D"], z=p["z"], dt_bias=p["dt_bias"], max_len=max(LENS), **kw)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_two_streams_at_once(cuda, dtype):
    sides = [setup(dtype, seed) for seed in (1, 2)]
    want, states = [], []
    for p, state, cu, rows in sides:
        c = ssm.StateCache(ssm=state.clone())
        want.append([call(c, p, cu, rows) for _ in range(6)])
        states.append(c.ssm_state)
    streams = [torch.cuda.Stream() for _ in sides]
    caches = [ssm.StateCache(ssm=state.clone()) for _, state, _, _ in sides]
    outs = [[torch.empty_like(y) for y in ys] for ys in want]
    torch.cuda.synchronize()
    for i in range(6):  # the steps of both in turn, each stream in its own order
        for s, c, (p, _, cu, rows), out in zip(streams, caches, sides, outs):
            call(c, p, cu, rows, out=out[i], stream=s)
    torch.cuda.synchronize()
    for c, state, got, ys in zip(caches, states, outs, want):
        assert torch.equal(c.ssm_state, state) and all(torch.equal(a, b) for a, b in zip(got, ys))


def test_replays_beside_eager_calls(cuda):
    p, state, cu, rows = setup(torch.bfloat16, 3)
    q, other, _, _ = setup(torch.bfloat16, 4)
    a, b, e = (ssm.StateCache(ssm=t.clone()) for t in (state, state, other))
    size = ssm.workspace_bytes(sum(LENS), len(LENS), H, G, P, N, max_len=max(LENS))
    assert size > 0
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")  # the graph's own
    call(b, p, cu, rows, workspace=ws)
    b.ssm_state.copy_(state)
    y = torch.empty_like(p["x"])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(b, p, cu, rows, out=y, workspace=ws)
    for i in range(4):
        p["x"].copy_(q["x"] * (i + 1) / 4)
        want = call(a, p, cu, rows)
        call(e, q, cu, rows)
        torch.cuda.synchronize()
        g.replay()
        call(e, q, cu, rows)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(a.ssm_state, b.ssm_state)
