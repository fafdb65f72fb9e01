"""Tokens before one whose inputs are not finite answer as without it, in its chunk too; rows that hold infinite states stay apart."""
import pytest
import torch

import mixer_oracle as M
from nebula_amd import ssm
from test_gpu_ssm import i32, problem, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,G,P,N", [(4, 2, 128, 128), (3, 1, 64, 64), (2, 2, 64, 256)])
@pytest.mark.parametrize("what", ["x", "B", "C", "dt", "z"])
def test_tokens_before_an_odd_one(cuda, dtype, H, G, P, N, what):
    gen = torch.Generator(device="cuda").manual_seed(N + P)
    T = 150
    p = problem(gen, dtype, T, H, G, P, N)
    p = {k: v.contiguous() if v is not None else None for k, v in p.items()}
    state = randn(gen, torch.float32, 1, 1, H, P, N)
    want, bound, _, _ = M.scan(p["x"], p["dt"], p["A"], p["B"], p["C"], state[0], [0], [0, T], p["D"], p["z"], p["dt_bias"], chunk=True)
    for at in (1, 17, 40, 63, 64, 100, 149):
        for odd in (float("nan"), float("inf"), -float("inf")):
            q = dict(p)
            q[what] = p[what].clone()
            q[what][at, ..., -1] = odd
            c = ssm.StateCache(ssm=state.clone())
            got = c.scan(0, q["x"], q["dt"], q["A"], q["B"], q["C"], None, i32(0, T), D=q["D"], z=q["z"], dt_bias=q["dt_bias"])
            M.check(got[:at], want[:at], bound[:at], f"{what}[{at}] = {odd}")
            if what in ("C", "z"):  # no part of the state
                after = got[at + 1:]
                M.check(after, want[at + 1:], bound[at + 1:], f"{what}[{at}] = {odd}, after it")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_runs_before_an_odd_one(cuda, dtype):
    """One long sequence, dealt to several workgroups: an odd token in a later run."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    H, G, P, N, T = 2, 1, 64, 64, 900
    assert "twice" in ssm.describe(T, 1, H, G, P, N)
    p = problem(gen, dtype, T, H, G, P, N)
    state = randn(gen, torch.float32, 1, 1, H, P, N)
    want, bound, _, _ = M.scan(p["x"], p["dt"], p["A"], p["B"], p["C"], state[0], [0], [0, T], p["D"], p["z"], p["dt_bias"], chunk=True)
    for what in ("x", "B", "dt"):
        for at in (300, 899):
            q = dict(p)
            q[what] = p[what].clone()
            q[what][at, ..., 0] = float("nan")
            c = ssm.StateCache(ssm=state.clone())
            got = c.scan(0, q["x"], q["dt"], q["A"], q["B"], q["C"], None, i32(0, T), D=q["D"], z=q["z"], dt_bias=q["dt_bias"])
            M.check(got[:at], want[:at], bound[:at], f"{what}[{at}]")
            # what reads it is lost from there on; x's other channels (its first one is odd in both heads) and dt's other head are whole
            assert torch.isnan(got[at, 0].float()).any()
            if what == "x":
                M.check(got[..., 1:], want[..., 1:], bound[..., 1:], f"x[{at}] the other channels")
            if what == "dt":
                M.check(got[:, 1], want[:, 1], bound[:, 1], f"dt[{at}] the other head")
