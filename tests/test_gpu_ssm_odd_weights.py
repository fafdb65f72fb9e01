"""Weights that are not finite are lost where they are used, and nowhere else."""
import pytest
import torch

from nebula_amd import ssm
from test_gpu_ssm import i32, problem, randn

pytestmark = pytest.mark.gpu

ODD = [float("nan"), float("inf"), -float("inf")]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [3, 70, 900])
@pytest.mark.parametrize("odd", ODD)
@pytest.mark.parametrize("what", ["D", "dt_bias"])
def test_of_a_scan(cuda, dtype, T, odd, what):
    gen = torch.Generator(device="cuda").manual_seed(T)
    H, G, P, N = 3, 1, 64, 128
    p = problem(gen, dtype, T, H, G, P, N)
    state = 0.1 * randn(gen, torch.float32, 1, 1, H, P, N)
    bad = p[what].clone()
    bad[1] = odd
    got = []
    for w in (p[what], bad):
        q = {**p, what: w}
        c = ssm.StateCache(ssm=state.clone())
        y = c.scan(0, q["x"], q["dt"], q["A"], q["B"], q["C"], None, i32(0, T), D=q["D"], z=q["z"], dt_bias=q["dt_bias"])
        got.append((y, c.ssm_state[0, 0]))
    (want, want_state), (y, s) = got
    assert torch.equal(y[:, [0, 2]], want[:, [0, 2]]) and torch.equal(s[[0, 2]], want_state[[0, 2]])
    if what == "D":  # no part of the state
        assert torch.equal(s[1], want_state[1]) and not torch.isfinite(y[:, 1].float()).any()
    elif odd == -float("inf"):  # a step of zero: the state as it is
        assert torch.equal(s[1], state[0, 0, 1]) and torch.isfinite(y[:, 1].float()).all()
    else:
        assert not torch.isfinite(s[1]).any() and not torch.isfinite(y[:, 1].float()).any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens", [None, [1, 5, 2], [70, 3]], ids=str)
@pytest.mark.parametrize("odd", ODD)
def test_of_a_convolution(cuda, dtype, lens, odd):
    gen = torch.Generator(device="cuda").manual_seed(1)
    C, W, n = 24, 4, 3 if lens is None else len(lens)
    T = n if lens is None else sum(lens)
    cu = None if lens is None else i32(*([0] + torch.tensor(lens).cumsum(0).tolist()))
    x, w, b, state = randn(gen, dtype, T, C), randn(gen, torch.float32, C, W), randn(gen, torch.float32, C), randn(gen, dtype, 1, n, W - 1, C)
    whole = [i for i in range(C) if i not in (5, 12)]
    got = []
    for value in (0.5, odd):
        w[5, 2], b[12] = value, value
        c = ssm.StateCache(conv=state.clone())
        got.append((c.conv(0, x, w, None, cu, bias=b, silu=False), c.conv_state))
    (want, kept), (y, k) = got
    assert torch.equal(k, kept) and torch.equal(y[:, whole], want[:, whole]) and not torch.isfinite(y[:, [5, 12]].float()).any()
