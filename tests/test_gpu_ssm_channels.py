"""Channels of a head are apart: what one holds, infinite or far larger, costs the others no digits."""
import pytest
import torch

import mixer_oracle as M
from nebula_amd import ssm
from test_gpu_ssm import i32, problem, randn

pytestmark = pytest.mark.gpu

INF = float("inf")
SIZES = [(2, 1, 64, 64), (3, 1, 64, 128), (2, 1, 128, 128), (2, 2, 64, 256)]


def scanned(p, state, T):
    c = ssm.StateCache(ssm=state.clone())
    y = c.scan(0, p["x"], p["dt"], p["A"], p["B"], p["C"], None, i32(0, T), D=p["D"], z=p["z"], dt_bias=p["dt_bias"])
    c.check()
    return y, c.ssm_state[0]


def expected(p, state, T):
    return M.scan(p["x"], p["dt"], p["A"], p["B"], p["C"], state[0], [0], [0, T], p["D"], p["z"], p["dt_bias"], chunk=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [70, 700])
@pytest.mark.parametrize("H,G,P,N", SIZES)
def test_states_of_channels_far_apart(cuda, dtype, T, H, G, P, N):
    """A state that is infinite (as one token with an infinite x leaves it), and states of 1e5 and 1e-5, in neighbouring channels."""
    gen = torch.Generator(device="cuda").manual_seed(N + T)
    p = problem(gen, dtype, T, H, G, P, N, gate=False)
    p["D"], p["A"] = None, p["A"] / 100
    p["x"] = p["x"] * 1e-4  # (the states are what comes out)
    state = randn(gen, torch.float32, 1, 1, H, P, N)
    state[..., 5, :] = INF
    state[..., 6, :] *= 1e5
    state[..., 7, :] *= 1e-5
    state[..., P - 1, :] = -INF
    whole = [i for i in range(P) if i not in (5, P - 1)]
    y, s = scanned(p, state, T)
    want, bound, S, off = expected(p, state, T)
    M.check(y[..., whole], want[..., whole], bound[..., whole], "outputs")
    M.check(s[:, :, whole], S[:, :, whole], off[:, :, whole], "states")
    assert not torch.isfinite(y[..., [5, P - 1]].float()).any() and not torch.isfinite(s[:, :, [5, P - 1]]).any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_prompt_behind_an_infinite_token(cuda, dtype):
    """A token with one infinite channel, then a chunk: that channel is lost, and no other."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    H, G, P, N, T = 2, 1, 64, 128, 100
    p = problem(gen, dtype, T, H, G, P, N)
    c = ssm.StateCache(ssm=3e5 * randn(gen, torch.float32, 1, 1, H, P, N))
    one = {k: v[:1].clone() if v is not None and v.shape[0] == T else v for k, v in p.items()}
    one["x"][0, :, 40] = INF
    c.scan(0, one["x"], one["dt"], one["A"], one["B"], one["C"], D=one["D"], z=one["z"], dt_bias=one["dt_bias"])
    state = c.ssm_state.clone()
    assert torch.isinf(state[..., 40, :]).all() and torch.isfinite(state[..., 41, :]).all()
    y, s = scanned(p, state, T)
    want, bound, S, off = expected(p, state, T)
    whole = [i for i in range(P) if i != 40]
    M.check(y[..., whole], want[..., whole], bound[..., whole], "outputs")
    M.check(s[:, :, whole], S[:, :, whole], off[:, :, whole], "states")
