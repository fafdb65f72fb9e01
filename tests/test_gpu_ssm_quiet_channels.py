"""The state's terms keep their digits in quiet channels beside loud ones, and before an x that is not finite."""
import pytest
import torch

import mixer_oracle as M
from test_gpu_ssm import problem, randn
from test_gpu_ssm_channels import SIZES, expected, scanned

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [64, 100, 700])
@pytest.mark.parametrize("H,G,P,N", SIZES)
def test_quiet_channels_beside_loud_ones(cuda, dtype, T, H, G, P, N):
    gen = torch.Generator(device="cuda").manual_seed(N + T)
    p = problem(gen, dtype, T, H, G, P, N, gate=False)
    p["D"], p["A"] = None, p["A"] / 100
    loud = 2.0 ** -torch.tensor([0, 12, 20, 22, 24, 26, 4, 26], device="cuda").repeat(P // 8)  # 2^14 to 2^-12 of a channel's x
    p["x"] = ((p["x"].float().abs() + 0.5).clamp(max=2) * 2.0 ** 13 * loud).to(dtype)
    p["B"], p["C"] = p["B"].clone(), p["C"] * 2.0 ** -6
    p["dt_bias"] = p["dt_bias"] - 3
    state = torch.zeros(1, 1, H, P, N, device="cuda")
    y, s = scanned(p, state, T)
    want, bound, S, off = expected(p, state, T)
    M.check(y, want, bound, "outputs")
    M.check(s, S, off, "states")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [60, 700])
@pytest.mark.parametrize("H,G,P,N", SIZES)
@pytest.mark.parametrize("odd", [float("inf"), float("nan")])
def test_small_inputs_before_one_that_is_not_finite(cuda, dtype, T, H, G, P, N, odd):
    gen = torch.Generator(device="cuda").manual_seed(N + T)
    p = problem(gen, dtype, T, H, G, P, N, gate=False)
    p["D"], p["A"] = None, p["A"] / 100
    p["x"] = p["x"] * 2.0 ** -12
    state = 2.0 ** -12 * randn(gen, torch.float32, 1, 1, H, P, N)
    p["x"][T - 9, :, 3] = odd
    whole = [i for i in range(P) if i != 3]
    y, s = scanned(p, state, T)
    want, bound, S, off = expected(p, state, T)
    M.check(y[..., whole], want[..., whole], bound[..., whole], "outputs")
    M.check(s[:, :, whole], S[:, :, whole], off[:, :, whole], "states")
    assert not torch.isfinite(s[:, :, 3]).any()
