"""Decays inside a chunk are exact to their own size: what was forgotten before them costs the tokens behind it no digits."""
import pytest
import torch

import mixer_oracle as M
from nebula_amd import ssm
from test_gpu_ssm import i32

pytestmark = pytest.mark.gpu


def recursion(x, dt, A, B, C):
    """Outputs of one head from zero, x [T, P], B and C [T, N], dt [T], all positive: a sum of positive terms is its own magnitude."""
    T = len(dt)
    S, out = torch.zeros(x.shape[1], B.shape[1], dtype=torch.float64), []
    for t in range(T):
        S = torch.exp(dt[t] * A) * S + dt[t] * x[t][:, None] * B[t]
        out.append(S @ C[t])
    return torch.stack(out), S


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("strong", [20.0, 100.0, 150.0, 1000.0])
@pytest.mark.parametrize("H,G,P,N", [(2, 1, 64, 64), (1, 1, 128, 128), (2, 2, 64, 256), (3, 1, 64, 128)])
def test_small_steps_behind_large_ones(cuda, dtype, strong, H, G, P, N):
    gen = torch.Generator(device="cuda").manual_seed(N)
    T, L = 96, 32 if N == 256 else 64
    new = lambda *s: 0.25 + torch.rand(*s, generator=gen, device="cuda")  # noqa: E731
    x, B, C = new(T, H, P).to(dtype), (new(T, G, N) / 64).to(dtype), new(T, G, N).to(dtype)
    dt, A = 0.02 * new(T, H), torch.full((H,), -1.0, device="cuda")
    for begin in range(0, T):
        dt[begin:begin + L // 2] = strong * (0.5 + 0.5 * torch.rand(L // 2, H, generator=gen, device="cuda")) if begin + L <= T else 0.01
    c = ssm.StateCache.create(1, 1, 64, 4, H, P, N, dtype)
    got = c.scan(0, x, dt, A, B, C, None, i32(0, T), softplus=False, held=i32(0))
    c.check()
    f = lambda t: t.double().cpu()  # noqa: E731
    for h in range(H):
        g = h // (H // G)
        y, S = recursion(f(x)[:, h], f(dt)[:, h], -1.0, f(B)[:, g], f(C)[:, g])
        # In fp32: N products and their sums (N / 4 + 8), 64 of a chunk's terms, and decays: an exponent e is off by 4 units of
        # itself (its constant, its product, the sums' two parts), which 2^-e makes 4 at most of a whole one, the exponential 4;
        # 2^-19 of a token's own exponents in a sum's low part; with what three chunks' states add, below 400 units. Weights and
        # states as operands are two parts of 8 bits: 2^-16 of each, 2^-15.
        mag = (2.0 ** -15 + 400 * M.U32 + 2.0 ** -19) * y
        M.check(got[:, h], y, 1.01 * M.rounded(y, mag, dtype), f"head {h}")
        M.check(c.ssm_state[0, 0, h], S, (2.0 ** -22 + 400 * M.U32) * S, f"head {h} state")
