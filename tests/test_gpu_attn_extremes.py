"""Attention at the ends of its types' ranges: scores so large that their product with the scale is rounded by
more than a weight's exponent holds."""
import math

import pytest
import torch

import attn_oracle as A
from nebula_amd import attn
from test_gpu_attn import BF16, F16, i32

pytestmark = pytest.mark.gpu


def one_winner(gen, dtype, n, m, D, size):
    """q [n, 1, D], k, v [m, 1, D]: of every row's scores, around +-size, one is above all others by size / 1000 or more."""
    q, k = torch.zeros(n, 1, D, device="cuda"), torch.zeros(m, 1, D, device="cuda")
    side = math.sqrt(size)
    q[:, 0, 0] = side * (1 + torch.rand(n, generator=gen, device="cuda"))
    k[:, 0, 0] = side * (0.5 + 0.4 * torch.rand(m, generator=gen, device="cuda"))
    win = torch.randint(m, (1,), generator=gen, device="cuda")
    k[win, 0, 0] = side
    q[::2] *= -1  # for these rows the least of k wins
    low = (win + 1) % m
    k[low, 0, 0] = 0.4 * side
    v = torch.randn(m, 1, D, generator=gen, device="cuda")
    want = torch.where((torch.arange(n, device="cuda") % 2 == 0)[:, None], v[low, 0], v[win, 0])
    return q.to(dtype), k.to(dtype), v.to(dtype), want.to(dtype)


SIZES = [(F16, s) for s in (1e6, 3e7, 2e8, 4e8, 1e9)] + [(BF16, s) for s in (1e6, 1e9, 5e9, 1e11, 1e15, 1e30)]


@pytest.mark.parametrize("dtype,size", SIZES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_the_largest_score_wins_alone(cuda, dtype, size, D):
    gen = torch.Generator(device="cuda").manual_seed(int(math.log2(size)) + D)
    for m in (5, 200, 900):
        for n in (1, 4, 130):  # the row kernel, alone and with others, and the tile kernel; keys shared between workgroups
            for scale in (1.0, 0.71):
                q, k, v, want = one_winner(gen, dtype, n, m, D, size)
                out, lse = attn.prompt(q, k, v, i32([0, n]), i32([0, m]), causal=False, scale=scale, with_lse=True)
                # The winner's weight and the output are rounded to the type, their sums (of one term) to fp32.
                over = (out[:, 0].double() - want.double()).abs() - (2 * A.U[dtype] + 8 * A.U32) * want.double().abs()
                assert over.max().item() <= 0, (m, n, scale)
                top = scale * (q[:, 0].double() @ k[:, 0].double().T).max(1).values
                # scale, log2 e, their product, its with the score, the logarithm added, ln 2 and its product: 5.5 U32
                assert bool(((lse[:, 0].double() - top).abs() <= 6 * A.U32 * top.abs()).all()), (m, n, scale)
