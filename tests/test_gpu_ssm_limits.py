"""Sizes and hints at their ends: a max_len that is too small, the widest rows, more tokens than a grid's second axis holds."""
import pytest
import torch

import mixer_oracle as M
from nebula_amd import ssm
from test_gpu_ssm import compare, i32, offsets, problem, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[200], [900], [130, 64, 300]], ids=str)
def test_a_max_len_that_is_too_small(cuda, lens):
    gen = torch.Generator(device="cuda").manual_seed(4)
    H, G, P, N, T, rows, cu = 2, 1, 64, 64, sum(lens), list(range(len(lens))), offsets(lens)
    p = problem(gen, torch.bfloat16, T, H, G, P, N)
    state = randn(gen, torch.float32, 1, len(lens), H, P, N)
    for most in (1, 64, 100):
        c = ssm.StateCache(ssm=state.clone())
        got = c.scan(0, p["x"], p["dt"], p["A"], p["B"], p["C"], None, i32(*cu), D=p["D"], z=p["z"], dt_bias=p["dt_bias"], max_len=most)
        c.check()
        compare(c, got, p, state[0], rows, cu, None, f"max_len={most}")


@pytest.mark.parametrize("f32", [True, False])
def test_steps_in_the_widest_rows(cuda, f32):
    gen = torch.Generator(device="cuda").manual_seed(5)
    H, G, P, N, T = 2, 1, 64, 64, 70
    p = problem(gen, torch.float16, T, H, G, P, N, dt_dtype=torch.float32 if f32 else None)
    wide = torch.empty(T * (1 << 22), dtype=p["dt"].dtype, device="cuda").view(T, 1 << 22)[:, :H]
    wide.copy_(p["dt"])
    state = randn(gen, torch.float32, 1, 1, H, P, N)
    got = []
    for dt in (p["dt"], wide):
        c = ssm.StateCache(ssm=state.clone())
        got.append((c.scan(0, p["x"], dt, p["A"], p["B"], p["C"], None, i32(0, T), dt_bias=p["dt_bias"]), c.ssm_state))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_a_convolution_of_two_million_tokens(cuda):
    gen = torch.Generator(device="cuda").manual_seed(6)
    T, C = 65536 * 32 + 5, 8
    x, w = randn(gen, torch.bfloat16, T, C), randn(gen, torch.float32, C, 4)
    c = ssm.StateCache(conv=torch.zeros(1, 1, 3, C, dtype=torch.bfloat16, device="cuda"))
    got = c.conv(0, x, w, None, i32(0, T))
    c.check()
    want, bound, kept = M.conv(x, w, None, torch.zeros(1, 3, C), [0], [0, T])
    M.check(got, want, bound)
    assert torch.equal(c.conv_state[0].double().cpu(), kept)
