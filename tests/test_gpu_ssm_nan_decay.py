"""A head whose decay is no number answers with none, in every kernel of the scan; the heads beside it answer as without it."""
import pytest
import torch

from nebula_amd import ssm
from test_gpu_ssm import i32, problem, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,kernel", [(1, "step"), (3, "step"), (70, "chunk"), (900, "twice")])
@pytest.mark.parametrize("H,G,P,N", [(4, 2, 64, 64), (3, 1, 64, 128), (2, 1, 128, 128), (2, 1, 128, 256)])
def test_a_decay_that_is_nan(cuda, dtype, T, kernel, H, G, P, N):
    assert kernel in ssm.describe(T, 1, H, G, P, N)
    gen = torch.Generator(device="cuda").manual_seed(T + N)
    p = problem(gen, dtype, T, H, G, P, N)
    state = 0.1 * randn(gen, torch.float32, 1, 1, H, P, N)
    bad = p["A"].clone()
    bad[1] = float("nan")
    for held in (None, i32(0)):
        got = []
        for A in (p["A"], bad):
            c = ssm.StateCache(ssm=state.clone())
            y = c.scan(0, p["x"], p["dt"], A, p["B"], p["C"], None, i32(0, T), D=p["D"], z=p["z"], dt_bias=p["dt_bias"], held=held)
            got.append((y, c.ssm_state[0, 0]))
            c.check()
        (want, want_state), (y, s) = got
        others = [h for h in range(H) if h != 1]
        assert torch.isnan(y[:, 1]).all() and torch.isnan(s[1]).all()
        assert torch.equal(y[:, others], want[:, others]) and torch.equal(s[others], want_state[others])


@pytest.mark.parametrize("T", [3, 70, 900])
def test_a_decay_that_forgets_all(cuda, T):
    """exp of minus infinity is 0: a token's own terms are what there is."""
    gen = torch.Generator(device="cuda").manual_seed(T)
    H, P, N = 2, 64, 64
    p = problem(gen, torch.bfloat16, T, H, 1, P, N)
    p["A"][1] = -float("inf")
    c = ssm.StateCache(ssm=randn(gen, torch.float32, 1, 1, H, P, N))
    y = c.scan(0, p["x"], p["dt"], p["A"], p["B"], p["C"], None, i32(0, T), dt_bias=p["dt_bias"])
    step = torch.nn.functional.softplus(p["dt"].double() + p["dt_bias"].double())[:, 1, None]
    f = lambda k: p[k].double()  # noqa: E731
    own = step * f("x")[:, 1] * (f("B")[:, 0] * f("C")[:, 0]).sum(-1, keepdim=True)
    mag = step * f("x")[:, 1].abs() * (f("B")[:, 0] * f("C")[:, 0]).abs().sum(-1, keepdim=True)
    # one rounding to bf16, weights in two parts (2^-15 at most), steps and N products in fp32
    bound = 1.01 * (2.0 ** -8 * own.abs() + (2.0 ** -15 + (N + 30) * 2.0 ** -24) * mag)
    assert ((y[:, 1].double() - own).abs() <= bound).all()
    last = step[-1, :, None] * f("x")[-1, 1, :, None] * f("B")[-1, 0]
    assert ((c.ssm_state[0, 0, 1].double() - last).abs() <= (2.0 ** -22 + 30 * 2.0 ** -24) * last.abs() + 1e-38).all()
