"""Attention where a row sees infinite values under weights that round to zero."""
import math

import numpy as np
import pytest
import torch

import attn_oracle as A
from nebula_amd import attn
from test_gpu_attn import BF16, F16, i32, make_cache, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,H,Hkv", [(64, 3, 1), (128, 12, 2), (256, 6, 1)])
@pytest.mark.parametrize("tokens", [1, 64])
def test_infinite_values_of_small_weights(cuda, dtype, D, H, Hkv, tokens):
    """A row sees an infinite value under a weight of exp(-120), whole tiles before its last key: its sum is infinite,
    not a number."""
    gen = torch.Generator(device="cuda").manual_seed(D + tokens)
    n = 300
    c, host = make_cache(gen, dtype, D, Hkv, 16, [n])
    q = randn(gen, dtype, tokens, H, D)
    q[:, :, 0] = 10.0
    at = (17, 100, 201)
    for j, value in zip(at, (math.inf, -math.inf, math.inf)):
        page = int(host.table[0, j // 16])
        for pool in (c.k, host.k):
            pool[1, page, :, j % 16] = 0
            pool[1, page, :, j % 16, 0] = -12.0
        for pool in (c.v, host.v):
            pool[1, page, :, j % 16, 5 + at.index(j) % 2] = value
    out = attn.paged(q, c, 1, i32([0]), cu_seqlens=i32([0, tokens]), max_len=n, scale=1.0)
    for h in range(H):
        g = h // (H // Hkv)
        want = A.attend(q[:, h], host.tokens(host.k, 1, 0, g), host.tokens(host.v, 1, 0, g), np.arange(tokens) + n - tokens + 1, 1.0, dtype)
        assert bool(torch.isinf(want[0][:, 5:7]).all())
        A.check(out[:, h], None, want, f"head {h}")
    c.check()
