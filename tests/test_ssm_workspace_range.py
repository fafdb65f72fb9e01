"""CPU test of the scan's workspace: what the query gives does not fall as the tokens or max_len grow, and covers what each call uses."""
import re

import pytest

from nebula_amd import ssm

SIZES = [(48, 16, 128, 128), (80, 1, 64, 128), (1, 1, 64, 64), (64, 8, 64, 256), (3, 3, 128, 256), (24, 1, 64, 64)]


@pytest.mark.parametrize("n", [1, 2, 3, 7, 20, 200, 1024])
@pytest.mark.parametrize("H,G,P,N", SIZES)
def test_sizes_over_lengths(n, H, G, P, N):
    before = 0
    for T in sorted({n, n + 1, 3 * n, 5 * n, 8 * n, 9 * n, 64, 65, 100, 128, 500, 1000, 1024, 2046, 4096, 8192, 30000, 100000, 1 << 20}):
        if T < n:
            continue
        sizes = []
        for most in (1, 64, 65, 128, 500, 1000, 5000, T):
            if most <= T:
                sizes.append(ssm.workspace_bytes(T, n, H, G, P, N, max_len=most))
                used = int(re.search(r"ws=(\d+)", ssm.describe(T, n, H, G, P, N, max_len=most))[1])
                assert used <= sizes[-1]
        assert sizes == sorted(sizes) and sizes[-1] == ssm.workspace_bytes(T, n, H, G, P, N) >= before
        before = sizes[-1]
