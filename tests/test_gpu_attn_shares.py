"""Few rows whose keys are shared between workgroups: the shares follow the lengths that the device finds, so
batches of none to many thousand tokens, of more entries than a wavefront has lanes, of one row, of rows
with several tokens and of groups past a prefix, all against the definition in 64 bits (tests/attn_oracle.py
and its bounds)."""
import math

import numpy as np
import pytest
import torch

from nebula_amd import attn
from test_gpu_attn import BF16, F16, check_cached, check_packed, cum, i32, make_cache, randn

pytestmark = pytest.mark.gpu


def ragged(rng, n, hi, zeros):
    lens = np.exp(rng.uniform(0, math.log(hi), n)).astype(int)
    lens[rng.choice(n, size=min(zeros, n - 1), replace=False)] = 0
    lens[rng.integers(n)] = hi
    return [int(x) for x in lens]


@pytest.mark.parametrize("dtype,D,H,Hkv,page", [(F16, 64, 2, 1, 16), (BF16, 128, 6, 1, 64), (F16, 256, 4, 2, 32), (BF16, 64, 20, 1, 64)])
@pytest.mark.parametrize("batch,hi,zeros", [(2, 5000, 0), (5, 3000, 2), (64, 1500, 5), (67, 1200, 9), (140, 700, 40)])
def test_ragged_single_tokens(cuda, dtype, D, H, Hkv, page, batch, hi, zeros):
    rng = np.random.default_rng(batch + D)
    lens = ragged(rng, batch, hi, zeros)
    gen = torch.Generator(device="cuda").manual_seed(batch)
    c, host = make_cache(gen, dtype, D, Hkv, page, lens, layers=1)
    rows = [int(r) for r in rng.permutation(batch)]
    q = randn(gen, dtype, batch, H, D)
    tiles = batch * Hkv * -(-(H // Hkv) // 16)  # one round of workgroups has to have more places than there are tiles
    assert ("shared" in attn.describe(attn.KIND_PAGED, batch, batch, H, Hkv, D, hi)) == (tiles < (256 if D == 256 else 512))
    out, lse = attn.paged(q, c, 0, i32(rows), max_len=hi, with_lse=True)
    c.check()
    check_cached(out, lse, q, host, 0, rows, np.arange(batch + 1), 1 / math.sqrt(D), f"{lens}")
    again = attn.paged(q, c, 0, i32(rows), max_len=hi)
    attn.paged(q[:1], c, 0, i32(rows[:1]), max_len=hi)
    assert torch.equal(out, again) and torch.equal(out, attn.paged(q, c, 0, i32(rows), max_len=hi))


@pytest.mark.parametrize("D,H,Hkv", [(64, 2, 1), (128, 6, 1), (256, 16, 1), (128, 48, 8)])
@pytest.mark.parametrize("n", [0, 1, 16, 127, 129, 4097, 20000])
def test_one_row(cuda, D, H, Hkv, n):
    gen = torch.Generator(device="cuda").manual_seed(n)
    c, host = make_cache(gen, BF16, D, Hkv, 64, [n], layers=1)
    q = randn(gen, BF16, 1, H, D)
    for cu in (None, i32([0, 1])):
        out, lse = attn.paged(q, c, 0, i32([0]), cu, max_len=max(n, 1), with_lse=True)
        check_cached(out, lse, q, host, 0, [0], [0, 1], 1 / math.sqrt(D), f"{n} tokens")
    out = attn.paged(q, c, 0, i32([0]), i32([0, 0]), out=torch.full_like(q, 3.0), max_len=max(n, 1))  # its one token is of no sequence
    assert bool((out == 3.0).all())


@pytest.mark.parametrize("D,H,Hkv", [(64, 3, 1), (128, 6, 2), (256, 6, 1)])
def test_several_tokens_a_row(cuda, D, H, Hkv):
    rng = np.random.default_rng(D)
    lens = ragged(rng, 70, 900, 6)
    news = [int(min(rng.integers(0, 5), n)) for n in lens]
    news[3], lens[3] = 4, 2  # more new tokens than the row holds: the first see nothing
    gen = torch.Generator(device="cuda").manual_seed(D)
    c, host = make_cache(gen, F16, D, Hkv, 32, lens, layers=1)
    cu = cum(news)
    q = randn(gen, F16, int(cu[-1]), H, D)
    assert "shared" in attn.describe(attn.KIND_PAGED, int(cu[-1]), 70, H, Hkv, D, 900)
    out, lse = attn.paged(q, c, 0, i32(range(70)), i32(cu), max_len=900, with_lse=True)
    c.check()
    check_cached(out, lse, q, host, 0, list(range(70)), cu, 1 / math.sqrt(D), "several tokens")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D,H,Hkv", [(64, 4, 1), (128, 2, 2), (256, 3, 1)])
def test_packed_rows_on_long_keys(cuda, D, H, Hkv, causal):
    rng = np.random.default_rng(D + causal)
    k_lens = ragged(rng, 66, 1000, 4)
    q_lens = [int(rng.integers(0, 4)) for _ in k_lens]
    cu_q, cu_k = cum(q_lens), cum(k_lens)
    gen = torch.Generator(device="cuda").manual_seed(D)
    q, k, v = randn(gen, BF16, int(cu_q[-1]), H, D), randn(gen, BF16, int(cu_k[-1]), Hkv, D), randn(gen, BF16, int(cu_k[-1]), Hkv, D)
    assert "shared" in attn.describe(attn.KIND_PROMPT, int(cu_q[-1]), 66, H, Hkv, D, 1000)
    out, lse = attn.prompt(q, k, v, i32(cu_q), i32(cu_k), causal=causal, max_k=1000, with_lse=True)
    check_packed(out, lse, q, k, v, cu_q, cu_k, causal, 1 / math.sqrt(D), f"causal={causal}")


def test_values_that_are_not_finite(cuda):
    """Infinities among the keys that one row of a batch sees stay that row's."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    lens = [900, 1, 2500, 300]
    c, host = make_cache(gen, BF16, 128, 2, 64, lens, layers=1)
    page, slot = int(host.table[2, 11]), 17
    for pool in (c.v, host.v):
        pool[0, page, 1, slot, 5] = float("inf")
        pool[0, page, 1, slot, 9] = float("nan")
    q = randn(gen, BF16, 4, 12, 128)
    out, lse = attn.paged(q, c, 0, max_len=2500, with_lse=True)
    check_cached(out, lse, q, host, 0, [0, 1, 2, 3], np.arange(5), 1 / math.sqrt(128), "not finite")


@pytest.mark.parametrize("D,H,Hkv", [(64, 4, 1), (128, 6, 1), (256, 6, 2)])
def test_groups_with_long_ends(cuda, D, H, Hkv):
    """Past their prefix the sequences of a group hold none to thousands of tokens."""
    page, prefix = 32, 200
    ends = [1, 2900, 33, 700, 0, 64]
    gen = torch.Generator(device="cuda").manual_seed(D)
    lens = [prefix + n for n in ends]
    c, host = make_cache(gen, F16, D, Hkv, page, lens, layers=1)
    whole = prefix // page
    for lo, hi in ((0, 4), (4, 6)):  # the first row's pages stand for all of its group
        for r in range(lo, hi):
            host.table[r, :whole] = host.table[lo, :whole]
    c.table.copy_(i32(host.table))
    q = randn(gen, F16, 6, H, D)
    assert "shared" in attn.describe(attn.KIND_SHARED, 6, 6, H, Hkv, D, max(lens), 2, prefix)
    out, lse = attn.shared_prefix(q, c, 0, i32(range(6)), i32([0, 4, 6]), i32([prefix, prefix]), max_prefix=prefix, max_len=max(lens), with_lse=True)
    c.check()
    check_cached(out, lse, q, host, 0, list(range(6)), np.arange(7), 1 / math.sqrt(D), "groups")
