"""attn.shared_prefix with lists of groups that are not what they have to be (from 0 to the batch's size, not
falling): reported, and every row answers from its own pages, whatever the workspace held before."""
import math

import numpy as np
import pytest
import torch

from nebula_amd import attn, hq
from test_gpu_attn import BF16, F16, check_cached, i32, make_cache, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,D,H,Hkv,page", [(BF16, 128, 12, 2, 16), (F16, 64, 4, 1, 32), (BF16, 256, 6, 1, 16)])
@pytest.mark.parametrize("starts", [[2, 4, 6], [0, 3, 5], [0, 7, 6], [1, 1, 1], [0, 0, 0], [-1, 3, 6], [0, 4, 2, 6], [3, 0, 6]])
def test_rows_of_bad_groups_share_nothing(cuda, dtype, D, H, Hkv, page, starts):
    gen = torch.Generator(device="cuda").manual_seed(len(starts))
    lens = [700, 130, 64, 900, 1, 333]
    c, host = make_cache(gen, dtype, D, Hkv, page, lens)
    q = randn(gen, dtype, 6, H, D)
    rows, groups = list(range(6)), len(starts) - 1
    ws = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    ws[1 << 20:] = 0x7F  # parts of no call (the counters before them stay zero)
    for max_prefix in (0, 600):
        out, lse = attn.shared_prefix(q, c, 1, i32(rows), i32(starts), i32([600] * groups), max_prefix=max_prefix, max_len=900,
                                      with_lse=True, workspace=ws)
        check_cached(out, lse, q, host, 1, rows, np.arange(7), 1 / math.sqrt(D), f"{starts}")
        with pytest.raises(hq.HQError, match="row number"):
            c.check()
    # A sound list through the same workspace.
    out = attn.shared_prefix(q, c, 1, i32(rows), i32([0, 1, 6]), i32([600, 0]), max_prefix=600, max_len=900, workspace=ws)
    check_cached(out, None, q, host, 1, rows, np.arange(7), 1 / math.sqrt(D), "sound")
    c.check()


def test_a_bad_list_of_many_groups(cuda):
    """The list is longer than a wavefront, its fault in the last entries."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    lens = [20 + 3 * i for i in range(100)]
    c, host = make_cache(gen, BF16, 64, 1, 16, lens)
    q = randn(gen, BF16, 100, 2, 64)
    rows = list(range(100))
    starts = list(range(99)) + [97, 100]
    out = attn.shared_prefix(q, c, 0, i32(rows), i32(starts), i32([16] * 100), max_prefix=16, max_len=320)
    check_cached(out, None, q, host, 0, rows, np.arange(101), 0.125, "falling")
    with pytest.raises(hq.HQError, match="row number"):
        c.check()
    starts = list(range(101))
    out = attn.shared_prefix(q, c, 0, i32(rows), i32(starts), i32([16] * 100), max_prefix=16, max_len=320)
    check_cached(out, None, q, host, 0, rows, np.arange(101), 0.125, "sound")
    c.check()
