"""CPU test: attention calls refuse an O whose strides put two of its elements in one place, and no other."""
import itertools

import pytest

from nebula_amd import attn, hq
from test_attn_abi import P, cache, call_prompt, io


def status(**kw):
    """Of a call whose list of offsets is misaligned: refused by that if O is not."""
    return call_prompt(io(**kw), kv_heads=1, cu_q=P + 1)


@pytest.mark.parametrize("o_row,o_head", [(128, 128), (256, 128), (128, 256), (6016, 128), (136, 264), (384, 256)])
def test_overlapping_outputs_are_refused(o_row, o_head):
    kw = dict(o_row=o_row, o_head=o_head)
    assert status(**kw) == hq.HQ_ERR_SHAPE and b"overlap" in hq.lib().hq_last_error()
    L = attn._lib()
    assert L.hq_attn_paged(io(**kw), cache(), 0, None, P + 1, 4, 0, None, 0, None) == hq.HQ_ERR_SHAPE
    assert L.hq_attn_shared_prefix(io(**kw), cache(), 0, None, 4, P + 1, P, 1, 0, 0, None, 0, None) == hq.HQ_ERR_SHAPE


def test_every_pair_of_small_strides():
    D = 64
    for rows, heads in ((1, 8), (4, 8), (8, 4), (3, 16), (2, 8)):
        for o_row, o_head in itertools.product(range(64, 640, 40), range(64, 640, 56)):
            at = sorted(t * o_row + h * o_head for t in range(rows) for h in range(heads))
            apart = all(b - a >= D for a, b in zip(at, at[1:]))
            got = status(rows=rows, heads=heads, head_dim=D, q_row=heads * D, q_head=D, o_row=o_row, o_head=o_head)
            assert got == (hq.HQ_ERR_ALIGNMENT if apart else hq.HQ_ERR_SHAPE), (rows, heads, o_row, o_head)


@pytest.mark.parametrize("kw", [dict(o_row=6144, o_head=128), dict(o_row=128, o_head=512), dict(o_row=136, o_head=1 << 20), dict(o_row=1 << 20, o_head=136),
                                dict(rows=1, o_row=0, o_head=128), dict(q_row=128, q_head=128)])
def test_other_layouts_pass(kw):
    assert status(**kw) == hq.HQ_ERR_ALIGNMENT
