"""CPU tests of how a shared-prefix call is planned: where the prefixes' lengths are not given, rows' own keys are
shared between workgroups as far as all keys may be theirs; and a step shares no prefix that fills no page."""
import re

import pytest
import torch

import test_decoder_attention_stream as T
from nebula_amd import attn, decoder as D


def grids(rows, heads, kv_heads, dim, keys, prefix):
    text = attn.describe(attn.KIND_SHARED, rows, rows, heads, kv_heads, dim, keys, 1, prefix)
    tile, row, splits = map(int, re.search(r"grid=(\d+)\+(\d+) splits=(\d+)", text).groups())
    return tile, row, splits, "shared" in text


@pytest.mark.parametrize("rows,heads,kv_heads,dim", [(4, 48, 8, 128), (1, 24, 4, 256), (12, 8, 1, 64)])
def test_an_unknown_prefix(rows, heads, kv_heads, dim):
    tile, row, splits, shared = grids(rows, heads, kv_heads, dim, 8192, 0)
    assert (tile, splits) == grids(rows, heads, kv_heads, dim, 8192, 8192)[::2]  # as if all keys were the prefix's
    assert (row, shared) == grids(rows, heads, kv_heads, dim, 8192, 1)[1::2] and shared  # and as if none were
    assert row > grids(rows, heads, kv_heads, dim, 8192, 8192)[1]


@pytest.mark.parametrize("lens,kind", [((0, 0), "paged"), ((15, 3), "paged"), ((0, 16), "shared"), ((64, 64), "shared")])
def test_a_step_without_whole_pages_to_share(monkeypatch, lens, kind):
    weights = {n: D.TernaryProjection(*D.SHAPES[n], None, None) for n in ("attn_q", "attn_k", "attn_v", "attn_output", "ffn_gate", "ffn_up", "ffn_down")}
    rows = D.StepRows([D.Chunk(0, 70, 1, False), D.Chunk(1, 75, 1, False)])
    step = D.StepCache(rows, {0: 0, 1: 1}, [([0], lens[0]), ([1], lens[1])], device="cpu")
    seen = T.Seen(monkeypatch)
    D.LayerProjections("attention", weights).attend(torch.zeros(2, D.EMBEDDING, dtype=torch.float16), seen, 0, step)
    assert [w for w, _ in seen.log if w in ("paged", "shared")] == [kind]
