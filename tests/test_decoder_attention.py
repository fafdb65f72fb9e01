"""What a step's attention layers have in common (nebula_amd.decoder.StepCache), on CPU tensors: host logic."""
import pytest
import torch

from nebula_amd.decoder import HEAD_DIM, HEADS, KV_HEADS, KV_OUT, MIXER_IN, Chunk, StepCache, StepRows


def test_heads_fill_the_projections():
    assert HEADS * HEAD_DIM == MIXER_IN and KV_HEADS * HEAD_DIM == KV_OUT and HEADS % KV_HEADS == 0


def test_lists_of_a_mixed_step():
    rows = StepRows([Chunk(7, 40, 64, True), Chunk(3, 12, 1, False), Chunk(5, 99, 1, False)])
    s = StepCache(rows, {3: 9, 5: 0, 7: 4}, device="cpu")
    assert s.M == 66 and s.decodes == 2 and s.max_len == 104 and s.prefix is None
    for got, want in ((s.rows, [9, 0, 4]), (s.counts, [1, 1, 64]), (s.cu, [0, 1, 2, 66]), (s.decode_rows, [9, 0]),
                      (s.chunk_rows, [4]), (s.chunk_cu, [0, 64])):
        assert got.dtype == torch.int32 and got.is_contiguous() and got.tolist() == want


def test_groups_follow_the_decode_requests():
    rows = StepRows([Chunk(i, 50 + i, 1, False) for i in (4, 2, 6)] + [Chunk(1, 0, 5, True)])
    s = StepCache(rows, {1: 1, 2: 2, 4: 4, 6: 6}, groups=[([4, 2], 48), ([6], 0)], device="cpu")
    starts, lens, most = s.prefix
    assert starts.tolist() == [0, 2, 3] and lens.tolist() == [48, 0] and most == 48
    for bad in ([([2, 4], 48), ([6], 0)], [([4, 2], 48)]):
        with pytest.raises(ValueError):
            StepCache(rows, {1: 1, 2: 2, 4: 4, 6: 6}, groups=bad, device="cpu")


def test_refusals():
    rows = StepRows([Chunk(1, 0, 1, False), Chunk(2, 0, 1, False)])
    with pytest.raises(KeyError):
        StepCache(rows, {1: 0}, device="cpu")
    with pytest.raises(ValueError):
        StepCache(rows, {1: 3, 2: 3}, device="cpu")
