"""Attention calls over a buffer, or a stream, that a call of the longest keys has made room on."""
import pytest
import torch

from nebula_amd import attn
from test_gpu_attn import BF16, i32, make_cache, randn

pytestmark = pytest.mark.gpu


def test_a_buffer_for_the_longest_serves_shorter_calls(cuda):
    gen = torch.Generator(device="cuda").manual_seed(1)
    c, _ = make_cache(gen, BF16, 128, 8, 64, [8192])
    q, rows, cu = randn(gen, BF16, 64, 48, 128), i32([0]), i32([0, 64])
    ws = torch.zeros(attn.workspace_bytes(attn.KIND_PAGED, 64, 1, 48, 8, 128, 8192), dtype=torch.uint8, device="cuda")
    for max_len in (8192, 8064, 8000, 6000, 777, 64):  # (a hint: the row is as long as it is)
        out = attn.paged(q, c, 0, rows, cu_seqlens=cu, max_len=max_len, workspace=ws)
        assert torch.equal(out, attn.paged(q, c, 0, rows, cu_seqlens=cu, max_len=max_len)), max_len
    assert not bool(ws[:4096].any())  # the counters


def test_a_stream_warmed_up_at_the_longest_captures_shorter_calls(cuda):
    gen = torch.Generator(device="cuda").manual_seed(2)
    c, _ = make_cache(gen, BF16, 128, 8, 64, [8192])
    q, rows, cu = randn(gen, BF16, 64, 48, 128), i32([0]), i32([0, 64])
    out, side = torch.empty_like(q), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    attn.paged(q, c, 0, rows, cu_seqlens=cu, max_len=8192, out=out, stream=side)
    side.synchronize()
    for max_len in (8191, 8064, 8000, 7680, 5184, 4992, 3000, 64):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            attn.paged(q, c, 0, rows, cu_seqlens=cu, max_len=max_len, out=out, stream=side)
        ref = attn.paged(q, c, 0, rows, cu_seqlens=cu, max_len=max_len)
        for r in range(2):
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ref), (max_len, r)
