"""LayerProjections.attend with a stream: every call, the caller's prepare and gate and every tensor made between
them belong to that stream. Host logic, with the calls and the stream recorded."""
import contextlib

import pytest
import torch

from nebula_amd import attn, decoder as D, hq


class Seen:
    def __init__(self, monkeypatch):
        self.now, self.log = "current", []
        monkeypatch.setattr(torch.cuda, "stream", self.on)
        new_empty = torch.Tensor.new_empty
        monkeypatch.setattr(torch.Tensor, "new_empty", lambda t, *a, **k: self.call("allocation", new_empty(t, *a, **k)))
        monkeypatch.setattr(hq, "gemm_fused", self.gemm)
        monkeypatch.setattr(attn, "paged", lambda q, *a, out, stream=None, **k: self.call("paged", out, stream))
        monkeypatch.setattr(attn, "shared_prefix", lambda q, *a, out, stream=None, **k: self.call("shared", out, stream))

    @contextlib.contextmanager
    def on(self, stream):
        before, self.now = self.now, stream
        yield
        self.now = before

    def call(self, what, result, stream=None):
        self.log.append((what, stream if stream is not None else self.now))
        return result

    def gemm(self, fmt, X, segs, group, outs=None, stream=None):
        return self.call("projections", [torch.zeros(X.shape[0], n, dtype=X.dtype) for _, _, n in segs], stream)

    def append(self, layer, k, v, rows, cu, stream=None):
        self.call("append", None, stream)

    page_tokens = 16


@pytest.mark.parametrize("stream", [None, "side"])
@pytest.mark.parametrize("groups", [None, [([0, 1], 32)]])
def test_one_stream_for_all(monkeypatch, stream, groups):
    weights = {n: D.TernaryProjection(*D.SHAPES[n], None, None) for n in ("attn_q", "attn_k", "attn_v", "attn_output", "ffn_gate", "ffn_up", "ffn_down")}
    layer = D.LayerProjections("attention", weights)
    rows = D.StepRows([D.Chunk(0, 40, 1, False), D.Chunk(1, 50, 1, False), D.Chunk(2, 0, 9, True)])
    step = D.StepCache(rows, {0: 0, 1: 1, 2: 2}, groups, device="cpu")
    seen = Seen(monkeypatch)

    def prepare(q_out, k, v):
        seen.call("prepare", None)
        return (t.unflatten(1, (-1, D.HEAD_DIM)) for t in (q_out[:, :D.MIXER_IN], k, v))

    def gate(y, q_out):
        return seen.call("gate", y * 1)

    out = layer.attend(torch.zeros(rows.M, D.EMBEDDING, dtype=torch.float16), seen, 0, step, prepare=prepare, gate=gate, stream=stream)
    assert out.shape == (rows.M, D.EMBEDDING)
    assert [w for w, _ in seen.log] == ["projections", "prepare", "append", "allocation", "paged" if groups is None else "shared", "paged", "gate",
                                        "projections"]
    assert {s for _, s in seen.log} == {stream or "current"}, seen.log
    assert seen.now == "current"
