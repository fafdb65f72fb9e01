"""What LayerProjections.mix gives the state space calls, and attend with a rotary its append: host logic, with the calls recorded."""
import contextlib

import pytest
import torch

from nebula_amd import attn, decoder as D, hq


class Seen:
    page_tokens = 16

    def __init__(self, monkeypatch):
        self.now, self.log = "current", []
        monkeypatch.setattr(torch.cuda, "stream", self.on)
        monkeypatch.setattr(hq, "gemm_fused", self.gemm)
        monkeypatch.setattr(attn, "paged", lambda q, *a, out, **k: self.note("paged"))

    @contextlib.contextmanager
    def on(self, stream):
        before, self.now = self.now, stream
        yield
        self.now = before

    def note(self, what, **k):
        self.log.append((what, self.now, k))

    def gemm(self, fmt, X, segs, group, outs=None, stream=None):
        self.note("projections", columns=[n for _, _, n in segs])
        return [torch.zeros(X.shape[0], n, dtype=X.dtype) for _, _, n in segs]

    def conv(self, layer, x, weight, rows, cu, bias, held, out):
        self.note("conv", x=x, rows=rows.tolist(), cu=None if cu is None else cu.tolist(), held=held.tolist(), out=out)

    def scan(self, layer, x, dt, A, B, C, rows, cu, D, z, dt_bias, held, max_len, out):
        self.note("scan", x=x, B=B, C=C, z=z, dt=dt, rows=rows.tolist(), cu=None if cu is None else cu.tolist(), held=held.tolist(), max_len=max_len, out=out)

    def append(self, *a):
        self.note("append")

    def append_rotated(self, layer, rotary, q, k, v, rows, cu, q_weight, k_weight, eps):
        self.note("append_rotated", rotary=rotary, q=q, rows=rows.tolist(), cu=cu.tolist(), q_weight=q_weight, k_weight=k_weight, eps=eps)
        return q


def layer_of(kind):
    names = [n for grp in D.FUSED_GROUPS[kind] + D.FUSED_GROUPS["ffn"] for n in grp]
    return D.LayerProjections(kind, {n: D.TernaryProjection(*D.SHAPES[n], None, None) for n in names})


def test_widths_fit():
    assert D.SSM_HEADS * D.SSM_HEAD_DIM == D.SSM_GATE == D.MIXER_IN
    assert D.SSM_GATE + 2 * D.SSM_GROUPS * D.SSM_STATE == D.SSM_QKV and D.SSM_STATE == D.SSM_HEAD_DIM


@pytest.mark.parametrize("stream", [None, "side"])
def test_mix(monkeypatch, stream):
    seen, layer = Seen(monkeypatch), layer_of("ssm")
    step = D.StepCache(D.StepRows([D.Chunk(0, 40, 1, False), D.Chunk(1, 50, 1, False), D.Chunk(2, 0, 9, True)]), {0: 4, 1: 1, 2: 2}, device="cpu")
    x, dt = torch.zeros(11, D.EMBEDDING, dtype=torch.float16), torch.zeros(11, 48)
    out = layer.mix(x, dt, D.StateMixer(None, None), seen, 3, step, stream=stream)
    assert out.shape == (11, D.EMBEDDING)
    assert [w for w, _, _ in seen.log] == ["projections", "conv", "scan", "conv", "scan", "projections"]
    assert {s for _, s, _ in seen.log} == {stream or "current"} and seen.now == "current"
    for at, rows, cu, held, most, n in ((1, [4, 1], None, [40, 50], 1, 2), (3, [2], [0, 9], [0], 9, 9)):
        (_, _, c), (_, _, s) = seen.log[at:at + 2]
        assert (c["rows"], c["cu"], c["held"]) == (rows, cu, held) == (s["rows"], s["cu"], s["held"]) and s["max_len"] == most
        assert c["x"].shape == (n, 10240) == c["out"].shape and s["dt"].shape == (n, 48)
        assert s["x"].shape == s["z"].shape == s["out"].shape == (n, 48, 128) and s["B"].shape == s["C"].shape == (n, 16, 128)
        # x, B and C side by side in what the convolution wrote
        first = c["out"].data_ptr()
        assert [s[k].data_ptr() - first for k in "xBC"] == [0, 2 * 6144, 2 * 8192] and s["x"].stride(0) == 10240


def test_steps_of_one_kind(monkeypatch):
    seen, layer = Seen(monkeypatch), layer_of("ssm")
    for chunks in ([D.Chunk(0, 40, 1, False)], [D.Chunk(0, 0, 40, True)]):
        del seen.log[:]
        step = D.StepCache(D.StepRows(chunks), {0: 0}, device="cpu")
        layer.mix(torch.zeros(step.M, D.EMBEDDING), torch.zeros(step.M, 48), D.StateMixer(None, None), seen, 0, step)
        assert [w for w, _, _ in seen.log] == ["projections", "conv", "scan", "projections"]


@pytest.mark.parametrize("stream", [None, "side"])
def test_attend_with_a_rotary(monkeypatch, stream):
    seen, layer = Seen(monkeypatch), layer_of("attention")
    step = D.StepCache(D.StepRows([D.Chunk(0, 40, 1, False), D.Chunk(2, 0, 9, True)]), {0: 4, 2: 2}, device="cpu")
    layer.attend(torch.zeros(10, D.EMBEDDING, dtype=torch.float16), seen, 0, step, stream=stream, rotary="turns", q_weight="wq", k_weight="wk", eps=1e-5)
    assert [w for w, _, _ in seen.log] == ["projections", "append_rotated", "paged", "paged", "projections"]
    assert {s for _, s, _ in seen.log} == {stream or "current"}
    k = seen.log[1][2]
    assert (k["rotary"], k["q_weight"], k["k_weight"], k["eps"], k["rows"], k["cu"]) == ("turns", "wq", "wk", 1e-5, [4, 2], [0, 1, 10])
    assert k["q"].shape == (10, 24, 256)
    with pytest.raises(ValueError, match="rotary"):
        layer.attend(torch.zeros(10, D.EMBEDDING), seen, 0, step, k_weight="wk")
    with pytest.raises(ValueError, match="kind"):
        layer.mix(torch.zeros(10, D.EMBEDDING), torch.zeros(10, 48), None, seen, 0, step)
