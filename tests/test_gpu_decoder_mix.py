"""A decoder's steps through attention layers with rotated heads (LayerProjections.attend with a rotary) and state space
layers (LayerProjections.mix): prompts in chunks beside decode tokens, over one cache and one set of states."""
import pytest
import torch

import mixer_oracle as M
from nebula_amd import attn, decoder as D, hq, rotary, ssm

pytestmark = pytest.mark.gpu

C = D.Chunk


class Model:
    """An attention layer and a state space layer over one residual stream, with weights of their own."""

    def __init__(self, dtype, pages=24, rows=4):
        self.gen, self.dtype = torch.Generator(device="cuda").manual_seed(3), dtype
        r = lambda *s: torch.randn(*s, generator=self.gen, device="cuda")  # noqa: E731
        self.attention, self.ssm = D.random_layer("attention", self.gen), D.random_layer("ssm", self.gen)
        self.rot = rotary.Rotary(64, base=1e7)
        self.wq, self.wk = 1 + 0.1 * r(D.HEAD_DIM), 1 + 0.1 * r(D.HEAD_DIM)
        steps = torch.exp(torch.rand(D.SSM_HEADS, generator=self.gen, device="cuda") * 4.6 - 6.9)
        self.mixer = D.StateMixer(0.5 * r(D.SSM_QKV, 4), -(1 + 15 * torch.rand(D.SSM_HEADS, generator=self.gen, device="cuda")), 0.1 * r(D.SSM_QKV),
                                  1 + 0.1 * r(D.SSM_HEADS), torch.log(torch.expm1(steps)))
        self.cache = attn.KVCache.create(1, pages, 16, D.KV_HEADS, D.HEAD_DIM, rows, 12, dtype)
        self.states = ssm.StateCache.create(1, rows, D.SSM_QKV, 4, D.SSM_HEADS, D.SSM_HEAD_DIM, D.SSM_STATE, dtype, refused=self.cache.refused)
        # what a row holds before its first chunk is not to matter
        self.states.ssm_state.fill_(float("nan"))
        self.states.conv_state.fill_(float("inf"))

    def x(self, n):
        return torch.randn(n, D.EMBEDDING, generator=self.gen, device="cuda").to(self.dtype)

    def dt(self, n):
        return (0.5 * torch.randn(n, D.SSM_HEADS, generator=self.gen, device="cuda")).to(self.dtype)

    def attend(self, x, step, **kw):
        return self.attention.attend(x, self.cache, 0, step, rotary=self.rot, q_weight=self.wq, k_weight=self.wk, **kw)

    def mix(self, x, dt, step, **kw):
        return self.ssm.mix(x, dt, self.mixer, self.states, 0, step, **kw)


STEPS = [[C(7, 0, 40, True)], [C(7, 40, 1, False), C(5, 0, 70, True)], [C(5, 70, 1, False), C(7, 41, 1, False)],
         [C(7, 42, 1, False), C(5, 71, 1, False), C(9, 0, 3, True)], [C(9, 3, 20, True)]]
ROW_OF = {7: 2, 5: 0, 9: 3}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_steps_of_both_layers(cuda, dtype):
    m = Model(dtype)
    other = attn.KVCache.create(1, 24, 16, D.KV_HEADS, D.HEAD_DIM, 4, 12, dtype)
    for chunks in STEPS:
        rows = D.StepRows(chunks)
        step = D.StepCache(rows, ROW_OF)
        step.reserve(m.cache)
        step.reserve(other)
        x, dt = m.x(rows.M), m.dt(rows.M)
        # attention: the same bits as rotation, append and attention one after the other
        got = m.attend(x, step)
        at = torch.cat([torch.arange(c.start_token, c.start_token + c.num_tokens) for c in rows.chunks]).to("cuda", torch.int32)

        def prepare(q_out, k, v):
            q, k, v = q_out[:, :D.MIXER_IN].unflatten(1, (D.HEADS, D.HEAD_DIM)), k.unflatten(1, (D.KV_HEADS, D.HEAD_DIM)), v.unflatten(1, (D.KV_HEADS, D.HEAD_DIM))
            return *rotary.rotate(q, k, m.rot, at, q_weight=m.wq, k_weight=m.wk), v

        assert torch.equal(got, m.attention.attend(x, other, 0, step, prepare=prepare))
        # state space: the convolution's and the scan's definitions on what the projections give
        before = (m.states.conv_state.clone(), m.states.ssm_state.clone())
        seen = {}
        mixer_out = m.ssm.mixer_out
        m.ssm.mixer_out = lambda y: seen.setdefault("out", mixer_out(seen.setdefault("y", y)))
        got = m.mix(x, dt, step)
        del m.ssm.mixer_out
        assert got is seen["out"]
        gate, qkv = m.ssm.mixer_in(x)
        own, cu = [ROW_OF[c.request_id] for c in rows.chunks], rows.offsets + [rows.M]
        held = [c.start_token for c in rows.chunks]
        w = m.mixer
        again = ssm.StateCache(conv=before[0].clone())
        lists = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in (own, cu, held)]
        xbc = again.conv(0, qkv, w.conv_weight, *lists[:2], bias=w.conv_bias, held=lists[2])
        want, bound, kept = M.conv(qkv, w.conv_weight, w.conv_bias, before[0][0], own, cu, held)
        M.check(xbc, want, bound, "convolution")
        assert torch.equal(m.states.conv_state[0, own].double().cpu(), kept[own]) and torch.equal(again.conv_state[0, own], m.states.conv_state[0, own])
        xs, B, Cs = (t.unflatten(1, (-1, 128)) for t in xbc.split([6144, 2048, 2048], 1))
        want, bound, S, off = M.scan(xs, dt, w.A, B, Cs, before[1][0], own, cu, w.D, gate.unflatten(1, (48, 128)), w.dt_bias, held=held, chunk=True)
        M.check(seen["y"].unflatten(1, (48, 128)), want, bound, "scan")
        M.check(m.states.ssm_state[0, own], S[own], off[own], "states")
        left = [r for r in range(4) if r not in own]
        assert torch.equal(m.states.ssm_state[0, left].view(torch.int32), before[1][0, left].view(torch.int32))
        m.cache.check()
        m.states.check()


def test_a_stream_of_the_callers(cuda):
    a, b = Model(torch.bfloat16), Model(torch.bfloat16)
    s = torch.cuda.Stream()
    for chunks in STEPS[:3]:
        rows = D.StepRows(chunks)
        step = D.StepCache(rows, ROW_OF)
        x, dt = a.x(rows.M), a.dt(rows.M)
        step.reserve(a.cache)
        want = a.attend(x, step), a.mix(x, dt, step)
        s.wait_stream(torch.cuda.current_stream())
        step.reserve(b.cache, stream=s)
        got = b.attend(x, step, stream=s), b.mix(x, dt, step, stream=s)
        s.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(got, want))
    assert torch.equal(a.states.ssm_state[0, [0, 2]], b.states.ssm_state[0, [0, 2]])


def test_a_captured_decode_step(cuda):
    """One captured step of both layers, replayed: lengths, pages and states go on as with eager calls."""
    a, b = Model(torch.bfloat16), Model(torch.bfloat16)
    for m in (a, b):
        for chunks in ([C(7, 0, 40, True)], [C(5, 0, 70, True)]):
            rows = D.StepRows(chunks)
            step = D.StepCache(rows, ROW_OF)
            step.reserve(m.cache)
            gen = torch.Generator(device="cuda").manual_seed(rows.M)
            x = torch.randn(rows.M, D.EMBEDDING, generator=gen, device="cuda").to(m.dtype)
            m.attend(x, step)
            m.mix(x, x[:, :D.SSM_HEADS].contiguous(), step)
    step = D.StepCache(D.StepRows([C(7, 40, 1, False), C(5, 70, 1, False)]), ROW_OF)
    step.max_len = 128
    x = a.x(2)
    dt = a.dt(2)

    def run(m):
        step.reserve(m.cache)
        return m.attend(x, step), m.mix(x, dt, step)

    run(a), run(b)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run(b)
    for _ in range(4):
        x.copy_(a.x(2))
        dt.copy_(a.dt(2))
        want = run(a)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(got, want))
        assert torch.equal(a.states.ssm_state[0, [0, 2]], b.states.ssm_state[0, [0, 2]])
    a.cache.check()
    b.cache.check()
    b.states.check()


def test_a_refused_step_leaves_the_states(cuda):
    m = Model(torch.float16, pages=3)
    step = D.StepCache(D.StepRows([C(7, 0, 48, True)]), ROW_OF)
    step.reserve(m.cache)
    x, dt = m.x(48), m.dt(48)
    m.attend(x, step)
    m.mix(x, dt, step)
    m.cache.check()
    m.states.check()
    before = (m.states.conv_state.clone(), m.states.ssm_state.clone())
    step = D.StepCache(D.StepRows([C(7, 48, 1, False)]), ROW_OF)
    step.reserve(m.cache)  # no page left
    m.attend(m.x(1), step)
    m.mix(m.x(1), m.dt(1), step)
    with pytest.raises(hq.HQError, match="free pages"):
        m.cache.check()
    for was, now in zip(before, (m.states.conv_state, m.states.ssm_state)):
        assert torch.equal(was[0, 2], now[0, 2])


def test_refusals(cuda):
    m = Model(torch.float16)
    step = D.StepCache(D.StepRows([C(7, 0, 2, True)]), ROW_OF)
    x, dt = m.x(2), m.dt(2)
    with pytest.raises(ValueError, match="kind"):
        m.attention.mix(x, dt, m.mixer, m.states, 0, step)
    with pytest.raises(ValueError, match="rows"):
        m.mix(x[:1], dt, step)
    with pytest.raises(ValueError, match="rows"):
        m.mix(x, dt[:1], step)
    with pytest.raises(ValueError, match="states"):
        m.mix(x.to(torch.bfloat16), dt, step)
    with pytest.raises(ValueError, match="rotary"):
        m.attention.attend(x, m.cache, 0, step, q_weight=m.wq)
