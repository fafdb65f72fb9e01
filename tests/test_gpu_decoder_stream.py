"""LayerProjections.attend on a stream of the caller's, with a prepare and a gate that compute: the same bits as
on the current stream, while the current stream allocates and writes beside it."""
import pytest
import torch

from nebula_amd import attn, decoder as D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_steps_on_a_side_stream(cuda, dtype):
    gen = torch.Generator(device="cuda").manual_seed(2)
    layers = [D.random_layer("attention", gen) for _ in range(2)]
    steps = [[D.Chunk(1, 0, 70, True)], [D.Chunk(1, 70, 1, False), D.Chunk(2, 0, 33, True)],
             [D.Chunk(2, 33, 1, False), D.Chunk(1, 71, 1, False)]]
    xs = [torch.randn(sum(c.num_tokens for c in chunks), D.EMBEDDING, generator=gen, device="cuda").to(dtype) for chunks in steps]

    def prepare(q_out, k, v):
        q, k, v = (t.unflatten(1, (-1, D.HEAD_DIM)) for t in (q_out[:, :D.MIXER_IN], k, v))
        return q * 0.5, k / k.float().norm(dim=-1, keepdim=True).to(k.dtype), v + 1

    def gate(y, q_out):
        return y * torch.sigmoid(q_out[:, D.MIXER_IN:])

    outs = []
    for stream in (None, torch.cuda.Stream()):
        cache = attn.KVCache.create(2, 24, 16, D.KV_HEADS, D.HEAD_DIM, 3, 12, dtype)
        torch.cuda.synchronize()
        ys = []
        for chunks, x in zip(steps, xs):
            step = D.StepCache(D.StepRows(chunks), {1: 2, 2: 0})
            if stream is not None:
                stream.wait_stream(torch.cuda.current_stream())
            step.reserve(cache, stream=stream)
            for li, layer in enumerate(layers):
                ys.append(layer.attend(x, cache, li, step, prepare=prepare, gate=gate, stream=stream))
                if stream is not None:
                    for n in (D.Q_OUT, D.KV_OUT, D.MIXER_IN):  # memory that the step's tensors would have had
                        torch.full((x.shape[0], n), float("nan"), dtype=dtype, device="cuda")
            torch.cuda.synchronize()  # the step's lists are dropped
        cache.check()
        outs.append(ys)
    for a, b in zip(*outs):
        assert bool(torch.isfinite(a).all()) and torch.equal(a, b)
