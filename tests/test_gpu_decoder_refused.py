"""A decoder's step whose cache has no room (StepCache.reserve, then LayerProjections.attend in every layer): the cached
keys and values stay, and the same step, tried again with room, answers as if the first try had not been."""
import pytest
import torch

from nebula_amd import attn, decoder as D, hq

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_refused_step_and_its_second_try(cuda, dtype):
    gen = torch.Generator(device="cuda").manual_seed(4)
    layers = [D.random_layer("attention", gen) for _ in range(2)]
    new = lambda n: torch.randn(n, D.EMBEDDING, generator=gen, device="cuda").to(dtype)  # noqa: E731
    row_of = {1: 0, 2: 1, 3: 2}
    cache = attn.KVCache.create(2, 6, 16, D.KV_HEADS, D.HEAD_DIM, 3, 8, dtype)

    def run(chunks, x):
        step = D.StepCache(D.StepRows(chunks), row_of)
        step.reserve(cache)
        return [layer.attend(x, cache, li, step) for li, layer in enumerate(layers)]

    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    run([D.Chunk(1, 0, 32, True)], new(32))
    cache.fork(i32(0), i32(1))  # both hold the two full pages
    run([D.Chunk(3, 0, 49, True)], new(49))
    cache.check()
    before = [t.clone() for t in (cache.k, cache.v, cache.table, cache.lens, cache.refs)]
    decode, x = [D.Chunk(1, 32, 1, False), D.Chunk(2, 32, 1, False)], new(2)
    run(decode, x)  # two pages for no page left
    with pytest.raises(hq.HQError, match="free pages"):
        cache.check()
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.k, cache.v, cache.table, cache.lens, cache.refs)))
    cache.free(i32(2))
    got = run(decode, x)
    cache.check()
    other = attn.KVCache.create(2, 8, 16, D.KV_HEADS, D.HEAD_DIM, 3, 8, dtype)
    other.k[:, :2], other.v[:, :2] = before[0][:, :2], before[1][:, :2]
    other.table[:2, :2] = before[2][:2, :2]
    other.lens[:2] = 32
    other.refs[:2] = 2
    cache = other
    want = run(decode, x)
    other.check()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
