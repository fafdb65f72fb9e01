"""LayerProjections.attend on the GPU: the projections, the cache and its attention as a decoder's steps
run them. A request's prompt in chunks beside other requests' decode tokens, forks that share its
prefix, freed and compacted pages. Every layer's attention is checked against the definition in 64 bits
on the queries, keys and values that the projections gave (tests/attn_oracle.py, its bounds)."""
import math

import pytest
import torch

import attn_oracle as A
from nebula_amd import attn, decoder as D

pytestmark = pytest.mark.gpu

LAYERS = 2


class Run:
    """Steps over a cache, and every request's queries' answers checked from a record of its keys."""

    def __init__(self, dtype, page_tokens=16, pages=48, rows=6, max_pages=12):
        gen = torch.Generator(device="cuda").manual_seed(11)
        self.gen, self.dtype = gen, dtype
        self.layers = [D.random_layer("attention", gen) for _ in range(LAYERS)]
        self.cache = attn.KVCache.create(LAYERS, pages, page_tokens, D.KV_HEADS, D.HEAD_DIM, rows, max_pages, dtype)
        self.kv = [{} for _ in range(LAYERS)]  # request -> (k, v) [tokens, KV_HEADS, HEAD_DIM], on the host

    def x(self, n):
        return torch.randn(n, D.EMBEDDING, generator=self.gen, device="cuda").to(self.dtype)

    def step(self, chunks, row_of, groups=None, rows_x=None, check=True):
        rows = D.StepRows(chunks)
        step = D.StepCache(rows, row_of, groups)
        step.reserve(self.cache)
        outs, ys = [], []
        x = self.x(rows.M) if rows_x is None else rows_x
        for li, layer in enumerate(self.layers):
            seen = {}

            def prepare(q_out, k, v):
                seen["q"], seen["k"], seen["v"] = (t.unflatten(1, (-1, D.HEAD_DIM)) for t in (q_out[:, :D.MIXER_IN], k, v))
                return seen["q"], seen["k"], seen["v"]

            def gate(y, q_out):
                seen["y"] = y
                return y

            out = layer.attend(x, self.cache, li, step, prepare=prepare, gate=gate)
            plain = layer.mixer_out(seen["y"])
            assert torch.equal(out, plain)
            outs.append(out)
            ys.append(seen["y"])
            if check:
                self.check(li, rows, seen)
        self.cache.check()
        return x, outs, ys

    def check(self, li, rows, seen):
        q, k, v = (seen[n].cpu() for n in "qkv")
        y = seen["y"].unflatten(1, (D.HEADS, D.HEAD_DIM)).cpu()
        for c, at in zip(rows.chunks, rows.offsets):
            own = slice(at, at + c.num_tokens)
            old = self.kv[li].get(c.request_id)
            keys, values = (new[own] if old is None else torch.cat([o, new[own]]) for o, new in zip(old or (None, None), (k, v)))
            assert keys.shape[0] == c.start_token + c.num_tokens
            self.kv[li][c.request_id] = (keys, values)
            limits = torch.arange(c.start_token, c.start_token + c.num_tokens) + 1
            for h in range(D.HEADS):
                g = h // (D.HEADS // D.KV_HEADS)
                want = A.attend(q[own, h], keys[:, g], values[:, g], limits, 1 / math.sqrt(D.HEAD_DIM), self.dtype)
                A.check(y[own, h], None, want, f"layer {li} request {c.request_id} tokens from {c.start_token} head {h}")

    def fork(self, parent, child, row_of):
        i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        self.cache.fork(i32(row_of[parent]), i32(row_of[child]))
        for kv in self.kv:
            kv[child] = kv[parent]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_prompt_its_forks_and_mixed_steps(cuda, dtype):
    run = Run(dtype)
    row_of = {10: 3, 11: 0, 12: 5, 13: 1}
    C = D.Chunk
    run.step([C(10, 0, 40, True)], row_of)                                    # a prompt, its first chunk
    run.step([C(10, 40, 23, True)], row_of)                                   # and its second
    run.fork(10, 11, row_of)
    run.fork(10, 12, row_of)
    decode = [C(r, 63, 1, False) for r in (10, 11, 12)]
    run.step(decode, row_of, groups=[([10, 11, 12], 63)])                     # 48 tokens of whole pages are shared
    decode = [C(r, 64, 1, False) for r in (12, 10, 11)]
    run.step(decode + [C(13, 0, 70, True)], row_of, groups=[([12], 0), ([10, 11], 63)])
    run.step([C(13, 70, 1, False), C(11, 65, 1, False)], row_of)              # no groups
    run.cache.free(torch.tensor([row_of[12]], dtype=torch.int32, device="cuda"))
    run.cache.compact()
    run.step([C(13, 71, 1, False), C(10, 65, 1, False), C(11, 66, 1, False)], row_of, groups=[([13], 0), ([10, 11], 63)])


def test_a_compacted_cache_answers_with_the_same_bits(cuda):
    outs = []
    for compact in (False, True):
        run = Run(torch.bfloat16)
        row_of = {1: 0, 2: 1, 3: 2}
        C = D.Chunk
        run.step([C(1, 0, 33, True)], row_of, check=False)
        run.step([C(2, 0, 50, True)], row_of, check=False)
        run.step([C(3, 0, 18, True)], row_of, check=False)
        if compact:
            run.cache.free(torch.tensor([0], dtype=torch.int32, device="cuda"))
            before = run.cache.table[1:].clone()
            run.cache.compact()
            assert not torch.equal(before, run.cache.table[1:])
        gen = torch.Generator(device="cuda").manual_seed(5)
        x = torch.randn(2, D.EMBEDDING, generator=gen, device="cuda").to(torch.bfloat16)
        outs.append(run.step([C(2, 50, 1, False), C(3, 18, 1, False)], row_of, rows_x=x, check=False)[1])
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_refusals(cuda):
    gen = torch.Generator(device="cuda").manual_seed(1)
    cache = attn.KVCache.create(1, 4, 16, D.KV_HEADS, D.HEAD_DIM, 1, 4, torch.float16)
    rows = D.StepRows([D.Chunk(0, 0, 1, False)])
    step = D.StepCache(rows, {0: 0})
    ssm = D.random_layer("ssm", gen)
    x = torch.zeros(1, D.EMBEDDING, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError):
        ssm.attend(x, cache, 0, step)
    layer = D.random_layer("attention", gen)
    with pytest.raises(ValueError):
        layer.attend(x.expand(2, -1).contiguous(), cache, 0, step)
    with pytest.raises(ValueError):  # the cache holds another type
        layer.attend(x.to(torch.bfloat16), cache, 0, step)
