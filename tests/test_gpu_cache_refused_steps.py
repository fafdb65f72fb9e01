"""A step whose KVCache.reserve was refused writes nothing: cached tokens, tables, lengths and counts stay, and
what is reserved again afterwards goes through. Against the same bookkeeping on the host (tests/attn_oracle.py)."""
import numpy as np
import pytest
import torch

from nebula_amd import hq
from test_gpu_cache import fresh, grow, i32, same

pytestmark = pytest.mark.gpu


def new(c, n):
    gen = torch.Generator(device="cuda").manual_seed(n)
    return [torch.randn(n, c.kv_heads, c.head_dim, generator=gen, device="cuda").to(c.k.dtype) for _ in range(2)]


def refused_step(c, rows, counts, match):
    """reserve, then append in every layer, as a step does; the fault is met at the end."""
    c.reserve(i32(rows), i32(counts))
    cu = np.concatenate([[0], np.cumsum(np.maximum(counts, 0))])
    for layer in range(c.layers):
        k, v = new(c, int(cu[-1]))
        if all(n == 1 for n in counts):
            c.append(layer, k, v, i32(rows))
        else:
            c.append(layer, k, v, i32(rows), cu_seqlens=i32(cu))
    with pytest.raises(hq.HQError, match=match):
        c.check()


@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_a_full_pool_leaves_the_cached_tokens(cuda, order):
    c, h = fresh(pages=6, order=order)
    rng = np.random.default_rng(1)
    grow(c, h, [0, 1], [32, 20], rng)  # 2 + 2 pages, row 0 ends with a full one
    c.fork(i32([0]), i32([2]))  # which row 2 shares
    h.fork([0], [2])
    c.check()
    grow(c, h, [4, 5], [16, 16], rng)  # no page is left
    for rows, counts, why in (([0], [1], "free pages"), ([2, 1], [1, 1], "free pages"), ([1, 0], [12, 5], "free pages"),
                              ([1], [1000], "row of the table"), ([1, 1], [1, 1], "row number"), ([1, 12], [1, 1], "row number"),
                              ([0, 1], [3, -1], "row number")):
        refused_step(c, rows, counts, why)
        same(c, h, f"{rows} {counts}")
    c.free(i32([4]))
    h.free([4])
    grow(c, h, [2, 1], [1, 1], rng)  # the same rows again, with room
    same(c, h, "again")
    grow(c, h, [1, 2], [2, 9], rng)
    same(c, h, "and on")


def test_a_step_beside_a_refused_one(cuda):
    """Two reserves, the second one refused: the first one's rows are written, the second one's are not."""
    c, h = fresh(pages=5)
    rng = np.random.default_rng(2)
    grow(c, h, [0, 1, 3], [30, 16, 16], rng)  # one page is left
    for first, second in ((0, 1), (3, 0)):  # (row 3 takes the last page)
        c.reserve(i32([first]), i32([1]))
        c.reserve(i32([second]), i32([40]))
        h.reserve([first], [1])
        assert h.reserve([second], [40]) == "pages"
        for layer in range(c.layers):
            k, v = new(c, 41)
            c.append(layer, k, v, i32([first, second]), cu_seqlens=i32([0, 1, 41]))
            h.append(layer, k[:1].cpu(), v[:1].cpu(), [first], [0, 1])
        with pytest.raises(hq.HQError, match="free pages"):
            c.check()
        same(c, h, f"{first} {second}")


def test_a_page_of_several_rows_is_not_written(cuda):
    """append without a reserve goes over a row's last tokens, but not where other rows hold them too."""
    c, h = fresh()
    rng = np.random.default_rng(3)
    grow(c, h, [0, 1], [32, 20], rng)
    c.fork(i32([0]), i32([2]))
    h.fork([0], [2])
    k, v = new(c, 2)
    c.append(1, k, v, i32([2, 1]))
    h.append(1, k[1:].cpu(), v[1:].cpu(), [1], [0, 1])
    with pytest.raises(hq.HQError, match="page"):
        c.check()
    same(c, h)
