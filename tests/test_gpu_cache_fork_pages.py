"""KVCache.fork where a parent's table holds a page number out of range: no child is made, whichever of the
parent's pages it is (all children or none)."""
import numpy as np
import pytest
import torch

from nebula_amd import hq
from test_gpu_cache import fresh, grow, i32, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [-1, 1 << 30, 40])
@pytest.mark.parametrize("at", [0, 3, 6])
def test_no_child_of_a_bad_parent(cuda, bad, at):
    c, h = fresh(rows=12)
    rng = np.random.default_rng(at)
    grow(c, h, [0, 1, 2], [5, 6 * 16 + 3, 33], rng)
    good = int(h.table[1, at])
    c.table[1, at] = bad
    h.table[1, at] = bad
    for parents, children in (([1], [3]), ([0, 2, 1], [3, 4, 5]), ([2, 1, 1, 0], [6, 7, 8, 9])):
        c.fork(i32(parents), i32(children))
        with pytest.raises(hq.HQError, match="page number"):
            c.check()
        same(c, h, f"{parents}")
    c.fork(i32([0, 2, 2]), i32([3, 4, 5]))  # the others' children
    h.fork([0, 2, 2], [3, 4, 5])
    c.check()
    same(c, h, "without it")
    c.table[1, at] = good
    h.table[1, at] = good
    c.fork(i32([1]), i32([8]))
    h.fork([1], [8])
    c.check()
    same(c, h, "mended")


def test_long_tables_of_many_parents(cuda):
    """Tables longer than a workgroup's wavefronts look at in one go, the bad entry in the last parent's last full page."""
    c, h = fresh(pages=900, rows=60, max_pages=300, layers=1, Hkv=1)
    rng = np.random.default_rng(1)
    counts = [int(x) for x in rng.integers(0, 200, 20)] + [260 * 16 + 7]
    grow(c, h, list(range(21)), counts, rng)
    parents, children = list(range(21)) + [20], list(range(30, 52))
    c.table[20, 259] = 900
    h.table[20, 259] = 900
    c.fork(i32(parents), i32(children))
    with pytest.raises(hq.HQError, match="page number"):
        c.check()
    same(c, h)
    page = int(np.flatnonzero(h.refs == 0)[-1])  # (the page that it was lost its number: another)
    c.table[20, 259] = page
    h.table[20, 259] = page
    c.refs[page] = 1
    h.refs[page] = 1
    c.fork(i32(parents), i32(children))
    h.fork(parents, children)
    c.check()
    same(c, h)


def test_a_workspace_of_the_caller(cuda):
    """Refused and good forks through one buffer, whose counters stay zero."""
    c, h = fresh()
    rng = np.random.default_rng(9)
    grow(c, h, [0, 1], [40, 33], rng)
    ws = torch.zeros(c.workspace_bytes(), dtype=torch.uint8, device="cuda")
    for n, (parents, children, why) in enumerate((([0, 1], [2, 3], None), ([1], [2], "row number"), ([1, 0], [4, 5], "page number"),
                                                  ([0], [6], "page number"), ([1, 1, 0], [7, 8, 9], None))):
        if why == "page number":
            c.table[0, 1] = 77
        c.fork(i32(parents), i32(children), workspace=ws)
        if why is None:
            h.fork(parents, children)
            c.check()
        else:
            with pytest.raises(hq.HQError, match=why):
                c.check()
        if why == "page number":
            c.table[0, 1] = int(h.table[0, 1])
        same(c, h, f"{n}")
        assert not bool(ws[:4096].any())
