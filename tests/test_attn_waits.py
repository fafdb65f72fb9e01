"""CPU test of the attention kernels' wait counts: as tests/test_waits.py, at every meeting of wavefronts in
the compiled code a wavefront's own copies into LDS have landed on every path."""
import pytest

import isa

pytestmark = pytest.mark.skipif(not (isa.OBJDUMP.exists() and isa.LIB.exists()), reason="needs llvm-objdump and the built library")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    return isa.kernels(tmp_path_factory.mktemp("isa"))


@pytest.mark.parametrize("family", ["hq_attn_tile_kernel", "hq_attn_row_kernel", "hq_attn_prefix_kernel"])
def test_copies_into_lds_land_before_they_are_published(kernels, family):
    found = {n: c for n, c in kernels.items() if family in n}
    assert found and all(any(op.startswith("buffer_load") and " lds" in args for _, op, args, _ in c) for c in found.values())
    late = {n: [hex(a) for a in isa.unlanded_copies(c)] for n, c in found.items()}
    assert not {n: a for n, a in late.items() if a}


@pytest.mark.parametrize("family", ["hq_attn_", "hq_cache_"])
def test_no_kernel_keeps_its_registers_in_memory(kernels, family):
    found = {n: c for n, c in kernels.items() if family in n}
    assert found
    spilled = [n for n, c in found.items() if any(op.startswith("scratch_") for _, op, _, _ in c)]
    assert not spilled
