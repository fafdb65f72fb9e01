"""KVCache.check waits for the device, whichever stream a call was enqueued on."""
import pytest
import torch

from nebula_amd import hq
from test_gpu_cache import fresh, i32

pytestmark = pytest.mark.gpu


def test_a_fault_on_another_stream_is_met(cuda):
    c, _ = fresh(pages=2)
    rows, counts = i32([0]), i32([100])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # the call is enqueued long before it runs
    c.reserve(rows, counts, stream=side)
    with pytest.raises(hq.HQError, match="free pages"):
        c.check()
    c.check()


def test_the_next_fault_on_another_stream_is_kept(cuda):
    """The word is clear when check() raises, and not some time after."""
    c, _ = fresh(pages=2)
    rows, counts, status = i32([0]), i32([100]), c.status
    side = torch.cuda.Stream()

    class Slow:
        def item(self):
            return status.item()

        def zero_(self):
            torch.cuda._sleep(200_000_000)
            status.zero_()

    c.reserve(rows, counts)
    c.status = Slow()
    with pytest.raises(hq.HQError, match="free pages"):
        c.check()
    c.reserve(rows, counts, stream=side)
    torch.cuda.synchronize()
    c.status = status
    with pytest.raises(hq.HQError, match="free pages"):
        c.check()
