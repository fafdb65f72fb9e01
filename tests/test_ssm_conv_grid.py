"""CPU test of the convolution's grid: a call whose workgroups one launch does not hold is refused by its sizes, before anything
touches a device."""
import pytest

from nebula_amd import hq
from test_ssm_abi import P, cache, conv


@pytest.mark.parametrize("tokens", [32765, 32766, 32767])
def test_short_sequences_of_the_most_channels(tokens):
    """One token a wavefront: 8192 times 2048 workgroups of 256, a thread more than 32 bits count."""
    C = 1 << 20
    c = cache(channels=C, conv_row=3 * C, conv_layer=16 * 3 * C)
    assert conv(c, X=P, ldx=C, Y=P + 4096, ldy=C, tokens=tokens, cu=P, n=1024) == hq.HQ_ERR_SHAPE
    assert b"workgroups" in hq.lib().hq_last_error()
