"""CPU test: an output of a rotation that is another operand, whose heads would be written while others read them, is refused."""
import pytest

from nebula_amd import hq
from test_rotary_abi import P, append, heads, rotate

A, B, C, D = (P + 4096 * i for i in range(4))


@pytest.mark.parametrize("q,k", [((A, C), (B, C)), ((A, B), (B, D)), ((A, C), (B, A)), ((A, B), (B, A)), ((A, B), (B, B)), ((A, A), (B, A)), ((A, A), (A, A))])
def test_rotate(q, k):
    assert rotate(q=heads(In=q[0], Out=q[1]), k=heads(In=k[0], Out=k[1])) == hq.HQ_ERR_INVALID_ARG
    assert b"Out" in hq.lib().hq_last_error()


@pytest.mark.parametrize("out", [B, C])
def test_append(out):
    assert append(q=heads(In=A, Out=out), k=heads(In=B), V=C) == hq.HQ_ERR_INVALID_ARG
    assert b"Out" in hq.lib().hq_last_error()
