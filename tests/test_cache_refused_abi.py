"""CPU test: reserve and append ask for the cache's `refused`, the other calls do not; a misaligned one is refused by all."""
import ctypes

from nebula_amd import attn, hq
from test_attn_abi import P, cache, io


def test_refused_is_asked_for():
    L = attn._lib()
    assert L.hq_cache_reserve(cache(), P, P, 1, None) == hq.HQ_ERR_INVALID_ARG and b"refused" in L.hq_last_error()
    assert L.hq_cache_append(cache(), 0, P, 1024, 128, P, 1024, 128, 1, P, None, 1, None) == hq.HQ_ERR_INVALID_ARG
    b = ctypes.c_size_t(0)
    assert L.hq_cache_workspace_bytes(cache(), ctypes.byref(b)) == hq.HQ_OK and b.value > 0
    odd = cache(refused=P + 2)
    for got in (L.hq_cache_reserve(odd, P, P, 1, None), L.hq_cache_fork(odd, P, P, 1, None, 0, None), L.hq_cache_free(odd, P, 1, None),
                L.hq_attn_paged(io(), odd, 0, None, None, 4, 0, None, 0, None), L.hq_cache_workspace_bytes(odd, ctypes.byref(b))):
        assert got == hq.HQ_ERR_ALIGNMENT
