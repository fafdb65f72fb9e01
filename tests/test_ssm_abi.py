"""CPU tests of the state space entry points (include/hq_ssm.h): exports, struct layouts, and that bad arguments are
refused before anything touches a device."""
import ctypes
import re
from pathlib import Path

import pytest

from nebula_amd import hq, ssm

ROOT = Path(__file__).resolve().parent.parent
HEADER = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "hq_ssm.h").read_text(), flags=re.S)
P = 1 << 20  # an address that is aligned and never followed


def test_library_exports_every_declared_symbol():
    declared = sorted(set(re.findall(r"\b(hq_[a-z0-9_]+)\s*\(", HEADER)))
    assert declared == sorted(ssm.EXPORTS)
    for name in declared:
        assert hasattr(hq.lib(), name), name


def test_structs_mirror_the_header():
    for cname, cls in (("hq_state_cache", ssm.StateCacheDesc), ("hq_ssm_io", ssm.ScanIO)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), HEADER, flags=re.S)[1]
        names = [n.strip().lstrip("*").split()[-1].lstrip("*") for line in body.split(";") if line.strip() for n in line.split(",")]
        assert names == [f[0] for f in cls._fields_]
    assert ssm._IO.size == ctypes.sizeof(ssm.ScanIO)
    assert f"#define HQ_SSM_MAX_BATCH {ssm.MAX_BATCH}u" in HEADER


def cache(**kw):
    d = dict(conv=P, ssm=P, conv_layer=16 * 3 * 512, conv_row=3 * 512, ssm_layer=16 * 65536, ssm_row=65536, layers=2, rows=16, channels=512, width=4,
             heads=4, head_dim=128, state_dim=128, dtype=1, status=P, refused=0)
    return ctypes.byref(ssm.StateCacheDesc(**{**d, **kw}))


def conv(c=None, layer=0, X=P, ldx=1024, Y=P + 4096, ldy=1024, W=P, bias=0, tokens=4, rows=P, held=0, cu=0, n=4):
    return ssm._lib().hq_ssm_conv(c or cache(), layer, X or None, ldx, Y or None, ldy, W or None, bias or None, 1, tokens, rows or None, held or None,
                                  cu or None, n, None)


def io(**kw):
    d = dict(X=P, B=P, C=P, dt=P, Z=0, Y=P + 4096, A=P, D=0, dt_bias=0, x_row=1024, x_head=128, b_row=1024, b_group=128, c_row=1024, c_group=128, dt_row=4,
             z_row=512, z_head=128, y_row=512, y_head=128, tokens=4, groups=2, dt_f32=0, softplus=1)
    return bytes(ssm.ScanIO(**{**d, **kw}))


def scan(c=None, layer=0, i=None, rows=P, held=0, cu=0, n=4, max_len=0, ws=0, wsb=0):
    return ssm._lib().hq_ssm_scan(c or cache(), layer, i or io(), rows or None, held or None, cu or None, n, max_len, ws or None, wsb, None)


BAD_CACHE = [(dict(dtype=0), hq.HQ_ERR_INVALID_ARG), (dict(status=0), hq.HQ_ERR_INVALID_ARG), (dict(status=P + 2), hq.HQ_ERR_ALIGNMENT),
             (dict(refused=P + 1), hq.HQ_ERR_ALIGNMENT), (dict(layers=0), hq.HQ_ERR_SHAPE), (dict(rows=0), hq.HQ_ERR_SHAPE), (dict(rows=1 << 21), hq.HQ_ERR_SHAPE)]
BAD_LISTS = [(dict(layer=2), hq.HQ_ERR_SHAPE), (dict(rows=P + 2), hq.HQ_ERR_ALIGNMENT), (dict(held=P + 1), hq.HQ_ERR_ALIGNMENT),
             (dict(cu=P + 2), hq.HQ_ERR_ALIGNMENT), (dict(n=0), hq.HQ_ERR_SHAPE), (dict(n=5), hq.HQ_ERR_SHAPE), (dict(n=1025, cu=P), hq.HQ_ERR_SHAPE),
             (dict(n=17, cu=P, rows=0), hq.HQ_ERR_SHAPE)]


@pytest.mark.parametrize("kw,status", BAD_CACHE)
def test_bad_cache(kw, status):
    assert conv(cache(**kw)) == status and scan(cache(**kw)) == status and hq.lib().hq_last_error()


@pytest.mark.parametrize("kw,status", BAD_LISTS)
def test_bad_lists(kw, status):
    assert conv(**kw) == status and scan(**kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(c=cache(conv=0)), hq.HQ_ERR_INVALID_ARG), (dict(c=cache(conv=P + 8)), hq.HQ_ERR_ALIGNMENT), (dict(c=cache(width=1)), hq.HQ_ERR_UNSUPPORTED),
    (dict(c=cache(width=5)), hq.HQ_ERR_UNSUPPORTED), (dict(c=cache(channels=0)), hq.HQ_ERR_SHAPE), (dict(c=cache(channels=508)), hq.HQ_ERR_SHAPE),
    (dict(c=cache(conv_row=1024)), hq.HQ_ERR_SHAPE), (dict(c=cache(conv_row=1540)), hq.HQ_ERR_ALIGNMENT), (dict(c=cache(conv_layer=8)), hq.HQ_ERR_SHAPE),
    (dict(c=cache(conv_layer=4096)), hq.HQ_ERR_SHAPE), (dict(c=cache(conv_row=1 << 50)), hq.HQ_ERR_SHAPE), (dict(X=0), hq.HQ_ERR_INVALID_ARG),
    (dict(Y=0), hq.HQ_ERR_INVALID_ARG), (dict(W=0), hq.HQ_ERR_INVALID_ARG), (dict(Y=P), hq.HQ_ERR_INVALID_ARG), (dict(X=P + 8), hq.HQ_ERR_ALIGNMENT),
    (dict(W=P + 4), hq.HQ_ERR_ALIGNMENT), (dict(bias=P + 4), hq.HQ_ERR_ALIGNMENT), (dict(ldx=504), hq.HQ_ERR_SHAPE), (dict(ldy=1028), hq.HQ_ERR_ALIGNMENT),
    (dict(ldx=-1024), hq.HQ_ERR_SHAPE), (dict(tokens=0, cu=P), hq.HQ_ERR_SHAPE), (dict(tokens=(1 << 24) + 1, cu=P), hq.HQ_ERR_SHAPE)])
def test_bad_conv(kw, status):
    assert conv(**kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(c=cache(ssm=0)), hq.HQ_ERR_INVALID_ARG), (dict(c=cache(ssm=P + 4)), hq.HQ_ERR_ALIGNMENT), (dict(c=cache(head_dim=96)), hq.HQ_ERR_UNSUPPORTED),
    (dict(c=cache(state_dim=16)), hq.HQ_ERR_UNSUPPORTED), (dict(c=cache(heads=0)), hq.HQ_ERR_SHAPE), (dict(c=cache(heads=1025)), hq.HQ_ERR_SHAPE),
    (dict(c=cache(ssm_row=65532)), hq.HQ_ERR_SHAPE), (dict(c=cache(ssm_row=65538)), hq.HQ_ERR_ALIGNMENT), (dict(c=cache(ssm_layer=65540)), hq.HQ_ERR_SHAPE),
    (dict(ws=P + 128, wsb=1 << 40, n=1, cu=P, i=io(tokens=1 << 16)), hq.HQ_ERR_ALIGNMENT), (dict(ws=P, wsb=8, n=1, cu=P, i=io(tokens=1 << 16)), hq.HQ_ERR_WORKSPACE)])
def test_bad_scan(kw, status):
    assert scan(**kw) == status
    assert ssm._lib().hq_ssm_scan(cache(), 0, None, P, None, None, 4, 0, None, 0, None) == hq.HQ_ERR_INVALID_ARG


@pytest.mark.parametrize("kw,status", [
    (dict(X=0), hq.HQ_ERR_INVALID_ARG), (dict(B=0), hq.HQ_ERR_INVALID_ARG), (dict(C=0), hq.HQ_ERR_INVALID_ARG), (dict(dt=0), hq.HQ_ERR_INVALID_ARG),
    (dict(Y=0), hq.HQ_ERR_INVALID_ARG), (dict(A=0), hq.HQ_ERR_INVALID_ARG), (dict(Y=P), hq.HQ_ERR_INVALID_ARG), (dict(X=P + 8), hq.HQ_ERR_ALIGNMENT),
    (dict(B=P + 2), hq.HQ_ERR_ALIGNMENT), (dict(C=P + 8), hq.HQ_ERR_ALIGNMENT), (dict(Z=P + 8), hq.HQ_ERR_ALIGNMENT), (dict(Y=P + 8), hq.HQ_ERR_ALIGNMENT),
    (dict(dt=P + 1), hq.HQ_ERR_ALIGNMENT), (dict(dt=P + 2, dt_f32=1), hq.HQ_ERR_ALIGNMENT), (dict(A=P + 2), hq.HQ_ERR_ALIGNMENT), (dict(D=P + 2), hq.HQ_ERR_ALIGNMENT),
    (dict(dt_bias=P + 1), hq.HQ_ERR_ALIGNMENT), (dict(groups=0), hq.HQ_ERR_SHAPE), (dict(groups=3), hq.HQ_ERR_SHAPE), (dict(x_row=1020), hq.HQ_ERR_ALIGNMENT),
    (dict(x_head=64), hq.HQ_ERR_SHAPE), (dict(b_group=64), hq.HQ_ERR_SHAPE), (dict(c_row=-8), hq.HQ_ERR_SHAPE), (dict(y_row=256), hq.HQ_ERR_SHAPE),
    (dict(Z=P, z_head=100), hq.HQ_ERR_ALIGNMENT), (dict(Z=P + 4096, z_row=1024), hq.HQ_ERR_SHAPE), (dict(dt_row=3), hq.HQ_ERR_SHAPE),
    (dict(dt_row=-4), hq.HQ_ERR_SHAPE), (dict(dt_row=1 << 50), hq.HQ_ERR_SHAPE), (dict(tokens=0), hq.HQ_ERR_SHAPE), (dict(tokens=5), hq.HQ_ERR_SHAPE),
    (dict(y_row=128, y_head=256), hq.HQ_ERR_SHAPE), (dict(x_row=(1 << 22) + 8), hq.HQ_ERR_SHAPE), (dict(b_row=1 << 23), hq.HQ_ERR_SHAPE), (dict(dt_row=(1 << 22) + 1), hq.HQ_ERR_SHAPE)])
def test_bad_io(kw, status):
    assert scan(i=io(**kw)) == status


def workspace(*a):
    b = ctypes.c_size_t(7)
    return ssm._lib().hq_ssm_workspace_bytes(*a, ctypes.byref(b)), b.value


def test_workspace_query():
    assert workspace(4, 4, 0, 48, 16, 128, 128, 0) == (hq.HQ_OK, 0)
    for bad, status in (((0, 1, 1, 48, 16, 128, 128, 0), hq.HQ_ERR_SHAPE), ((5, 4, 0, 48, 16, 128, 128, 0), hq.HQ_ERR_SHAPE),
                        ((5, 0, 1, 48, 16, 128, 128, 0), hq.HQ_ERR_SHAPE), ((5, 1, 1, 0, 16, 128, 128, 0), hq.HQ_ERR_SHAPE),
                        ((5, 1, 1, 48, 7, 128, 128, 0), hq.HQ_ERR_SHAPE), ((5, 1, 1, 48, 0, 128, 128, 0), hq.HQ_ERR_SHAPE),
                        ((5, 1, 1, 48, 16, 32, 128, 0), hq.HQ_ERR_UNSUPPORTED), ((5, 1, 1, 48, 16, 128, 512, 0), hq.HQ_ERR_UNSUPPORTED)):
        assert workspace(*bad)[0] == status
    assert ssm._lib().hq_ssm_workspace_bytes(4, 4, 0, 48, 16, 128, 128, 0, None) == hq.HQ_ERR_INVALID_ARG
    assert "hq_ssm" in ssm.describe(4, 4, 48, 16, 128, 128, single=True)
    for n in (1, 3, 16):
        for H in (1, 8, 48, 128):
            last = 0
            for T in [16, 64, 65, 100, 128, 200, 500, 640, 1000, 1600, 2000, 4096, 6000, 8192, 20000, 65536, 1 << 20]:
                size = ssm.workspace_bytes(T, n, H, 1, 128, 128)
                assert size >= last, (n, H, T)
                last = size
