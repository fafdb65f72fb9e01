"""CPU tests of the rotary entry points (include/hq_rotary.h): exports, struct layouts, frequencies, and that bad arguments
are refused before anything touches a device."""
import ctypes
import math
import re
from pathlib import Path

import numpy as np
import pytest

from nebula_amd import attn, hq, rotary

ROOT = Path(__file__).resolve().parent.parent
HEADER = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "hq_rotary.h").read_text(), flags=re.S)
P = 1 << 20  # an address that is aligned and never followed


def test_library_exports_every_declared_symbol():
    declared = sorted(set(re.findall(r"\b(hq_[a-z0-9_]+)\s*\(", HEADER)))
    assert declared == sorted(rotary.EXPORTS)
    for name in declared:
        assert hasattr(hq.lib(), name), name


def test_structs_mirror_the_header():
    for cname, cls in (("hq_rotary", rotary.RotaryDesc), ("hq_rotary_heads", rotary.RotaryHeads)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), HEADER, flags=re.S)[1]
        names = [n.strip().lstrip("*").split()[-1].lstrip("*") for line in body.split(";") if line.strip() for n in line.split(",")]
        assert names == [f[0] for f in cls._fields_]
    assert rotary._HEADS.size == ctypes.sizeof(rotary.RotaryHeads)
    for name, value in rotary.LAYOUTS.items():
        assert f"HQ_ROTARY_{name.upper()} = {value}" in HEADER


def rot(**kw):
    return ctypes.byref(rotary.RotaryDesc(**{**dict(turns=P, dim=64, layout=1, scale=1.0), **kw}))


def heads(**kw):
    return bytes(rotary.RotaryHeads(**{**dict(In=P, Out=P + 4096, in_row=1024, in_head=128, out_row=1024, out_head=128, weight=0, heads=8, eps=1e-6), **kw}))


def cache(**kw):
    d = dict(K=P, V=P, layer_stride=64 * 65536, page_stride=65536, head_stride=8192, token_stride=128, layers=2, pages=64, kv_heads=8,
             page_tokens=64, head_dim=128, dtype=1, table=P, table_stride=32, rows=16, max_pages=32, lens=P, refs=P, status=P, refused=P)
    return ctypes.byref(attn.KVCacheDesc(**{**d, **kw}))


def rotate(r=None, q=None, k=None, tokens=4, D=128, dtype=1, pos=P):
    return rotary._lib().hq_rotate(r or rot(), q or heads(), k, tokens, D, dtype, pos or None, None)


def append(c=None, layer=0, r=None, q=None, k=None, V=P, v_row=1024, v_head=128, tokens=4, rows=P, cu=0, n=4):
    return rotary._lib().hq_cache_append_rotated(c or cache(), layer, r or rot(), q, k or heads(), V or None, v_row, v_head, tokens, rows or None,
                                                 cu or None, n, None)


BAD_ROTARY = [(dict(turns=0), hq.HQ_ERR_INVALID_ARG), (dict(turns=P + 4), hq.HQ_ERR_ALIGNMENT), (dict(layout=0), hq.HQ_ERR_INVALID_ARG),
              (dict(layout=3), hq.HQ_ERR_INVALID_ARG), (dict(dim=0), hq.HQ_ERR_SHAPE), (dict(dim=24), hq.HQ_ERR_SHAPE),
              (dict(dim=144), hq.HQ_ERR_SHAPE), (dict(scale=0.0), hq.HQ_ERR_INVALID_ARG), (dict(scale=float("inf")), hq.HQ_ERR_INVALID_ARG),
              (dict(scale=float("nan")), hq.HQ_ERR_INVALID_ARG)]
BAD_HEADS = [(dict(In=0), hq.HQ_ERR_INVALID_ARG), (dict(In=P + 8), hq.HQ_ERR_ALIGNMENT), (dict(heads=0), hq.HQ_ERR_SHAPE),
             (dict(heads=1025), hq.HQ_ERR_SHAPE), (dict(in_row=1020), hq.HQ_ERR_ALIGNMENT), (dict(in_head=64), hq.HQ_ERR_SHAPE),
             (dict(in_row=-8), hq.HQ_ERR_SHAPE), (dict(in_row=1 << 50), hq.HQ_ERR_SHAPE), (dict(weight=P + 4), hq.HQ_ERR_ALIGNMENT),
             (dict(weight=P, eps=-1.0), hq.HQ_ERR_INVALID_ARG), (dict(weight=P, eps=float("nan")), hq.HQ_ERR_INVALID_ARG)]
BAD_OUT = [(dict(Out=0), hq.HQ_ERR_INVALID_ARG), (dict(Out=P + 2), hq.HQ_ERR_ALIGNMENT), (dict(out_row=512), hq.HQ_ERR_SHAPE),
           (dict(out_head=132), hq.HQ_ERR_ALIGNMENT), (dict(Out=P, out_row=2048), hq.HQ_ERR_SHAPE), (dict(Out=P, out_head=256, out_row=4096), hq.HQ_ERR_SHAPE)]


@pytest.mark.parametrize("kw,status", BAD_ROTARY)
def test_bad_rotary(kw, status):
    assert rotate(r=rot(**kw)) == status and append(r=rot(**kw)) == status
    assert hq.lib().hq_last_error()


@pytest.mark.parametrize("kw,status", BAD_HEADS + BAD_OUT)
def test_bad_heads(kw, status):
    assert rotate(q=heads(**kw)) == status and rotate(k=heads(**kw)) == status and append(q=heads(**kw)) == status


@pytest.mark.parametrize("kw,status", BAD_HEADS)
def test_bad_keys_of_an_append(kw, status):
    assert append(k=heads(**{**kw, "Out": 0, "out_row": 0, "out_head": 0})) == status


@pytest.mark.parametrize("kw,status", [(dict(tokens=0), hq.HQ_ERR_SHAPE), (dict(tokens=(1 << 24) + 1), hq.HQ_ERR_SHAPE), (dict(D=96), hq.HQ_ERR_UNSUPPORTED),
                                       (dict(dtype=0), hq.HQ_ERR_INVALID_ARG), (dict(pos=0), hq.HQ_ERR_INVALID_ARG), (dict(pos=P + 2), hq.HQ_ERR_ALIGNMENT)])
def test_bad_rotate(kw, status):
    assert rotate(**kw) == status
    assert rotary._lib().hq_rotate(rot(), None, None, 4, 128, 1, P, None) == hq.HQ_ERR_INVALID_ARG
    assert rotary._lib().hq_rotate(None, heads(), None, 4, 128, 1, P, None) == hq.HQ_ERR_INVALID_ARG


@pytest.mark.parametrize("kw,status", [
    (dict(layer=2), hq.HQ_ERR_SHAPE), (dict(V=0), hq.HQ_ERR_INVALID_ARG), (dict(V=P + 8), hq.HQ_ERR_ALIGNMENT), (dict(v_row=4), hq.HQ_ERR_ALIGNMENT),
    (dict(v_head=0), hq.HQ_ERR_SHAPE), (dict(tokens=5), hq.HQ_ERR_SHAPE), (dict(rows=0), hq.HQ_ERR_INVALID_ARG), (dict(rows=P + 1), hq.HQ_ERR_ALIGNMENT),
    (dict(cu=P + 2), hq.HQ_ERR_ALIGNMENT), (dict(n=0), hq.HQ_ERR_SHAPE), (dict(n=1025, cu=P), hq.HQ_ERR_SHAPE), (dict(tokens=0, cu=P), hq.HQ_ERR_SHAPE),
    (dict(k=heads(heads=4)), hq.HQ_ERR_SHAPE), (dict(c=cache(refused=0)), hq.HQ_ERR_INVALID_ARG), (dict(c=cache(page_tokens=48)), hq.HQ_ERR_SHAPE),
    (dict(c=cache(dtype=7)), hq.HQ_ERR_INVALID_ARG)])
def test_bad_append(kw, status):
    assert append(**kw) == status


def test_frequencies():
    i = np.arange(32)
    f, s = rotary.frequencies(64, 1e4)
    assert s == 1.0 and np.allclose(f, 1e4 ** (-2 * i / 64), rtol=1e-14, atol=0)
    assert np.array_equal(rotary.frequencies(64, 1e4, rotary.Linear(4.0))[0], f / 4)
    # The slowest pair turns 1 / factor as far, the fastest one as far.
    g, s = rotary.frequencies(64, 1e4, rotary.Base(8.0))
    assert s == 1.0 and g[0] == 1.0 and math.isclose(g[-1], f[-1] / 8, rel_tol=1e-12)
    # By parts: pairs with 32 turns and more in 4096 positions as they are, those with one or less at a fourth.
    g, s = rotary.frequencies(64, 1e4, rotary.Stretch(4.0, 4096))
    turns = 4096 * f / (2 * math.pi)
    assert math.isclose(s, 0.1 * math.log(4.0) + 1)
    assert np.array_equal(g[turns > 40], f[turns > 40]) and np.allclose(g[turns < 0.8], f[turns < 0.8] / 4, rtol=1e-14, atol=0)
    middle = (turns < 30) & (turns > 1.2)
    assert middle.sum() > 5 and (g[middle] < f[middle]).all() and (g[middle] > f[middle] / 4).all() and (np.diff(g) < 0).all()
    assert rotary.frequencies(64, 1e4, rotary.Stretch(4.0, 4096, scale=1.0))[1] == 1.0 and rotary.frequencies(64, 1e4, rotary.Stretch(0.5, 4096))[1] == 1.0
    for bad in (dict(dim=0), dict(dim=20), dict(dim=64, base=0.0), dict(dim=64, base=float("inf")), dict(dim=64, scaling=rotary.Linear(0.0)),
                dict(dim=64, scaling=rotary.Stretch(4.0, 0)), dict(dim=64, scaling=rotary.Stretch(4.0, 4096, fast=1.0)),
                dict(dim=64, base=0.5, scaling=rotary.Stretch(4.0, 4096))):
        with pytest.raises(ValueError):
            rotary.frequencies(**bad)
    with pytest.raises((TypeError, AttributeError)):
        rotary.frequencies(64, scaling="linear")


def test_rotary_keeps_turns():
    r = rotary.Rotary(64, base=1e6, device="cpu")
    assert np.allclose(r.turns.numpy() * 2 * np.pi, 1e6 ** (-2 * np.arange(32) / 64), rtol=1e-14, atol=0) and r.scale == 1.0
    r = rotary.Rotary(32, angles=np.linspace(1, 0, 16), scale=2.0, layout="interleaved", device="cpu")
    assert np.allclose(r.turns.numpy(), np.linspace(1, 0, 16) / (2 * np.pi)) and r.scale == 2.0
    for bad in (dict(layout="pairs"), dict(angles=[1.0] * 15), dict(angles=[float("nan")] * 16)):
        with pytest.raises(ValueError):
            rotary.Rotary(32, device="cpu", **bad)
