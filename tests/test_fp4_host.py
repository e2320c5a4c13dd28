"""CPU tests of the 4-bit KV pool: its oracle, row layout and the refusals of the C entries.

Refused calls return before anything is launched, so they need no GPU; the pointers they are
given are never followed.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from minisgl_b200 import _native as nat
from oracle import fp4 as F

PTR = 1 << 20  # a 16-byte aligned address that nothing reads


def test_oracle_known_values():
    x = np.zeros((1, 16))
    x[0, :9] = [6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.01]  # scale 1: every border between two codes
    v = F.roundtrip(x)
    np.testing.assert_array_equal(v[0, :9], [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -6.0])
    assert (F.roundtrip(np.full((2, 16), 0.0)) == 0).all()
    big = F.roundtrip(np.array([[np.inf, -1e9, np.nan] + [1.0] * 13]))
    np.testing.assert_array_equal(big[0, :3], [2688.0, -2688.0, 0.0])
    assert (F.roundtrip(np.full((1, 16), 0.005)) == 0).all()  # below 6 * 2^-10 a block vanishes


def test_oracle_error_of_normal_blocks():
    """A code is off by at most half a step of its octave (25%), or by the scale's rounding (2^-4) at the top."""
    x = np.random.default_rng(0).standard_normal((400, 16))
    v = F.roundtrip(x)
    amax = np.abs(x).max(-1, keepdims=True)
    assert (np.abs(v - x) <= amax / 6 * (1 + 2.0 ** -4) + 1e-12).all()
    np.testing.assert_array_equal(F.roundtrip(v), v)  # stored values are kept


@pytest.mark.parametrize("Hkv", [1, 2, 3, 4, 8, 16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_row_bytes(Hkv, D):
    n = nat.LIB.b2a_fp4_row_bytes(Hkv, D)
    assert n == F.row_bytes(Hkv, D) and n % 16 == 0 and n % 128 != 0 and n >= Hkv * D * 9 // 8


@pytest.mark.parametrize("Hkv,D", [(0, 128), (-1, 128), (8, 96), (8, 0), (8, 512), (1 << 20, 128)])
def test_row_bytes_of_unsupported_shapes(Hkv, D):
    assert nat.LIB.b2a_fp4_row_bytes(Hkv, D) == 0


def _store(**kw):
    a = dict(k=PTR, ks=1024, v=PTR, vs=1024, loc=PTR, pool=PTR, slots=64, T=4, Hkv=8, D=128, gk=1.0, gv=1.0, dt=1)
    a.update(kw)
    nat.call("b2a_fp4_store_kv", a["k"], a["ks"], a["v"], a["vs"], a["loc"], a["pool"], a["slots"], a["T"], a["Hkv"],
             a["D"], a["gk"], a["gv"], a["dt"], None)


@pytest.mark.parametrize("kw", [dict(T=-1), dict(Hkv=0), dict(D=96), dict(gk=0.0), dict(gk=3.0), dict(gv=-2.0),
                                dict(gv=float("inf")), dict(gk=float("nan")), dict(dt=7), dict(k=None), dict(v=None),
                                dict(loc=None), dict(pool=None), dict(slots=0), dict(ks=1023), dict(vs=1023),
                                dict(pool=PTR + 8), dict(k=PTR + 1), dict(v=PTR + 1), dict(T=1 << 40)])
def test_store_refusals(kw):
    with pytest.raises((ValueError, nat.B200AttnError)):
        _store(**kw)


def test_store_of_nothing_is_fine():
    _store(T=0, k=None, v=None, loc=None)


def _load(**kw):
    a = dict(pool=PTR, slots=64, loc=PTR, n=4, Hkv=8, D=128, gk=1.0, gv=1.0, k=PTR, v=PTR, dt=1)
    a.update(kw)
    nat.call("b2a_fp4_load_kv", a["pool"], a["slots"], a["loc"], a["n"], a["Hkv"], a["D"], a["gk"], a["gv"], a["k"],
             a["v"], a["dt"], None)


@pytest.mark.parametrize("kw", [dict(n=-1), dict(Hkv=0), dict(D=32), dict(gk=0.75), dict(dt=5), dict(pool=None),
                                dict(loc=None), dict(k=None), dict(v=None), dict(slots=-3), dict(k=PTR + 2)])
def test_load_refusals(kw):
    with pytest.raises((ValueError, nat.B200AttnError)):
        _load(**kw)


def _decode(**kw):
    a = dict(q=PTR, pool=PTR, slots=64, idx=PTR, P=16, cta=PTR, segs=PTR, nc=148, merge=PTR, npart=0, B=4, Hq=16,
             Hkv=8, D=128, scale=0.1, gk=1.0, gv=1.0, ws=PTR, wsb=0, out=PTR, dt=1)
    a.update(kw)
    nat.call("b2a_fp4_decode", a["q"], a["pool"], a["slots"], a["idx"], a["P"], a["cta"], a["segs"], a["nc"],
             a["merge"], a["npart"], a["B"], a["Hq"], a["Hkv"], a["D"], a["scale"], a["gk"], a["gv"], a["ws"],
             a["wsb"], a["out"], a["dt"], None)


@pytest.mark.parametrize("kw", [dict(B=-1), dict(Hq=15), dict(Hkv=0), dict(Hkv=3, Hq=6), dict(Hkv=32, Hq=32),
                                dict(Hq=128), dict(D=96), dict(dt=2), dict(dt=9), dict(scale=0.0), dict(scale=-1.0),
                                dict(scale=float("nan")), dict(scale=float("inf")), dict(gk=1.5), dict(cta=None),
                                dict(segs=None), dict(segs=PTR + 4), dict(nc=0), dict(q=None), dict(pool=None),
                                dict(idx=None), dict(out=None), dict(slots=0), dict(q=PTR + 8), dict(P=12),
                                dict(P=8192), dict(npart=-1), dict(npart=5), dict(npart=5, wsb=1 << 30, ws=PTR + 16),
                                dict(npart=5, wsb=1 << 30, merge=None)])
def test_decode_refusals(kw):
    with pytest.raises((ValueError, nat.B200AttnError)):
        _decode(**kw)


def test_tile_sizes_and_refusals():
    for Hq, Hkv, D, dt in ((16, 8, 128, 1), (8, 8, 64, 0), (64, 8, 256, 1)):
        assert 1 <= nat.fp4_extend_tile_q(Hq, Hkv, D, dt) <= 256
    for Hq, Hkv, D, dt in ((24, 8, 128, 1), (16, 8, 96, 1), (16, 8, 128, 2), (15, 8, 128, 1), (256, 8, 128, 1)):
        with pytest.raises((ValueError, nat.B200AttnError)):
            nat.fp4_extend_tile_q(Hq, Hkv, D, dt)


def _extend(**kw):
    a = dict(q=PTR, pool=PTR, slots=64, qo=PTR, kv=PTR, idx=PTR, lpl=PTR, P=16, work=PTR, nw=4, rk=128, ns=1, T=9, B=2, Hq=16,
             Hkv=8, D=128, scale=0.1, gk=1.0, gv=1.0, ws=PTR, wsb=0, out=PTR, dt=1)
    a.update(kw)
    nat.call("b2a_fp4_extend", a["q"], a["pool"], a["slots"], a["qo"], a["kv"], a["idx"], a["lpl"], a["P"], a["work"],
             a["nw"], a["rk"], a["ns"], a["T"], a["B"], a["Hq"], a["Hkv"], a["D"], a["scale"], a["gk"], a["gv"], a["ws"],
             a["wsb"], a["out"], a["dt"], None)


@pytest.mark.parametrize("kw", [dict(nw=-1), dict(T=-1), dict(B=-1), dict(Hq=24), dict(Hq=15), dict(D=96), dict(dt=2),
                                dict(scale=0.0), dict(scale=float("nan")), dict(gk=0.3), dict(P=24), dict(ns=0),
                                dict(ns=65), dict(ns=2, rk=0), dict(ns=2, rk=64), dict(ns=2, rk=200), dict(q=None), dict(pool=None),
                                dict(qo=None), dict(kv=None), dict(idx=None), dict(work=None), dict(out=None),
                                dict(work=PTR + 8), dict(q=PTR + 8), dict(slots=0), dict(ns=2),
                                dict(ns=2, ws=None, wsb=1 << 40), dict(ns=2, ws=PTR + 16, wsb=1 << 40)])
def test_extend_refusals(kw):
    with pytest.raises((ValueError, nat.B200AttnError)):
        _extend(**kw)


def test_extend_workspace():
    f = nat.LIB.b2a_fp4_extend_workspace_bytes
    assert f(8, 1, 8, 128) == 0 and f(0, 4, 8, 128) == 0
    assert f(8, 4, 8, 128) == 256 + 8 * 8 * 4 * 256 * 130 * 4


def _tables(**kw):
    a = dict(table=PTR, rows_=8, stride=64, rows=PTR, cached=PTR, lens=PTR, B=4, P=16, tile=64, qo=PTR, pos=PTR,
             loc=PTR, qcap=16, last=PTR, kv=PTR, idx=PTR, icap=16, lpl=PTR, work=PTR, wcap=8, counts=PTR)
    a.update(kw)
    nat.call("b2a_extend_metadata", a["table"], a["rows_"], a["stride"], a["rows"], a["cached"], a["lens"], a["B"],
             a["P"], a["tile"], a["qo"], a["pos"], a["loc"], a["qcap"], a["last"], a["kv"], a["idx"], a["icap"],
             a["lpl"], a["work"], a["wcap"], a["counts"], None)


@pytest.mark.parametrize("kw", [dict(B=-1), dict(B=8193), dict(P=3), dict(P=0), dict(tile=0), dict(tile=257),
                                dict(rows_=0), dict(stride=0), dict(stride=1 << 32), dict(qcap=-1), dict(icap=-1),
                                dict(wcap=-1), dict(wcap=(1 << 24) + 1), dict(table=None), dict(rows=None),
                                dict(cached=None), dict(lens=None), dict(qo=None), dict(pos=None), dict(loc=None),
                                dict(last=None), dict(kv=None), dict(idx=None), dict(lpl=None), dict(work=None),
                                dict(counts=None), dict(work=PTR + 4)])
def test_tables_refusals(kw):
    with pytest.raises((ValueError, nat.B200AttnError)):
        _tables(**kw)


def test_pool_needs_a_power_of_two_scale_and_a_known_shape():
    torch = pytest.importorskip("torch")
    from minisgl_b200 import FP4KVCache

    for kw in (dict(k_scale=3.0), dict(v_scale=0.0), dict(k_scale=-1.0), dict(v_scale=float("inf"))):
        with pytest.raises(ValueError):
            FP4KVCache(1, 16, 8, 128, torch.bfloat16, **kw)
    for shape in ((1, 16, 8, 96), (1, 16, 0, 128), (0, 16, 8, 128), (1, 0, 8, 128)):
        with pytest.raises(ValueError):
            FP4KVCache(*shape, torch.bfloat16)
    with pytest.raises(ValueError):
        FP4KVCache(1, 16, 8, 128, torch.int32)


def test_engine_config_names_the_pool():
    from minisgl_b200.engine import EngineConfig

    assert EngineConfig(spec=None).kv_cache_dtype == "auto"
