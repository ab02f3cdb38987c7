"""The C entries of the gated projection refuse what their kernels do not take, with the documented status codes,
before they touch a device: no pointer here is ever read."""
import ctypes

import pytest

from test_operators_capi import P, _weight, hb  # noqa: F401  (the fixture)


def _gated(hb, gate=None, up=None, **kw):  # noqa: F811
    gate, up = (_weight(hb) if w is None else w for w in (gate, up))
    a = dict(type=0, x=P, xs=gate.k, rows=70, gb=None, ub=None, f32=0, act=2, z=None, y=P, ys=gate.n, ws=P, nws=1 << 40,
             counters=P, stream=None)
    a.update(kw)
    return hb.lib().xtq_gated_dev(ctypes.byref(gate), ctypes.byref(up), *a.values())


def _bwd(hb, gate=None, up=None, **kw):  # noqa: F811
    gate, up = (_weight(hb) if w is None else w for w in (gate, up))
    a = dict(type=0, dy=P, dys=gate.n, z=P, act=2, rows=70, dx=P, dxs=gate.k, dgb=None, dub=None, f32=0, ws=P,
             nws=1 << 40, stream=None)
    a.update(kw)
    return hb.lib().xtq_gated_bwd_dev(ctypes.byref(gate), ctypes.byref(up), *a.values())


@pytest.mark.parametrize("entry", (_gated, _bwd))
@pytest.mark.parametrize("kw,rc", [
    (dict(k=0), 6), (dict(k=130), 6), (dict(n=64), 6), (dict(K=1), 9), (dict(K=8), 9), (dict(code=b"qtip_1mad"), 8),
    (dict(code=b"mcg"), 8), (dict(code=None), 12), (dict(trellis=None), 12), (dict(suh=P + 1), 12), (dict(k=384), 6),
    (dict(n=256), 6)])
def test_weights(hb, entry, kw, rc):  # noqa: F811
    """Of either weight, and of one beside the other."""
    assert entry(hb, up=_weight(hb, **kw)) == rc
    assert entry(hb, gate=_weight(hb, **kw)) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(type=2), 15), (dict(type=16 | 2), 15), (dict(act=4), 15), (dict(act=-1), 15), (dict(rows=-1), 6),
    (dict(rows=1048561), 6), (dict(x=None), 12), (dict(x=P + 1), 12), (dict(xs=255), 6), (dict(y=None), 12),
    (dict(ys=383), 6), (dict(z=P + 2), 12), (dict(gb=P + 1), 12), (dict(gb=P + 2, f32=1), 12), (dict(ub=P + 2, f32=2), 12),
    (dict(counters=None), 12), (dict(counters=P + 2), 12), (dict(ws=None), 12), (dict(ws=P + 8), 12),
    (dict(nws=100), 14), (dict(nws=100, rows=3), 14), (dict(nws=100, rows=70, type=17), 14)])
def test_gated(hb, kw, rc):  # noqa: F811
    assert _gated(hb, **kw) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(type=2), 15), (dict(act=4), 15), (dict(rows=0), 6), (dict(rows=1048561), 6), (dict(dy=None), 12),
    (dict(dys=383), 6), (dict(z=None), 12), (dict(z=P + 2), 12), (dict(dx=None), 12), (dict(dxs=255), 6),
    (dict(dgb=P + 1), 12), (dict(dub=P + 2, f32=2), 12), (dict(ws=None), 12), (dict(ws=P + 8), 12), (dict(nws=100), 14)])
def test_gradient(hb, kw, rc):  # noqa: F811
    assert _bwd(hb, **kw) == rc


def test_no_rows_and_scratch(hb):  # noqa: F811
    assert _gated(hb, rows=0, x=None, y=None, ws=None, nws=0, counters=None) == 0
    L = hb.lib()
    p = ctypes.byref(_weight(hb))
    for gradient in (0, 1):
        assert L.xtq_gated_ws_bytes(p, 0, gradient) == 0 and L.xtq_gated_ws_bytes(p, -1, gradient) == -6
        assert L.xtq_gated_ws_bytes(p, 1048561, gradient) == -6
        assert L.xtq_gated_ws_bytes(ctypes.byref(_weight(hb, k=1)), 5, gradient) == -6
        for rows in (1, 16, 17, 64, 65, 1000, 1048560):
            assert L.xtq_gated_ws_bytes(p, rows, gradient) > 0
    # sizes past 32 bits
    big = ctypes.byref(_weight(hb, k=65536, n=65536))
    assert L.xtq_gated_ws_bytes(big, 1048560, 0) > 4 * 65536 * (1048560 + 65536)
    assert L.xtq_gated_ws_bytes(big, 1048560, 1) > 4 * 65536 * (1048560 + 65536)
