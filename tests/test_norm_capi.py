"""The C entries of the norms refuse what their kernels do not take, with the documented status codes, before they
touch a device: no pointer here is ever read."""
import ctypes

import pytest

from test_operators_capi import P, hb  # noqa: F401  (the fixture)


def _params(hb, **kw):  # noqa: F811
    a = dict(kind=1, post=2, gate_act=1, f32=0, eps=1e-6, post_eps=1e-6, scale_number=1.0, weight=P, bias=None,
             scale=P, post_weight=P, post_bias=None)
    a.update(kw)
    return hb.NormParams(*a.values())


def _norm(hb, params=None, **kw):  # noqa: F811
    a = dict(type=0, rows=5, d=100, x=P, xs=100, res=P, rs=100, gate=P, gs=100, y=P, ys=100, h=P, hs=100, stats=P,
             stream=None)
    a.update(kw)
    return hb.lib().xtq_norm_dev(ctypes.byref(_params(hb) if params is None else params), *a.values())


def _bwd(hb, params=None, dparam=(P, None, P, P, None), **kw):  # noqa: F811
    a = dict(type=0, rows=5, d=100, x=P, xs=100, res=P, rs=100, gate=P, gs=100, stats=P, dy=P, dys=100, dh=P, dhs=100,
             dx=P, dres=P, dgate=P, dparam=dparam and (ctypes.c_void_p * 5)(*dparam), ws=P, nws=1 << 40, stream=None)
    a.update(kw)
    return hb.lib().xtq_norm_bwd_dev(ctypes.byref(_params(hb) if params is None else params), *a.values())


@pytest.mark.parametrize("entry", (_norm, _bwd))
@pytest.mark.parametrize("kw,rc", [
    (dict(kind=3), 15), (dict(kind=-1), 15), (dict(post=3), 15), (dict(gate_act=3), 15), (dict(gate_act=-1), 15),
    (dict(weight=P + 1), 12), (dict(weight=P + 2, f32=1), 12), (dict(bias=P + 2, f32=2), 12),
    (dict(scale=P + 2, f32=4), 12), (dict(post_weight=P + 2, f32=8), 12), (dict(post_bias=P + 2, f32=16), 12)])
def test_params(hb, entry, kw, rc):  # noqa: F811
    assert entry(hb, _params(hb, **kw)) == rc


@pytest.mark.parametrize("entry", (_norm, _bwd))
@pytest.mark.parametrize("kw,rc", [
    (dict(type=2), 15), (dict(type=16), 15), (dict(d=0), 6), (dict(d=32769), 6), (dict(rows=-1), 6),
    (dict(rows=(1 << 30) + 1), 6), (dict(x=None), 12), (dict(x=P + 1), 12), (dict(xs=99), 6), (dict(res=P + 1), 12),
    (dict(rs=99), 6), (dict(gate=P + 1), 12), (dict(gs=99), 6), (dict(stats=P + 8), 12), (dict(res=None), 15)])
def test_inputs(hb, entry, kw, rc):  # noqa: F811
    assert entry(hb, **kw) == rc


@pytest.mark.parametrize("kw,rc", [(dict(y=None), 12), (dict(ys=99), 6), (dict(h=None), 12), (dict(h=P + 1), 12),
                                   (dict(hs=99), 6)])
def test_results(hb, kw, rc):  # noqa: F811
    assert _norm(hb, **kw) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(rows=0), 6), (dict(stats=None), 12), (dict(dy=P + 1), 12), (dict(dys=99), 6), (dict(dh=P + 1), 12),
    (dict(dhs=99), 6), (dict(dx=P + 1), 12), (dict(dres=P + 1), 12), (dict(dgate=P + 1), 12), (dict(dparam=None), 12),
    (dict(ws=None), 12), (dict(ws=P + 8), 12), (dict(nws=100), 14), (dict(gate=None), 15)])
def test_gradient(hb, kw, rc):  # noqa: F811
    assert _bwd(hb, **kw) == rc


def test_gradients_of_what_is_not_there(hb):  # noqa: F811
    none = dict(res=None, gate=None, dy=None, dres=None, dgate=None)
    plain = _params(hb, post=0, scale=None, post_weight=None)
    for i in (2, 3, 4):
        assert _bwd(hb, plain, [P if k == i else None for k in range(5)], **none) == 15
    assert _bwd(hb, plain, [None] * 5, **{**none, "dx": None}) == 12
    assert _bwd(hb, plain, [None] * 5, **{**none, "dy": P}) == 15
    assert _bwd(hb, plain, [None] * 5, **{**none, "dres": P}) == 15
    assert _bwd(hb, _params(hb, kind=0), [None] * 5) == 15                      # dh of no norm
    assert _bwd(hb, _params(hb, kind=0), [P, None, None, None, None], dh=None) == 15
    assert _bwd(hb, dparam=[P + 2, None, None, None, None], params=_params(hb, f32=1)) == 12
    # a plain norm has a kind, and no gate, scale or post norm
    for kw in (dict(kind=0, post=0, scale=None), dict(post=1, scale=None), dict(post=0, scale=P)):
        assert _norm(hb, _params(hb, **kw), res=None, gate=None) == 15


def test_no_rows_and_scratch(hb):  # noqa: F811
    assert _norm(hb, rows=0, x=None, res=P, gate=None, y=None, h=None, stats=None) == 0
    L = hb.lib()
    assert L.xtq_norm_bwd_ws_bytes(0, 100, 5) == 0 and L.xtq_norm_bwd_ws_bytes(7, 100, 0) == 0
    assert L.xtq_norm_bwd_ws_bytes(7, 100, 2) >= 800 and L.xtq_norm_bwd_ws_bytes(1 << 30, 32768, 5) > 0
    for bad in ((5, 0, 1), (5, 32769, 1), (-1, 5, 1), (5, 5, 6), (5, 5, -1)):
        assert L.xtq_norm_bwd_ws_bytes(*bad) == -6
