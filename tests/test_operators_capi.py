"""The C entries of the operators on trellis weights refuse what their kernels do not take, with the documented
status codes, before they touch a device: no pointer here is ever read."""
import ctypes
import os
import subprocess

import pytest

from conftest import PKG

P = 0x10000                             # an address of every alignment


@pytest.fixture(scope="module")
def hb():
    if not os.path.exists(os.path.join(PKG, "lib", "libexl3vit.so")):
        subprocess.run(["make", "-s", "-C", PKG], check=True)
    import hip_backend
    hip_backend.lib()
    return hip_backend


def _weight(hb, k=256, n=384, K=4, code=b"exl3_mul1", trellis=P, suh=P, svh=P):
    return hb.TrellisWeight(trellis, suh, svh, 1.0, k, n, K, code)


def _linear(hb, w=None, **kw):
    w = _weight(hb) if w is None else w
    a = dict(type=0, x=P, xs=w.k, rows=5, bias=None, f32=0, act=0, res=None, rs=0, z=None, y=P, ys=w.n, ws=P,
             nws=1 << 40, counters=P, stream=None)
    a.update(kw)
    return hb.lib().xtq_linear_dev(ctypes.byref(w), *a.values())


def _bwd(hb, w=None, **kw):
    w = _weight(hb) if w is None else w
    a = dict(type=0, dy=P, dys=w.n, z=P, act=2, rows=5, dx=P, dxs=w.k, dbias=None, f32=0, ws=P, nws=1 << 40,
             counters=P, stream=None)
    a.update(kw)
    return hb.lib().xtq_linear_bwd_dev(ctypes.byref(w), *a.values())


def _moe(hb, **kw):
    a = dict(table=P, experts=8, d=256, f=384, code=b"mul1", type=0, x=P, xs=256, rows=5, router=P, f32=0, top=2,
             act=2, renorm=1, valid=None, res=None, rs=0, y=P, ys=256, ids=P, weights=P, ws=P, nws=1 << 40,
             counters=P, stream=None)
    a.update(kw)
    return hb.lib().xtq_moe_dev(*a.values())


def _gram(hb, **kw):
    a = dict(type=0, x=P, xs=256, rows=5, k=256, valid=None, prev=None, out=P, ws=P, nws=1 << 40, stream=None)
    a.update(kw)
    return hb.lib().xtq_gram_dev(*a.values())


@pytest.mark.parametrize("entry", (_linear, _bwd))
@pytest.mark.parametrize("kw,rc", [
    (dict(k=0), 6), (dict(k=130), 6), (dict(n=64), 6), (dict(n=-128), 6), (dict(k=(1 << 22) + 128), 6),
    (dict(K=1), 9), (dict(K=8), 9), (dict(code=b"qtip_1mad"), 8), (dict(code=b"ih2x2"), 8), (dict(code=None), 12),
    (dict(trellis=None), 12), (dict(suh=None), 12), (dict(svh=None), 12), (dict(trellis=P + 1), 12),
    (dict(svh=P + 1), 12)])
def test_weights(hb, entry, kw, rc):
    assert entry(hb, _weight(hb, **kw)) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(type=2), 15), (dict(type=-1), 15), (dict(act=4), 15), (dict(act=-1), 15), (dict(rows=-1), 6),
    (dict(rows=1048561), 6), (dict(x=None), 12), (dict(x=P + 1), 12), (dict(xs=255), 6), (dict(y=None), 12),
    (dict(ys=383), 6), (dict(res=P, rs=383), 6), (dict(res=P + 1, rs=384), 12), (dict(z=P + 1), 12),
    (dict(bias=P + 1), 12), (dict(bias=P + 2, f32=1), 12), (dict(counters=None), 12), (dict(counters=P + 2), 12),
    (dict(ws=None), 12), (dict(ws=P + 8), 12), (dict(nws=100), 14)])
def test_linear(hb, kw, rc):
    assert _linear(hb, **{"rows": 70, **kw}) == rc      # (rows whose product takes scratch)


@pytest.mark.parametrize("kw,rc", [
    (dict(type=2), 15), (dict(act=4), 15), (dict(rows=0), 6), (dict(rows=1048561), 6), (dict(dy=None), 12),
    (dict(dys=383), 6), (dict(z=None), 12), (dict(z=P + 1), 12), (dict(dx=None), 12), (dict(dxs=255), 6),
    (dict(dbias=P + 1), 12), (dict(dbias=P + 2, f32=1), 12), (dict(counters=None), 12), (dict(ws=None), 12),
    (dict(nws=100), 14)])
def test_linear_bwd(hb, kw, rc):
    assert _bwd(hb, **kw) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(table=None), 12), (dict(table=P + 4), 12), (dict(code=None), 12), (dict(code=b"1mad"), 8),
    (dict(type=3), 15), (dict(act=9), 15), (dict(rows=65), 6), (dict(rows=-1), 6), (dict(experts=0), 6),
    (dict(experts=513), 6), (dict(top=0), 6), (dict(top=9), 6), (dict(top=17, experts=64), 6), (dict(d=200, xs=200), 6),
    (dict(f=64), 6), (dict(d=(1 << 20) + 128, xs=1 << 21, ys=1 << 21), 6), (dict(x=None), 12), (dict(xs=255), 6),
    (dict(y=None), 12), (dict(ys=255), 6), (dict(res=P, rs=255), 6), (dict(router=None), 12),
    (dict(router=P + 2, f32=1), 12), (dict(ids=None), 12), (dict(weights=P + 2), 12), (dict(counters=None), 12),
    (dict(ws=P + 8), 12), (dict(nws=100), 14)])
def test_moe(hb, kw, rc):
    assert _moe(hb, **kw) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(type=2), 15), (dict(k=0), 6), (dict(k=130, xs=130), 6), (dict(k=(1 << 22) + 128, xs=1 << 23), 6),
    (dict(rows=-1), 6), (dict(rows=(1 << 30) + 1), 6), (dict(x=None), 12), (dict(x=P + 1), 12), (dict(xs=255), 6),
    (dict(out=None), 12), (dict(out=P + 2), 12), (dict(prev=P + 2), 12), (dict(rows=9000, ws=None), 12),
    (dict(rows=9000, nws=100), 14)])
def test_gram(hb, kw, rc):
    assert _gram(hb, **kw) == rc


def test_no_rows(hb):
    assert _linear(hb, rows=0, x=None, ws=None, nws=0, counters=None) == 0
    assert _moe(hb, rows=0, x=None, ws=None, nws=0, counters=None) == 0


def test_scratch_sizes(hb):
    L = hb.lib()
    w = _weight(hb)
    p = ctypes.byref(w)
    assert L.xtq_linear_ws_bytes(p, 0, 0) == 0 and L.xtq_linear_ws_bytes(p, 5, 3) == -15
    assert L.xtq_linear_ws_bytes(p, -1, 0) == -6 and L.xtq_linear_ws_bytes(ctypes.byref(_weight(hb, k=1)), 5, 0) == -6
    for rows in (1, 16, 17, 64, 65, 1000, 1048560):
        one, two = L.xtq_linear_ws_bytes(p, rows, 0), L.xtq_linear_ws_bytes(p, rows, 2)
        assert 0 <= one <= two and L.xtq_linear_ws_bytes(p, rows, 1) > 0
    assert L.xtq_moe_ws_bytes(0, 8, 2, 256, 384) == 0 and L.xtq_moe_ws_bytes(65, 8, 2, 256, 384) == -6
    assert L.xtq_moe_ws_bytes(64, 8, 2, 256, 384) > L.xtq_moe_ws_bytes(1, 8, 2, 256, 384) > 0
    assert L.xtq_gram_ws_bytes(5, 256) == 0 and L.xtq_gram_ws_bytes(9000, 256) > 0 and L.xtq_gram_ws_bytes(5, 3) == -6
    # sizes past 32 bits
    big = _weight(hb, k=65536, n=65536)
    assert L.xtq_linear_ws_bytes(ctypes.byref(big), 1048560, 0) > 2 * 65536 * (1048560 + 65536)
    assert L.xtq_gram_ws_bytes(1 << 30, 256) > 2 * 256 << 30


def test_table(hb):
    L = hb.lib()

    def table(*ws):
        host = (hb.TrellisWeight * len(ws))(*ws)
        words = (ctypes.c_int64 * (4 * len(ws)))()
        return L.xtq_moe_table(host, len(ws) // 3, words), words

    gate, down = _weight(hb), _weight(hb, k=384, n=256, K=5, trellis=P + 64)
    rc, words = table(gate, gate, down)
    assert rc == 0 and words[0] == P and words[8] == P + 64 and words[11] >> 32 == 5
    assert table(gate, gate, gate)[0] == 6 and table(gate, down, down)[0] == 6
    assert table(gate, _weight(hb, K=9), down)[0] == 9
    assert table(gate, _weight(hb, code=b"mcg"), down)[0] == 8
    assert table(gate, _weight(hb, suh=None), down)[0] == 12
    assert L.xtq_moe_table(None, 1, words) == 12
    host = (hb.TrellisWeight * 3)(gate, gate, down)
    assert L.xtq_moe_table(host, 0, words) == 6 and L.xtq_moe_table(host, 513, words) == 6


def test_messages(hb):
    for rc in (6, 8, 9, 12, 14, 15):
        assert hb.lib().xtq_vit_strerror(rc) not in (b"", b"unknown status")
