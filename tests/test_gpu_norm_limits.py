"""The ends of the norms' documented range: rows (for "layer" their deviations) of a 2-norm just below 2^64, and with
eps 0 of a root mean square just above 2^-63; forward and gradients against the definitions in 64 bits.

Tolerances as in test_gpu_norm.py: a row is held to its one rounding, u, and 2e-5 of its norm, a gradient to u and 4e-5
of the row before its projections.  At the lower end a square is off by half of fp32's smallest step, 2^-150, which is
2^-24 of its mean (2^-126) at most: within those."""
import pytest
import torch

import trellis_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def xt():
    import trellis_ops
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    trellis_ops._hb.lib()
    return trellis_ops


def _centred(t, kind):
    return t - t.mean(-1, keepdim=True) if kind == "layer" else t


def _rows(m, d, kind, size, mean):
    """bfloat16 rows whose 2-norm (of the deviations) is `size`, within their rounding, around `mean` of their rms."""
    g = torch.Generator("cuda").manual_seed(d)
    x = torch.randn(m, d, generator=g, device="cuda", dtype=torch.float64)
    x = _centred(x, "layer")
    x = x / x.norm(dim=-1, keepdim=True) * size
    return (x + (mean * size / d ** 0.5 if kind == "layer" else 0.0)).bfloat16()


def _check(xt, x, kind, eps):
    m, d = x.shape
    g = torch.Generator("cuda").manual_seed(1)
    w = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).requires_grad_()
    dh = torch.randn(m, d, generator=g, device="cuda").bfloat16()
    x.requires_grad_()
    h = xt.norm(x, w, kind=kind, eps=eps)
    dx, dw = torch.autograd.grad(h, (x, w), dh)
    xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    c = _centred(xd, kind)
    rstd = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    want = c * rstd * wd
    wx, ww = torch.autograd.grad(want, (xd, wd), dh.double())
    u = R.roundoff(torch.bfloat16)
    assert bool(((h.double() - want).norm(dim=-1) <= (u + 2e-5) * want.norm(dim=-1)).all())
    before = (dh.double() * wd * rstd).norm(dim=-1)
    assert bool(((dx.double() - wx).norm(dim=-1) <= u * wx.norm(dim=-1) + 4e-5 * before).all())
    assert float((dw.double() - ww).norm()) <= 4e-5 * float((dh.double() * c * rstd).detach().norm())


@pytest.mark.parametrize("kind", ("rms", "layer"))
@pytest.mark.parametrize("m,d", [(5, 7), (20, 100), (9, 200), (5, 400), (7, 1000), (3, 5120), (2, 9000), (2, 32768)])
def test_large_rows(xt, m, d, kind):
    _check(xt, _rows(m, d, kind, 0.99 * 2.0 ** 64, 0.5), kind, 1e-6)


@pytest.mark.parametrize("kind", ("rms", "layer"))
@pytest.mark.parametrize("m,d", [(5, 7), (20, 100), (9, 200), (5, 400), (7, 1000), (3, 5120), (2, 9000), (2, 32768)])
def test_small_rows_without_eps(xt, m, d, kind):
    _check(xt, _rows(m, d, kind, 1.02 * 2.0 ** -63 * d ** 0.5, 0.5), kind, 0.0)
