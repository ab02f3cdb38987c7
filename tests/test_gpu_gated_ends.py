"""The gated projection at the ends of its range: as many rows as a call takes, and more blocks of columns than there are
counters, against the definition in 64 bits where it is sampled.  Float16: everything is rounded once, and the error is
held to that of the rounded exact result and 2 % (the operands' 22 bits), as in test_gpu_gated.py."""
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


def _ratio(got, want):
    off = float((got.detach().cpu().double() - want).norm())
    return off and off / float((want.to(got.dtype).double() - want).norm())


def _want(x, dy, Wg, Wu, b):
    zg, zu = x @ Wg + b, x @ Wu
    dg, du = dy * zu * R.slope(zg, "silu"), dy * R.act(zg, "silu")
    return R.act(zg, "silu") * zu, dg @ Wg.t() + du @ Wu.t(), dg


def test_most_rows(xt, oracle_mod):
    m, k, n = 1048560, 128, 128
    ws = [R.random_weight(k, n, 4, s) for s in (1, 2)]
    ls, (Wg, Wu) = [xt.TrellisLinear(*w, 4) for w in ws], [R.dense(oracle_mod, *w, 4, "exl3_mul1") for w in ws]
    g = torch.Generator("cuda").manual_seed(3)
    x, dy = (torch.randn(m, k, generator=g, device="cuda").half() for _ in range(2))
    b = torch.randn(n, generator=g, device="cuda").requires_grad_()
    x.requires_grad_()
    y = xt.gated(x, *ls, b)
    dx, db = torch.autograd.grad(y, (x, b), dy)
    for at in (0, 16383, 524288 - 7, m - 100):
        rows = slice(at, at + 100)
        wy, wx, _ = _want(x[rows].detach().cpu().double(), dy[rows].cpu().double(), Wg, Wu, b.detach().cpu().double())
        assert _ratio(y[rows], wy) <= 1.02 and _ratio(dx[rows], wx) <= 1.02
    _, _, dg = _want(x.detach().double(), dy.double(), Wg.cuda(), Wu.cuda(), b.detach().double())
    # sums of a million fp32 terms by chains of 16384 additions: 2^-24 of the terms' norm and the root of that, twice
    assert float((db.double() - dg.sum(0)).norm()) <= 2 * 2.0 ** -24 * 128 * float(dg.norm())
    with pytest.raises(Exception, match="rc=6"):
        xt.gated(torch.zeros(m + 1, k, device="cuda", dtype=torch.float16), *ls)


@pytest.mark.parametrize("m", (1, 40))
def test_more_columns_than_counters(xt, oracle_mod, m):
    k, n, cut = 128, 128 * 16385, 640
    ws = [R.random_weight(k, n, 2, s) for s in (1, 2)]
    ls = [xt.TrellisLinear(*w, 2) for w in ws]
    g = torch.Generator("cuda").manual_seed(3)
    x = torch.randn(m, k, generator=g, device="cuda").half().requires_grad_()
    places = [0, n // 2 // 128 * 128, n - cut]
    dy = torch.zeros(m, n, device="cuda", dtype=torch.float16)
    for at in places:
        dy[:, at:at + cut] = torch.randn(m, cut, generator=g, device="cuda").half()
    y = xt.gated(x, *ls)
    dx, = torch.autograd.grad(y, x, dy)
    xd, total = x.detach().cpu().double(), 0.0
    for at in places:
        dense = [R.dense(oracle_mod, tr[:, at // 16:(at + cut) // 16].contiguous(), suh, svh[at:at + cut], 2, "exl3_mul1")
                 for tr, suh, svh in ws]
        wy, wx, _ = _want(xd, dy[:, at:at + cut].cpu().double(), *dense, 0.0)
        assert _ratio(y[:, at:at + cut], wy) <= 1.02
        total = total + wx
    assert _ratio(dx, total) <= 1.02
