"""Infinite parameters of a residual sum: the sums over the rows that they make infinite are infinite, as the definition's
are, however many of a workgroup's places have a row; the other channels' are finite and right.

Tolerance: a channel's sum of m products of fp32 values, each off by a few units of 2^-24: 1e-5 of the products' norm."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def xt():
    import trellis_ops
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    trellis_ops._hb.lib()
    return trellis_ops


@pytest.mark.parametrize("d", (7, 100, 200, 400, 1000, 7000))
@pytest.mark.parametrize("m", (1, 5, 16, 33))
@pytest.mark.parametrize("name", ("scale", "post_weight"))
@pytest.mark.parametrize("gate", (False, True))
def test_sums_over_the_rows(xt, d, m, name, gate):
    g = torch.Generator("cuda").manual_seed(d + m)
    x, res, dy = (torch.randn(m, d, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    dy = dy.abs() * x.sign()                        # every product of the infinite channel has one sign
    e = torch.rand(m, d, generator=g, device="cuda").bfloat16() + 0.5 if gate else None
    v = {n: (1 + torch.rand(d, generator=g, device="cuda")) for n in ("scale", "post_weight")}
    v[name][0] = float("inf")
    leaves = {n: t.clone().requires_grad_() for n, t in v.items()}
    y, _ = xt.residual_norm(x, res, kind=None, post="rms", gate=e, **leaves)
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    xd, dyd = x.double(), dy.double() * (1.0 if e is None else e.double())
    hat = xd / torch.sqrt((xd * xd).mean(-1, keepdim=True) + 1e-6)
    for n, other in (("scale", "post_weight"), ("post_weight", "scale")):
        terms = dyd * hat * v[other].double()
        want = terms.sum(0)
        assert float(want[0]) == (float("inf") if n != name else float(want[0])), n
        assert float(got[n][0]) == float("inf") if n != name else bool(got[n][0].isfinite()), n
        off = (got[n][1:].double() - want[1:]).norm()
        assert float(off) <= 1e-5 * float(terms[:, 1:].norm()), n
