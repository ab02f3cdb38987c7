"""Products with trellis weights and Grams on paths of their kernels that take sizes of their own, against the
definitions in 64 bits."""
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


def _x(m, k, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g)
    x[:, ::96] *= 10.0
    return (x * torch.exp(torch.randn(m, 1, generator=g) * 0.3)).to(dtype).cuda()


def _whole(got, want):
    return float(R.row_errors(got.reshape(1, -1), want.reshape(1, -1)).max())


@pytest.mark.parametrize("m", (70, 300))
@pytest.mark.parametrize("k", (128, 256))
@pytest.mark.parametrize("act,dtype", [("relu", torch.bfloat16), ("relu", torch.float16), ("silu", torch.float16),
                                       ("none", torch.float16)])
def test_two_terms_unsplit(xt, oracle_mod, m, k, act, dtype):
    """Many rows of 22 bits whose summed dimension is not cut, and their gradient.  Results are rounded once;
    gradients too, and take slopes at a rounded z (half a rounding more); relu's 4e-7 of wrong sides are 5e-4."""
    n, K = 384, 4
    w = R.random_weight(k, n, K, 81)
    W = R.dense(oracle_mod, *w, K, "exl3_mul1")
    x = _x(m, k, dtype, m).requires_grad_()
    dy = _x(m, n, dtype, m + 1)
    y = xt.linear(x, xt.TrellisLinear(*w, K), act=act)
    dx, = torch.autograd.grad(y, x, dy)
    z = x.detach().cpu().double() @ W
    u = R.roundoff(dtype)
    assert _whole(y, R.act(z, act)) <= u + 2e-5
    # (bf16: dz enters its product with 11 bits)
    tol = 1.5 * u + 5e-4 + (2.0 ** -11 if dtype == torch.bfloat16 else 0.0)
    assert _whole(dx, (dy.cpu().double() * R.slope(z, act)) @ W.t()) <= tol


@pytest.mark.parametrize("act", ("none", "relu", "silu", "gelu"))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("bias_dtype", ("same", torch.float32))
@pytest.mark.parametrize("m", (1, 19, 300))
def test_bias_gradient_alone(xt, oracle_mod, act, dtype, bias_dtype, m):
    """Only the bias needs a gradient: the sum of dy times slopes at a rounded z (less than one rounding of the
    activations' type; relu's wrong sides 5e-4), rounded to the bias' type."""
    k, n, K = 256, 640, 3
    bias_dtype = dtype if bias_dtype == "same" else bias_dtype
    w = R.random_weight(k, n, K, 91)
    x, dy = _x(m, k, dtype, m), _x(m, n, dtype, m + 1)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(1)).to(bias_dtype).cuda().requires_grad_()
    y = xt.linear(x, xt.TrellisLinear(*w, K), bias=bias, act=act)
    db, = torch.autograd.grad(y, bias, dy)
    assert db.dtype == bias_dtype and db.shape == (n,)
    z = x.cpu().double() @ R.dense(oracle_mod, *w, K, "exl3_mul1") + bias.detach().cpu().double()
    want = (dy.cpu().double() * R.slope(z, act)).sum(0)
    slopes = {"none": 0.0, "relu": 5e-4}.get(act, R.roundoff(dtype))
    assert _whole(db, want) <= slopes + R.roundoff(bias_dtype) + 1e-5


@pytest.mark.parametrize("t,k", [(9000, 384), (8900, 640), (8193, 1152)])
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_gram_half_tiles(xt, t, k, dtype):
    """Grams over transposed rows whose last tile of 256 columns is half empty, in parts over several columns of
    tiles.  fp32 sums of t / 32 steps are off by 2^-24 of their size a step at most."""
    valid = torch.rand(t, generator=torch.Generator().manual_seed(t)) < 0.8
    x = _x(t, k, dtype, t)
    xd = x.double() * valid.cuda()[:, None]
    want = xd.t().contiguous() @ xd
    x[~valid.cuda()] = float("nan")
    prev = torch.randn(k, k, generator=torch.Generator().manual_seed(k)).cuda()
    got = xt.input_gram(x, valid=valid.cuda())
    assert torch.equal(got, got.t())
    assert float((got - want).norm() / want.norm()) <= t / 32 * 2 ** -24
    assert torch.equal(xt.input_gram(x, valid=valid.cuda(), prev=prev), prev + got)
    acc = prev.clone()
    xt.input_gram(x, valid=valid.cuda(), prev=acc, out=acc)
    assert torch.equal(acc, prev + got)
