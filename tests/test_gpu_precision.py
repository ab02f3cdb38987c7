"""How far results of products with trellis weights may be from the definition: no further than their own
rounding puts them.

Tolerances.  A float16 result that is exact before it is rounded is off by the rounding of the exact value; x
enters with 22 bits and sums are fp32, together about 1e-5 of a result's norm, which adds in squares to the
2e-4 of the rounding: 2 % covers it.  (x rounded to 11 bits would add as much as the rounding itself, 40 %.)"""
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
    x[:, ::96] *= 15.0
    return (x * torch.exp(torch.randn(m, 1, generator=g) * 0.5)).to(dtype).cuda()


def _ratio(got, want):
    """The error of `got` over that of the rounded exact result (one row's bias gradient may have none)."""
    off = float((got.detach().cpu().double() - want).norm())
    return off and off / float((want.to(got.dtype).double() - want).norm())


ROWS = (1, 5, 16, 17, 40, 64, 65, 300)


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("act", ("none", "silu"))
@pytest.mark.parametrize("k,n,K", [(1280, 256, 4), (512, 384, 7)])
def test_fp16_results_are_rounded_once(xt, oracle_mod, m, act, k, n, K):
    w = R.random_weight(k, n, K, k + m)
    x = _x(m, k, torch.float16, m)
    want = R.act(x.cpu().double() @ R.dense(oracle_mod, *w, K, "exl3_mul1"), act)
    assert _ratio(xt.linear(x, xt.TrellisLinear(*w, K), act=act), want) <= 1.02


@pytest.mark.parametrize("K", range(2, 8))
@pytest.mark.parametrize("code", sorted(R.CODES))
def test_fp16_rows_apart(xt, oracle_mod, K, code):
    """Every width and codebook, rows transformed before the product in one, two and four groups of 16."""
    k, n = 1280, 128
    w = R.random_weight(k, n, K, 5 * K)
    W = R.dense(oracle_mod, *w, K, code)
    for m in (9, 30, 50):
        x = _x(m, k, torch.float16, m + K)
        assert _ratio(xt.linear(x, xt.TrellisLinear(*w, K, code=code)), x.cpu().double() @ W) <= 1.02


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("act", ("none", "relu", "silu", "gelu"))
@pytest.mark.parametrize("fast", (False, True))
def test_same_result_with_a_gradient(xt, dtype, act, fast):
    """A call under no_grad and one whose inputs need gradients: the same bits."""
    k, n, K = 1280, 384, 4
    layer = xt.TrellisLinear(*R.random_weight(k, n, K, 3), K)
    for m in ROWS:
        x = _x(m, k, dtype, m)
        with torch.no_grad():
            want = layer(x, act=act, fast=fast)
        assert torch.equal(layer(x.requires_grad_(), act=act, fast=fast).detach(), want), m


@pytest.mark.parametrize("m", (3, 12, 40, 300))
def test_fast(xt, oracle_mod, m):
    """The caller's choice of 11 bits: two roundings of 2^-11 in float16 (root of 2, and a tenth for the rows'
    spread in 128 values), nothing in bfloat16 without relu."""
    k, n, K = 1280, 384, 4
    w = R.random_weight(k, n, K, 4)
    layer = xt.TrellisLinear(*w, K)
    x = _x(m, k, torch.float16, m)
    want = x.cpu().double() @ R.dense(oracle_mod, *w, K, "exl3_mul1")
    assert _ratio(layer(x, fast=True), want) <= 1.1 * 2 ** 0.5
    b = _x(m, k, torch.bfloat16, m)
    assert torch.equal(layer(b, fast=True), layer(b))


@pytest.mark.parametrize("m", (1, 16, 40, 300))
@pytest.mark.parametrize("act", ("none", "silu", "gelu"))
def test_fp16_gradients_are_rounded_once(xt, oracle_mod, m, act):
    """dx and dbias.  The slope is taken at z rounded to float16: |z act''(z)| <= 0.32 times z's rounding, over a
    slope of 0.6 at the root of the mean square: 0.53 of the result's own rounding, 1.13 in squares; 1.2 for the
    chance of few rows."""
    k, n, K = 512, 1280, 4
    w = R.random_weight(k, n, K, 6)
    W = R.dense(oracle_mod, *w, K, "exl3_mul1")
    x = _x(m, k, torch.float16, m).requires_grad_()
    bias = torch.randn(n, generator=torch.Generator().manual_seed(1)).half().cuda().requires_grad_()
    dy = _x(m, n, torch.float16, m + 1)
    y = xt.linear(x, xt.TrellisLinear(*w, K), bias=bias, act=act)
    dx, db = torch.autograd.grad(y, (x, bias), dy)
    dz = dy.cpu().double() * R.slope(x.detach().cpu().double() @ W + bias.detach().cpu().double(), act)
    most = 1.02 if act == "none" else 1.2
    assert _ratio(dx, dz @ W.t()) <= most
    assert _ratio(db, dz.sum(0)) <= most
