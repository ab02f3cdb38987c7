"""Products with trellis weights (trellis_ops.linear), their gradients, and the input Gram, against the
definitions in 64 bits.

Tolerances.  An activation is rounded to fp16 once after its transform (relative 2^-11 of each value; the
weight's incoherent columns carry that into a result's row as the same share of its norm, up to twice it at
128 columns), a result once to its type; sums are fp32 (2^-24 sqrt(k) and less).  A row's error is held to
2 (u + 2 * 2^-11) of its norm, u the result's roundoff: the factor 2 is for activations, whose slopes go up to
1.13 while they make the row smaller.  A saved pre-activation is rounded to the activations' type, which moves
a gradient by less than u / 2 of its norm; where slopes are taken at it, it comes from activations of 22 bits
(relu, and fp16), or its error is below bf16's roundoff.  Gram sums are fp32 sums of exact products: 2^-24 times the steps'
chain of at most rows / 16 additions is their worst case, 1e-6 of the norm covers its square root."""
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


def _x(m, k, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g)
    x[:, ::96] *= 15.0
    return (x * torch.exp(torch.randn(m, 1, generator=g) * spread)).to(dtype).cuda()


def _tol(dtype):
    return 2 * (R.roundoff(dtype) + 2 * 2.0 ** -11)


ROWS = (1, 2, 15, 16, 17, 48, 63, 64, 65, 130, 257)


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("k,n,K", [(128, 128, 4), (640, 384, 3), (1152, 896, 7)])
def test_linear_rows(xt, oracle_mod, m, k, n, K):
    """Row counts around the tiles of 16, 64 and 256 rows; widths that end inside a tile of 256 columns."""
    dtype = torch.float16 if m % 2 else torch.bfloat16
    w = R.random_weight(k, n, K, k + K)
    x = _x(m, k, dtype, m)
    want = x.cpu().double() @ R.dense(oracle_mod, *w, K, "exl3_mul1")
    got = xt.linear(x, xt.TrellisLinear(*w, K))
    assert got.dtype == dtype and got.shape == (m, n)
    assert float(R.row_errors(got, want).max()) <= _tol(dtype)


@pytest.mark.parametrize("K", range(2, 8))
@pytest.mark.parametrize("code", sorted(R.CODES))
@pytest.mark.parametrize("m", (3, 200))
def test_linear_codes(xt, oracle_mod, K, code, m):
    """Every width and codebook, forward and gradient, with a scale of the whole weight."""
    k, n = 384, 256
    w = R.random_weight(k, n, K, 7 * K)
    x = _x(m, k, torch.float16, K).requires_grad_()
    W = R.dense(oracle_mod, *w, K, code, scale=0.375)
    y = xt.linear(x, xt.TrellisLinear(*w, K, code=code, scale=0.375))
    assert float(R.row_errors(y, x.detach().cpu().double() @ W).max()) <= _tol(torch.float16)
    dy = _x(m, n, torch.float16, K + 50)
    dx, = torch.autograd.grad(y, x, dy)
    assert float(R.row_errors(dx, dy.cpu().double() @ W.t()).max()) <= _tol(torch.float16)


@pytest.mark.parametrize("K", range(2, 8))
@pytest.mark.parametrize("code", sorted(R.CODES))
def test_linear_rows_apart(xt, oracle_mod, K, code):
    """Few rows that are transformed before the product's launch, in one, two and four groups of 16, places of the
    last group left over."""
    k, n = 1280, 128
    w = R.random_weight(k, n, K, 3 * K)
    W = R.dense(oracle_mod, *w, K, code)
    for m in (9, 30, 50):
        x = _x(m, k, torch.bfloat16, m + K)
        y = xt.linear(x, xt.TrellisLinear(*w, K, code=code))
        assert float(R.row_errors(y, x.cpu().double() @ W).max()) <= _tol(torch.bfloat16)


@pytest.mark.parametrize("m,k,n", [(9000, 128, 1152), (3000, 2048, 384), (1815, 4096, 2176)])
def test_linear_cuts(xt, oracle_mod, m, k, n):
    """Every way in which a product of many rows is cut: both heights of tile, whole and in parts."""
    w = R.random_weight(k, n, 4, 5)
    W = R.dense(oracle_mod, *w, 4, "exl3_mul1").cuda()
    x = _x(m, k, torch.float16, m, spread=0.5)
    y = xt.linear(x, xt.TrellisLinear(*w, 4))
    assert float(R.row_errors(y.cpu(), (x.double() @ W).cpu()).max()) <= _tol(torch.float16)


@pytest.mark.parametrize("act", ("none", "relu", "silu", "gelu"))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("m,with_bias,with_res", [(5, True, False), (40, False, True), (300, True, True)])
def test_linear_epilogue(xt, oracle_mod, act, dtype, m, with_bias, with_res):
    k, n, K = 256, 384, 5
    w = R.random_weight(k, n, K, 11)
    x = _x(m, k, dtype, m)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(1)).cuda()
    bias = (bias if m == 300 else bias.to(dtype)) if with_bias else None
    res = _x(m, n, dtype, m + 1) if with_res else None
    z = x.cpu().double() @ R.dense(oracle_mod, *w, K, "exl3_mul1")
    if with_bias:
        z = z + bias.cpu().double()
    want = R.act(z, act) + (res.cpu().double() if with_res else 0)
    got = xt.linear(x, xt.TrellisLinear(*w, K), bias=bias, act=act, residual=res)
    assert float(R.row_errors(got, want).max()) <= _tol(dtype)


@pytest.mark.parametrize("act", ("none", "relu", "silu", "gelu"))
@pytest.mark.parametrize("dtype,bias_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("m", (1, 33, 270))
def test_linear_gradient(xt, oracle_mod, act, dtype, bias_dtype, m):
    """dx, dbias and dresidual against the formula, dx and dbias also against differences of the function."""
    k, n, K = 512, 256, 4
    w = R.random_weight(k, n, K, 21)
    W = R.dense(oracle_mod, *w, K, "exl3_mul1")
    x = _x(m, k, dtype, m).requires_grad_()
    bias = torch.randn(n, generator=torch.Generator().manual_seed(2)).to(bias_dtype).cuda().requires_grad_()
    res = _x(m, n, dtype, 5).requires_grad_()
    dy = _x(m, n, dtype, 6, spread=0.3)
    y = xt.linear(x, xt.TrellisLinear(*w, K), bias=bias, act=act, residual=res)
    dx, db, dr = torch.autograd.grad(y, (x, bias, res), dy)
    assert dx.dtype == dtype and db.dtype == bias_dtype and torch.equal(dr, dy)
    xd, bd, dyd = x.detach().cpu().double(), bias.detach().cpu().double(), dy.cpu().double()
    z = xd @ W + bd
    dz = dyd * R.slope(z, act)
    tol = _tol(dtype) + R.roundoff(dtype) / 2
    assert float(R.row_errors(dx, dz @ W.t()).max()) <= tol
    assert float(R.row_errors(db[None], dz.sum(0)[None]).max()) <= tol
    # differences along a direction that the gradient itself does not know
    g = torch.Generator().manual_seed(3)
    v, u = torch.randn(m, k, generator=g).double(), torch.randn(n, generator=g).double()
    h = 1e-6

    def f(a, b):
        return float((dyd * R.act(a @ W + b, act)).sum())

    dif = (f(xd + h * v, bd) - f(xd - h * v, bd)) / (2 * h)
    got = float((dx.cpu().double() * v).sum())
    assert abs(got - dif) <= tol * float((dz @ W.t()).norm() * 4) + 1e-5
    dif = (f(xd, bd + h * u) - f(xd, bd - h * u)) / (2 * h)
    got = float((db.cpu().double() * u).sum())
    assert abs(got - dif) <= tol * float(dz.sum(0).norm() * 4) + 1e-5


@pytest.mark.parametrize("act,dtype", [("relu", torch.bfloat16), ("relu", torch.float16), ("silu", torch.float16),
                                       ("gelu", torch.float16)])
@pytest.mark.parametrize("m", (12, 40, 300))
def test_linear_gradient_takes_exact_slopes(xt, oracle_mod, act, dtype, m):
    """The slopes are those at the exact z: with an error e of z's norm, relu would take the wrong side of zero for
    e / pi of all values and be off by sqrt(2 e / pi) (0.011 for activations of 11 bits).  Tolerance of the whole
    dx: 3/4 of the result's roundoff and of 2^-11 (their root mean squares are below), and for e = 4e-7 (22 bits,
    fp32 sums) 5e-4."""
    k, n, K = 512, 512, 4
    w = R.random_weight(k, n, K, 71)
    W = R.dense(oracle_mod, *w, K, "exl3_mul1")
    x = _x(m, k, dtype, m, spread=0.3).requires_grad_()
    dy = _x(m, n, dtype, 7, spread=0.3)
    y = xt.linear(x, xt.TrellisLinear(*w, K), act=act)
    dx, = torch.autograd.grad(y, x, dy)
    z = x.detach().cpu().double() @ W
    want = (dy.cpu().double() * R.slope(z, act)) @ W.t()
    tol = 0.75 * (R.roundoff(dtype) + 2.0 ** -11) + 5e-4
    assert float(R.row_errors(dx.reshape(1, -1), want.reshape(1, -1)).max()) <= tol


@pytest.mark.parametrize("m", (3, 70))
def test_linear_magnitudes(xt, oracle_mod, m):
    """Rows of very different size, of zeros, and with values near the type's ends."""
    k, n, K = 384, 256, 4
    w = R.random_weight(k, n, K, 31)
    W = R.dense(oracle_mod, *w, K, "exl3_mul1")
    layer = xt.TrellisLinear(*w, K)
    for dtype, sizes in ((torch.bfloat16, (1e30, 0.0, 1e-30)), (torch.float16, (6e4, 0.0, 2e-4))):
        x = _x(m, k, torch.float32, 9, spread=0.0)
        x = (x / x.abs().max() * torch.tensor([sizes[i % 3] for i in range(m)]).cuda()[:, None]).to(dtype)
        want = x.cpu().double() @ W
        got = xt.linear(x, layer)
        # the smallest fp16 results are multiples of 2^-24
        err = (got.cpu().double() - want).norm(dim=1)
        floor = 2.0 ** -24 * n ** 0.5 if dtype == torch.float16 else 0.0
        assert bool((err <= _tol(dtype) * want.norm(dim=1) + floor).all())
        assert bool((got[1::3] == 0).all())


@pytest.mark.parametrize("m,step", [(3, 2 ** 31), (70, 2 ** 26)])
def test_far_rows(xt, m, step):
    """Rows whose offsets pass 2^32 elements give what the same rows give side by side, bit for bit."""
    k, n = 256, 384
    near, res = _x(m, k, torch.float16, 3), _x(m, n, torch.float16, 4)
    slots = torch.empty(70 * 2 ** 26, dtype=torch.float16, device="cuda")
    x, r = slots.as_strided((m, k), (step, 1)), slots.as_strided((m, n), (step, 1), 2048)
    x.copy_(near)
    r.copy_(res)
    w = xt.TrellisLinear(*R.random_weight(k, n, 4, 9), 4)
    assert torch.equal(xt.linear(x, w, residual=r), xt.linear(near, w, residual=res))
    assert torch.equal(xt.input_gram(x), xt.input_gram(near))
    x.requires_grad_()
    far, = torch.autograd.grad(xt.linear(x, w, act="silu"), x, res)
    near.requires_grad_()
    side, = torch.autograd.grad(xt.linear(near, w, act="silu"), near, res)
    assert torch.equal(far, side)
    if m <= 64:
        gate, down = xt.TrellisLinear(*R.random_weight(k, n, 3, 1), 3), xt.TrellisLinear(*R.random_weight(n, k, 4, 2), 4)
        experts = xt.TrellisExperts([gate, gate], [gate, gate], [down, down])
        router = _x(2, k, torch.float16, 5)
        with torch.no_grad():
            assert torch.equal(xt.moe(x, router, experts, 1, residual=x),
                               xt.moe(near, router, experts, 1, residual=near))


@pytest.mark.parametrize("m", (4, 80))
def test_linear_nonfinite_rows(xt, m):
    """A NaN or an infinity stays in its row."""
    k, n, K = 256, 256, 3
    w = R.random_weight(k, n, K, 41)
    layer = xt.TrellisLinear(*w, K)
    x = _x(m, k, torch.bfloat16, 4)
    clean = xt.linear(x, layer)
    bad = x.clone()
    bad[1, 5] = float("nan")
    bad[3, 200] = float("inf")
    got = xt.linear(bad, layer)
    keep = [i for i in range(m) if i not in (1, 3)]
    assert torch.equal(got[keep], clean[keep])
    assert not bool(torch.isfinite(got[1]).any()) and not bool(torch.isfinite(got[3]).all())


@pytest.mark.parametrize("m", (6, 100))
def test_linear_layouts(xt, m):
    """Leading dimensions, rows apart, odd addresses, transposed inputs, results in a residual's place; no rows."""
    k, n, K = 256, 128, 4
    w = R.random_weight(k, n, K, 51)
    layer = xt.TrellisLinear(*w, K)
    x = _x(m, k, torch.float16, 4)
    want = layer(x)
    assert torch.equal(layer(x.view(2, m // 2, k)), want.view(2, m // 2, n))
    wide = torch.full((m, k + 3), 7.0, dtype=x.dtype, device="cuda")
    wide[:, 1:k + 1] = x
    assert torch.equal(layer(wide[:, 1:k + 1]), want)
    assert torch.equal(layer(x.t().contiguous().t()), want)
    res = _x(m, n + 8, torch.float16, 8)[:, 3:n + 3]
    both = layer(x, residual=res)
    assert torch.equal(both, layer(x, residual=res.contiguous()))
    assert layer(x[:0]).shape == (0, n)
    assert layer(x[0]).shape == (n,)
    e = x[:0].detach().requires_grad_()
    b = torch.zeros(n, device="cuda", requires_grad=True)
    g = torch.autograd.grad(layer(e, bias=b).sum(), (e, b))
    assert g[0].shape == (0, k) and bool((g[1] == 0).all())
    ex = x[:1].expand(m, k)
    assert torch.equal(layer(ex), layer(ex.contiguous()))


@pytest.mark.parametrize("m", (2, 90))
def test_linear_repeats_and_streams(xt, m):
    """The same bits on every call, on another stream, and in a replayed graph with eager work in between."""
    k, n, K = 1024, 384, 4
    layer = xt.TrellisLinear(*R.random_weight(k, n, K, 61), K)
    x, x2 = _x(m, k, torch.bfloat16, 4), _x(m, k, torch.bfloat16, 5)
    want, want2 = layer(x, act="silu"), layer(x2, act="silu")
    for _ in range(5):
        assert torch.equal(layer(x, act="silu"), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = [layer(x, act="silu") for _ in range(3)]
    b = [layer(x2, act="silu") for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in a) and all(torch.equal(t, want2) for t in b)
    buf = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(buf, act="silu")
    for i in range(4):
        buf.copy_(x2 if i % 2 else x)
        graph.replay()
        assert torch.equal(layer(x, act="silu"), want)
        torch.cuda.synchronize()
        assert torch.equal(y, want2 if i % 2 else want)


def test_linear_refusals(xt):
    tr, su, sv = R.random_weight(256, 128, 4, 1)
    w = xt.TrellisLinear(tr, su, sv, 4)
    x = _x(3, 256, torch.float16, 1)
    for bad in (lambda: xt.linear(x.float(), w), lambda: xt.linear(x.cpu(), w), lambda: xt.linear(x[:, :128], w),
                lambda: xt.linear(x, w, act="tanh"), lambda: xt.linear(x, w, bias=sv[:64]),
                lambda: xt.linear(x, w, bias=sv.double()), lambda: xt.linear(x, w, residual=x),
                lambda: xt.linear(x, w, residual=torch.zeros(3, 128, device="cuda")),
                lambda: xt.TrellisLinear(tr, su, sv, 8), lambda: xt.TrellisLinear(tr, su, sv, 5),
                lambda: xt.TrellisLinear(tr, su[:128], sv, 4), lambda: xt.TrellisLinear(tr.int(), su, sv, 4),
                lambda: xt.TrellisLinear(tr.cpu(), su, sv, 4), lambda: xt.TrellisLinear(tr[:4], su[:64], sv, 4),
                lambda: xt.TrellisLinear(tr, su.float(), sv, 4)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        xt.TrellisLinear(tr, su, sv, 4, code="qtip_1mad")


@pytest.mark.parametrize("t,k", [(1, 128), (31, 256), (64, 384), (65, 128), (300, 640), (1000, 256), (5000, 128)])
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_gram(xt, t, k, dtype):
    g = torch.Generator().manual_seed(t)
    x = _x(t, k, dtype, t)
    valid = (torch.rand(t, generator=g) < 0.7).cuda()
    hidden = x.clone()
    hidden[~valid] = float("nan")
    prev = torch.randn(k, k, generator=g).cuda()
    xd = x.cpu().double()
    full, some = xd.t() @ xd, xd[valid.cpu()].t() @ xd[valid.cpu()]
    for got, want in ((xt.input_gram(x), full), (xt.input_gram(hidden, valid=valid), some),
                      (xt.input_gram(hidden, valid=valid, prev=prev), some + prev.cpu().double())):
        assert float(R.row_errors(got.reshape(1, -1), want.reshape(1, -1)).max()) <= 1e-6
    got = xt.input_gram(x)
    assert torch.equal(got, got.t())
    acc = prev.clone()
    assert xt.input_gram(x, prev=acc, out=acc) is acc
    assert torch.equal(acc, xt.input_gram(x, prev=prev))


@pytest.mark.parametrize("t,k,dtype", [(9000, 256, torch.float16), (1700, 4096, torch.bfloat16)])
def test_gram_many(xt, t, k, dtype):
    """Sums that come through transposed fragments: in parts that are joined, and finished by the product itself.
    fp32 sums of t / 32 steps are off by 2^-24 of their size a step at most."""
    valid = torch.rand(t, generator=torch.Generator().manual_seed(t)) < 0.7
    x = _x(t, k, dtype, t)
    xd = x.double() * valid.cuda()[:, None]
    want = xd.t().contiguous() @ xd
    x[~valid.cuda()] = float("inf")
    prev = torch.randn(k, k).cuda()
    got = xt.input_gram(x, valid=valid.cuda())
    assert torch.equal(got, got.t())
    assert float((got - want).norm() / want.norm()) <= t / 32 * 2 ** -24
    assert torch.equal(xt.input_gram(x, valid=valid.cuda(), prev=prev), prev + got)


def test_gram_edges(xt):
    x = _x(24, 256, torch.float16, 1)
    prev = torch.randn(256, 256).cuda()
    none = torch.zeros(24, dtype=torch.bool, device="cuda")
    assert bool((xt.input_gram(x, valid=none) == 0).all())
    assert torch.equal(xt.input_gram(x, valid=none, prev=prev), prev)
    assert torch.equal(xt.input_gram(x[:0], prev=prev), prev)
    assert bool((xt.input_gram(x[:0]) == 0).all())
    assert torch.equal(xt.input_gram(x.view(2, 12, 256)), xt.input_gram(x))
    wide = torch.full((24, 300), float("inf"), dtype=torch.float16, device="cuda")
    wide[:, 7:263] = x
    assert torch.equal(xt.input_gram(wide[:, 7:263]), xt.input_gram(x))
    for bad in (lambda: xt.input_gram(x.float()), lambda: xt.input_gram(x[:, :100]), lambda: xt.input_gram(x.cpu()),
                lambda: xt.input_gram(x, valid=none[:5]), lambda: xt.input_gram(x, valid=none.int()),
                lambda: xt.input_gram(x, prev=prev.double()), lambda: xt.input_gram(x, out=prev.t()),
                lambda: xt.input_gram(x, prev=prev[:128])):
        with pytest.raises(ValueError):
            bad()


def test_calibrate_quantize_run(xt):
    """The path of a calibration: run a quantized layer, gather the Gram of what it gives, quantize the next
    weight with it, multiply with that."""
    import quantize as xq
    g = torch.Generator().manual_seed(8)
    W1, W2 = torch.randn(256, 256, generator=g) / 16, torch.randn(128, 256, generator=g) / 16
    x = torch.randn(400, 256, generator=g).to(torch.bfloat16).cuda()
    G1 = xt.input_gram(x)
    r1 = xq.quantize_linear(W1, G1.cpu() / 400, K=4, device="cuda", channel_scales=True)
    h = xt.linear(x, xt.TrellisLinear.from_result(r1), act="silu")
    want = R.act(x.cpu().double() @ r1["W_hat"].double().t(), "silu")
    # suh and svh are what W_hat was computed from, in fp32: 1e-5 beside the results' own rounding
    assert float(R.row_errors(h, want).max()) <= _tol(torch.bfloat16) + 1e-5
    G2 = xt.input_gram(h[:200])
    xt.input_gram(h[200:], prev=G2, out=G2)
    r2 = xq.quantize_linear(W2, G2.cpu() / 400, K=3, device="cuda", channel_scales=False)
    y = xt.linear(h, xt.TrellisLinear.from_result(r2))
    want = h.cpu().double() @ r2["W_hat"].double().t()
    assert float(R.row_errors(y, want).max()) <= _tol(torch.bfloat16) + 1e-5
