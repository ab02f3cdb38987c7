"""The gated projection on two trellis weights (trellis_ops.gated) and its gradients, against the definition in 64
bits.

Tolerances.  Each factor's activations are rounded once after their transform (as in test_gpu_linear.py: 2^-11 of a
row's norm and up to twice it at 128 columns; 2^-22 in float16 and for relu), and the result once, by at most u of
itself.  A row's product takes both factors' errors, of other elements each, and the activation's slope is up to 1.13
where it makes the factor smaller: 2 (u + 4 * 2^-11) of its norm.  Where 22 bits enter, what is left beside the one
rounding is 1e-5 of the norm a factor, and adds in squares: 2 % of the rounding covers it.  The factors are kept in
fp32 for the gradient, so the same holds there."""
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


def _x(m, k, dtype, seed, spread=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g)
    x[:, ::96] *= 15.0
    return (x * torch.exp(torch.randn(m, 1, generator=g) * spread)).to(dtype).cuda()


def _pair(xt, O, k, n, K1, K2, code="exl3_mul1", seed=1, scales=(1.0, 1.0)):
    """(gate, up) to multiply with and their dense weights in 64 bits."""
    ws = [R.random_weight(k, n, K, seed + i) for i, K in enumerate((K1, K2))]
    return ([xt.TrellisLinear(*w, K, code=code, scale=s) for w, K, s in zip(ws, (K1, K2), scales)],
            [R.dense(O, *w, K, code, s) for w, K, s in zip(ws, (K1, K2), scales)])


def _tol(dtype):
    return 2 * (R.roundoff(dtype) + 4 * 2.0 ** -11)


def _ratio(got, want):
    """The error of `got` over that of the rounded exact result."""
    off = float((got.detach().cpu().double() - want).norm())
    return off and off / float((want.to(got.dtype).double() - want).norm())


ROWS = (1, 2, 15, 16, 17, 33, 63, 64, 65, 128, 130, 192, 193, 256, 257)


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("k,n,K1,K2", [(128, 128, 4, 4), (640, 384, 3, 6), (1152, 896, 7, 2)])
def test_rows(xt, oracle_mod, m, k, n, K1, K2):
    """Row counts around the groups of 16 and the tiles, one block of columns and odd numbers of them."""
    dtype = torch.float16 if m % 2 else torch.bfloat16
    ls, (Wg, Wu) = _pair(xt, oracle_mod, k, n, K1, K2)
    x = _x(m, k, dtype, m)
    xd = x.cpu().double()
    got = xt.gated(x, *ls)
    assert got.dtype == dtype and got.shape == (m, n)
    assert float(R.row_errors(got, R.act(xd @ Wg, "silu") * (xd @ Wu)).max()) <= _tol(dtype)


@pytest.mark.parametrize("K", range(2, 8))
@pytest.mark.parametrize("code", sorted(R.CODES))
@pytest.mark.parametrize("m", (3, 12, 30, 50, 300))
def test_codes(xt, oracle_mod, K, code, m):
    """Every width and codebook beside another width, every kernel of few rows, forward and gradient, with scales of
    the whole weights.  Float16: everything is rounded once."""
    k, n = 1280, 256
    ls, (Wg, Wu) = _pair(xt, oracle_mod, k, n, K, 9 - K, code, seed=7 * K, scales=(0.375, 1.5))
    x = _x(m, k, torch.float16, K).requires_grad_()
    dy = _x(m, n, torch.float16, K + 50)
    y = xt.gated(x, *ls, act="gelu")
    dx, = torch.autograd.grad(y, x, dy)
    xd, dyd = x.detach().cpu().double(), dy.cpu().double()
    zg, zu = xd @ Wg, xd @ Wu
    assert _ratio(y, R.act(zg, "gelu") * zu) <= 1.02
    assert _ratio(dx, (dyd * zu * R.slope(zg, "gelu")) @ Wg.t() + (dyd * R.act(zg, "gelu")) @ Wu.t()) <= 1.02


@pytest.mark.parametrize("m,k,n", [(9000, 128, 640), (3000, 2048, 256), (1815, 1024, 2176), (300, 4096, 384),
                                   (150, 2048, 6144), (5000, 128, 1664), (1815, 4096, 1408), (333, 4096, 2816)])
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_cuts(xt, oracle_mod, m, k, n, dtype):
    """Every way in which the products of many rows are cut: every height of tile, whole and in parts."""
    ls, ws = _pair(xt, oracle_mod, k, n, 4, 5)
    Wg, Wu = (w.cuda() for w in ws)
    x = _x(m, k, dtype, m).requires_grad_()
    dy = _x(m, n, dtype, 3)
    y = xt.gated(x, *ls)
    dx, = torch.autograd.grad(y, x, dy)
    xd, dyd = x.detach().double(), dy.double()
    zg, zu = xd @ Wg, xd @ Wu
    a = zg / (1 + torch.exp(-zg))
    sig = 1 / (1 + torch.exp(-zg))
    want = (dyd * zu * sig * (1 + zg * (1 - sig))) @ Wg.t().contiguous() + (dyd * a) @ Wu.t().contiguous()
    assert float(R.row_errors(y, (a * zu).cpu()).max()) <= _tol(dtype)
    assert float(R.row_errors(dx, want.cpu()).max()) <= _tol(dtype)


@pytest.fixture(scope="module")
def wide(xt, oracle_mod):
    """A pair of more blocks of 128 columns than there are compute units: few rows' runs go over their ends."""
    ls, ws = _pair(xt, oracle_mod, 2048, 16640, 3, 5, seed=9)
    return ls, [w.cuda() for w in ws]


@pytest.mark.parametrize("m", (1, 7, 16, 30, 50, 64, 100, 130, 256))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_runs_over_blocks(xt, wide, m, dtype):
    ls, (Wg, Wu) = wide
    x = _x(m, 2048, dtype, m).requires_grad_()
    zg, zu = x.detach().double() @ Wg, x.detach().double() @ Wu
    want = (zg / (1 + torch.exp(-zg)) * zu).cpu()
    y = xt.gated(x, *ls)
    assert float(R.row_errors(y, want).max()) <= _tol(dtype)
    if dtype == torch.float16:
        assert _ratio(y, want) <= 1.02
    with torch.no_grad():
        assert all(torch.equal(xt.gated(x, *ls), y) for _ in range(5))


@pytest.mark.parametrize("act", ("none", "relu", "silu", "gelu"))
@pytest.mark.parametrize("dtype,bias_dtypes", [(torch.bfloat16, (torch.bfloat16, torch.float32)),
                                               (torch.float16, (torch.float32, torch.float16)),
                                               (torch.float16, (None, torch.float16)), (torch.bfloat16, (None, None))])
@pytest.mark.parametrize("m", (1, 5, 40, 300))
def test_gradient(xt, oracle_mod, act, dtype, bias_dtypes, m):
    """y, dx and the biases' gradients against the formula, and against differences of the function."""
    k, n = 512, 384
    ls, (Wg, Wu) = _pair(xt, oracle_mod, k, n, 5, 3, seed=21)
    x = _x(m, k, dtype, m).requires_grad_()
    g = torch.Generator().manual_seed(2)
    biases = [None if t is None else torch.randn(n, generator=g).to(t).cuda().requires_grad_() for t in bias_dtypes]
    dy = _x(m, n, dtype, 6, spread=0.3)
    y = xt.gated(x, *ls, gate_bias=biases[0], up_bias=biases[1], act=act)
    leaves = [t for t in (x, *biases) if t is not None]
    got = dict(zip([i for i, t in enumerate((x, *biases)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    xd, dyd = x.detach().cpu().double(), dy.cpu().double()
    bd = [torch.zeros(n, dtype=torch.float64) if b is None else b.detach().cpu().double() for b in biases]
    zg, zu = xd @ Wg + bd[0], xd @ Wu + bd[1]
    assert float(R.row_errors(y, R.act(zg, act) * zu).max()) <= _tol(dtype)
    dg, du = dyd * zu * R.slope(zg, act), dyd * R.act(zg, act)
    want = {0: dg @ Wg.t() + du @ Wu.t(), 1: dg.sum(0)[None], 2: du.sum(0)[None]}
    # relu's slope at the nearest zeros: e = 4e-7 of all values on the other side (22 bits), sqrt(2 e / pi) = 5e-4
    for i, t in got.items():
        assert t.dtype == leaves[list(got).index(i)].dtype
        t = t if i == 0 else t[None]
        assert float((t.cpu().double() - want[i]).norm() / want[i].norm()) <= _tol(dtype) + 5e-4, i
    h = 1e-6
    v = [torch.randn(*t.shape, generator=g).double() for t in (xd, *bd)]

    def f(s):
        a, b = xd @ Wg + bd[0], xd @ Wu + bd[1]
        a, b = a + s * (v[0] @ Wg + v[1]), b + s * (v[0] @ Wu + v[2])
        return float((dyd * R.act(a, act) * b).sum())

    if len(got) == 3:
        dif = (f(h) - f(-h)) / (2 * h)
        mine = sum(float((got[i].cpu().double() * v[i]).sum()) for i in range(3))
        size = sum(float(want[i].norm()) for i in range(3))
        assert abs(mine - dif) <= 4 * (_tol(dtype) + 5e-4) * size + 1e-4


@pytest.mark.parametrize("m", (1, 5, 16, 17, 40, 64, 65, 200, 300))
@pytest.mark.parametrize("act", ("none", "silu", "gelu"))
def test_rounded_once(xt, oracle_mod, m, act):
    """Float16 results and gradients are off by their one rounding; bfloat16's by that and 11 bits of the rows (0.0003
    of the norm a factor beside 0.0017, in squares: 6 %; both slopes in the gradient: 15 %).  The bias' bfloat16
    gradient is held to its worst rounding instead, u of each entry, and 2^-11 a factor: dy is 15 times as large in 14
    of the 1280 columns, whose sums make 0.71 of its square (14 * 225 / (14 * 225 + 1266)), and the roundings of 14 numbers, uniform in their steps, have a root mean square that
    varies by a quarter of itself, which a ratio to it would take for an error."""
    k, n = 768, 1280
    ls, (Wg, Wu) = _pair(xt, oracle_mod, k, n, 4, 6, seed=3)
    for dtype, y_most, g_most in ((torch.float16, 1.02, 1.02), (torch.bfloat16, 1.06, 1.15)):
        x = _x(m, k, dtype, m).requires_grad_()
        bias = torch.randn(n, generator=torch.Generator().manual_seed(1)).to(dtype).cuda().requires_grad_()
        dy = _x(m, n, dtype, m + 1)
        y = xt.gated(x, *ls, gate_bias=bias, act=act)
        dx, db = torch.autograd.grad(y, (x, bias), dy)
        xd, dyd = x.detach().cpu().double(), dy.cpu().double()
        zg, zu = xd @ Wg + bias.detach().cpu().double(), xd @ Wu
        assert _ratio(y, R.act(zg, act) * zu) <= y_most
        dg = dyd * zu * R.slope(zg, act)
        assert _ratio(dx, dg @ Wg.t() + (dyd * R.act(zg, act)) @ Wu.t()) <= g_most
        if dtype == torch.float16:
            assert _ratio(db, dg.sum(0)) <= g_most
        else:
            assert float((db.cpu().double() - dg.sum(0)).norm() / dg.sum(0).norm()) <= R.roundoff(dtype) + 2 * 2.0 ** -11


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("act", ("none", "relu", "silu", "gelu"))
@pytest.mark.parametrize("fast", (False, True))
def test_same_result_with_a_gradient(xt, oracle_mod, dtype, act, fast):
    ls, _ = _pair(xt, oracle_mod, 1280, 384, 4, 3)
    for m in (1, 5, 16, 17, 40, 64, 65, 200, 300):
        x = _x(m, 1280, dtype, m)
        with torch.no_grad():
            want = xt.gated(x, *ls, act=act, fast=fast)
        assert torch.equal(xt.gated(x.requires_grad_(), *ls, act=act, fast=fast).detach(), want), m


@pytest.mark.parametrize("m", (3, 12, 40, 300))
def test_fast(xt, oracle_mod, m):
    """The caller's choice of 11 bits: two factors' roundings of 2^-11 beside float16's own (root of 3, and a tenth),
    nothing in bfloat16 without relu."""
    ls, (Wg, Wu) = _pair(xt, oracle_mod, 1280, 384, 4, 4)
    x = _x(m, 1280, torch.float16, m)
    xd = x.cpu().double()
    assert _ratio(xt.gated(x, *ls, act="none", fast=True), (xd @ Wg) * (xd @ Wu)) <= 1.1 * 3 ** 0.5
    b = _x(m, 1280, torch.bfloat16, m)
    assert torch.equal(xt.gated(b, *ls, fast=True), xt.gated(b, *ls))


def test_biases_alone(xt, oracle_mod):
    """Gradients of one bias, or both, without the rows'."""
    ls, (Wg, Wu) = _pair(xt, oracle_mod, 256, 384, 4, 4)
    for m in (3, 200):
        x, dy = _x(m, 256, torch.float16, m), _x(m, 384, torch.float16, 5)
        b = [torch.randn(384, device="cuda", requires_grad=True) for _ in range(2)]
        both = torch.autograd.grad(xt.gated(x, *ls, *b), b, dy)
        xx = x.clone().requires_grad_()
        assert all(torch.equal(s, t) for s, t in zip(both, torch.autograd.grad(xt.gated(xx, *ls, *b), [xx, *b], dy)[1:]))
        for i in range(2):
            one = [t if j == i else t.detach() for j, t in enumerate(b)]
            assert torch.equal(torch.autograd.grad(xt.gated(x, *ls, *one), one[i], dy)[0], both[i])


@pytest.mark.parametrize("m", (3, 70))
def test_magnitudes(xt, oracle_mod, m):
    """Rows of very different size, and of zeros."""
    k, n = 384, 256
    ls, (Wg, Wu) = _pair(xt, oracle_mod, k, n, 4, 4)
    for dtype, sizes in ((torch.bfloat16, (1e15, 0.0, 1e-15)), (torch.float16, (1e2, 0.0, 1e-1))):
        x = _x(m, k, torch.float32, 9, spread=0.0)
        x = (x / x.abs().max() * torch.tensor([sizes[i % 3] for i in range(m)]).cuda()[:, None]).to(dtype)
        xd = x.cpu().double()
        want = R.act(xd @ Wg, "relu") * (xd @ Wu)
        got = xt.gated(x, *ls, act="relu")
        err = (got.cpu().double() - want).norm(dim=1)
        floor = 2.0 ** -24 * n ** 0.5 if dtype == torch.float16 else 0.0        # (the smallest fp16 steps)
        assert bool((err <= _tol(dtype) * want.norm(dim=1) + floor).all())
        assert bool((got[1::3] == 0).all())


@pytest.mark.parametrize("m", (4, 30, 80))
def test_nonfinite_rows(xt, oracle_mod, m):
    """A NaN or an infinity stays in its row, forward and in dx."""
    ls, _ = _pair(xt, oracle_mod, 256, 256, 3, 4)
    x, dy = _x(m, 256, torch.bfloat16, 4).requires_grad_(), _x(m, 256, torch.bfloat16, 5)
    clean = xt.gated(x, *ls)
    cx, = torch.autograd.grad(clean, x, dy)
    bad = x.detach().clone()
    bad[1, 5] = float("nan")
    bad[3, 200] = float("inf")
    bad.requires_grad_()
    got = xt.gated(bad, *ls)
    bx, = torch.autograd.grad(got, bad, dy)
    keep = [i for i in range(m) if i not in (1, 3)]
    assert torch.equal(got[keep], clean[keep]) and torch.equal(bx[keep], cx[keep])
    assert not bool(got[1].isfinite().any()) and not bool(got[3].isfinite().all())
    worse = dy.clone()
    worse[2, 7] = float("nan")
    wx, = torch.autograd.grad(xt.gated(x, *ls), x, worse)
    keep = [i for i in range(m) if i != 2]
    assert torch.equal(wx[keep], cx[keep]) and not bool(wx[2].isfinite().any())


@pytest.mark.parametrize("m", (6, 100))
def test_layouts(xt, oracle_mod, m):
    """Leading dimensions, rows apart, odd addresses, transposed and expanded inputs, strided biases; no rows."""
    k, n = 256, 128
    ls, _ = _pair(xt, oracle_mod, k, n, 4, 5)
    x, dy = _x(m, k, torch.float16, 4), _x(m, n, torch.float16, 5)
    want = xt.gated(x, *ls)
    assert torch.equal(xt.gated(x.view(2, m // 2, k), *ls), want.view(2, m // 2, n))
    wide = torch.full((m, k + 3), 7.0, dtype=x.dtype, device="cuda")
    wide[:, 1:k + 1] = x
    assert torch.equal(xt.gated(wide[:, 1:k + 1], *ls), want)
    assert torch.equal(xt.gated(x.t().contiguous().t(), *ls), want)
    assert torch.equal(xt.gated(x[0], *ls), xt.gated(x[:1], *ls)[0])
    ex = x[:1].expand(m, k)
    assert torch.equal(xt.gated(ex, *ls), xt.gated(ex.contiguous(), *ls))
    b = torch.randn(2 * n, device="cuda")
    assert torch.equal(xt.gated(x, *ls, b[::2], b[1::2]), xt.gated(x, *ls, b[::2].contiguous(), b[1::2].contiguous()))
    leaf = x.clone().requires_grad_()
    far = torch.full((m, n + 5), float("nan"), dtype=dy.dtype, device="cuda")
    far[:, 3:n + 3] = dy
    grads = [torch.autograd.grad(xt.gated(leaf, *ls), leaf, d)[0]
             for d in (dy, far[:, 3:n + 3], dy.t().contiguous().t())]
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])
    e = x[:0].detach().requires_grad_()
    b = torch.zeros(n, device="cuda", requires_grad=True)
    y = xt.gated(e, *ls, up_bias=b)
    g = torch.autograd.grad(y.sum(), (e, b))
    assert y.shape == (0, n) and g[0].shape == (0, k) and bool((g[1] == 0).all())


@pytest.mark.parametrize("m,step", [(3, 2 ** 31), (70, 2 ** 26)])
def test_far_rows(xt, oracle_mod, m, step):
    """Rows whose offsets pass 2^32 elements give what the same rows give side by side, bit for bit."""
    k, n = 256, 384
    ls, _ = _pair(xt, oracle_mod, k, n, 4, 4)
    near, dnear = _x(m, k, torch.float16, 3), _x(m, n, torch.float16, 4)
    slots = torch.empty(70 * 2 ** 26, dtype=torch.float16, device="cuda")
    x, dy = slots.as_strided((m, k), (step, 1)), slots.as_strided((m, n), (step, 1), 2048)
    x.copy_(near)
    dy.copy_(dnear)
    out = []
    for a, d in ((x, dy), (near, dnear)):
        a.requires_grad_()
        y = xt.gated(a, *ls)
        out.append((y.detach(), torch.autograd.grad(y, a, d)[0]))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])


@pytest.mark.parametrize("m", (2, 20, 90, 300))
def test_repeats_streams_and_graphs(xt, oracle_mod, m):
    """The same bits on every call, on another stream, and in a replayed graph with eager work in between."""
    ls, _ = _pair(xt, oracle_mod, 1024, 384, 4, 5)
    xs = [_x(m, 1024, torch.bfloat16, s).requires_grad_() for s in (4, 5)]
    b = torch.randn(384, device="cuda", requires_grad=True)
    dy = _x(m, 384, torch.bfloat16, 6)

    def step(x):
        y = xt.gated(x, *ls, gate_bias=b)
        return [y.detach(), *torch.autograd.grad(y, (x, b), dy)]

    def equal(s, t):
        return all(torch.equal(p, q) for p, q in zip(s, t))

    want, want2 = step(xs[0]), step(xs[1])
    assert not equal(want, want2) and all(equal(step(xs[0]), want) for _ in range(4))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s = [step(xs[0]) for _ in range(3)]
    t = [step(xs[1]) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(equal(p, want) for p in s) and all(equal(p, want2) for p in t)
    buf = xs[0].detach().clone().requires_grad_()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step(buf)
        with torch.cuda.graph(graph, stream=side):
            got = step(buf)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        with torch.no_grad():
            buf.copy_(xs[i % 2])
        graph.replay()
        assert equal(step(xs[0]), want)
        torch.cuda.synchronize()
        assert equal(got, want2 if i % 2 else want)


def test_two_graphs(xt, oracle_mod):
    """Two captured calls that are replayed on two streams at once share no workspace and no counters."""
    ls, _ = _pair(xt, oracle_mod, 1024, 384, 4, 5)
    bufs = [_x(m, 1024, torch.bfloat16, m) for m in (2, 40)]
    want = [xt.gated(b, *ls) for b in bufs]
    graphs = [torch.cuda.CUDAGraph() for _ in bufs]
    got = []
    for g, b in zip(graphs, bufs):
        with torch.cuda.graph(g):
            got.append(xt.gated(b, *ls))
    streams = [torch.cuda.Stream() for _ in bufs]
    for _ in range(5):
        for t in got:
            t.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(20):
                    g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(xt, oracle_mod):
    (gate, up), _ = _pair(xt, oracle_mod, 256, 128, 4, 5)
    (other, _), _ = _pair(xt, oracle_mod, 128, 128, 4, 5)
    (mcg, _), _ = _pair(xt, oracle_mod, 256, 128, 4, 4, "exl3_mcg")
    x, b = _x(3, 256, torch.float16, 1), torch.zeros(128, device="cuda")
    for bad in (lambda: xt.gated(x.float(), gate, up), lambda: xt.gated(x.cpu(), gate, up),
                lambda: xt.gated(x[:, :128], gate, up), lambda: xt.gated(x, gate, other), lambda: xt.gated(x, gate, mcg),
                lambda: xt.gated(x, gate, up, act="tanh"), lambda: xt.gated(x, gate, up, b[:5]),
                lambda: xt.gated(x, gate, up, None, b.double()), lambda: xt.gated(x, gate, up, b.bfloat16()),
                lambda: xt.gated(x, gate, up, b.cpu())):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("name", ("x", "gate_bias", "up_bias"))
def test_derivatives_refused(xt, oracle_mod, name):
    """No forward mode, no second derivative."""
    import torch.autograd.forward_ad as fad
    ls, _ = _pair(xt, oracle_mod, 256, 128, 4, 5)
    v = {"x": _x(3, 256, torch.float16, 1), "gate_bias": torch.ones(128, device="cuda"),
         "up_bias": torch.ones(128, device="cuda")}
    with fad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        w = {**v, name: fad.make_dual(v[name], torch.ones_like(v[name]))}
        xt.gated(w["x"], *ls, w["gate_bias"], w["up_bias"])
    v[name].requires_grad_()
    y = xt.gated(v["x"], *ls, v["gate_bias"], v["up_bias"])
    g, = torch.autograd.grad(y, v[name], torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), v[name])


def test_block(xt, oracle_mod):
    """A gated block as it is used: norm, gate and up, down, the residual sum with the next norm; its gradients
    through frozen weights, in the operators' own roundings (each step's result is rounded once: 4 of them, doubled,
    and each factor's 11 bits)."""
    d, f, m = 256, 384, 33
    ls, (Wg, Wu) = _pair(xt, oracle_mod, d, f, 4, 5)
    w = R.random_weight(f, d, 4, 30)
    down, Wd = xt.TrellisLinear(*w, 4), R.dense(oracle_mod, *w, 4, "exl3_mul1")
    dtype = torch.bfloat16
    x = _x(m, d, dtype, 2).requires_grad_()
    wn, wp, s = ((1 + 0.2 * torch.randn(d, device="cuda")).requires_grad_() for _ in range(3))
    h = xt.norm(x, wn)
    y, n = xt.residual_norm(xt.linear(xt.gated(h, *ls), down), x, kind="layer", post="rms", post_weight=wp, scale=s)
    dy, dn = _x(m, d, dtype, 3, spread=0.1), _x(m, d, dtype, 4, spread=0.1)
    got = torch.autograd.grad((y, n), (x, wn, wp, s), (dy, dn))
    leaves = [t.detach().cpu().double().requires_grad_() for t in (x, wn, wp, s)]
    xd, wnd, wpd, sd = leaves

    def rms(t):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6)

    hd = rms(xd) * wnd
    zg = hd @ Wg
    b = (zg / (1 + torch.exp(-zg)) * (hd @ Wu)) @ Wd
    yd = xd + sd * rms(b) * wpd
    c = yd - yd.mean(-1, keepdim=True)
    nd = rms(c)
    want = torch.autograd.grad((yd, nd), leaves, (dy.cpu().double(), dn.cpu().double()))
    tol = 8 * R.roundoff(dtype) + 16 * 2.0 ** -11
    for g, v in zip((y, n, *got), (yd.detach(), nd.detach(), *want)):
        assert float((g.detach().cpu().double() - v).norm() / v.norm()) <= tol
