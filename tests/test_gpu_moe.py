"""The mixture layer on trellis experts (trellis_ops.moe) against its definition in 64 bits.

Tolerances.  Activations enter both products with 22 bits (two fp16 terms), sums are fp32 and the result is
rounded once: a row's error is the result's roundoff u, and 2e-5 for the rest (2^-22 for the terms, 2^-24 times
the root of the at most 1,152 summed products, three products in a row).  Routing weights are fp32 softmaxes of
logits that are off by about 2^-24 of their row's norm: 1e-5."""
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


def _tol(dtype):
    return R.roundoff(dtype) + 2e-5


class Layer:
    """Random experts, Ks[e] = (gate, up, down), and their dense weights."""

    def __init__(self, xt, O, d, f, Ks, seed, code="exl3_mul1", scale=1.0):
        make = lambda k, n, K, s: R.random_weight(k, n, K, s)  # noqa: E731
        parts = [(make(d, f, kg, seed + 3 * e), make(d, f, ku, seed + 3 * e + 1), make(f, d, kd, seed + 3 * e + 2))
                 for e, (kg, ku, kd) in enumerate(Ks)]
        self.dense = [[R.dense(O, *w, K, code, scale) for w, K in zip(p, ks)] for p, ks in zip(parts, Ks)]
        lin = [[xt.TrellisLinear(*w, K, code=code, scale=scale) for w, K in zip(p, ks)] for p, ks in zip(parts, Ks)]
        self.experts = xt.TrellisExperts(*zip(*lin))
        self.d, self.n = d, len(Ks)

    def want(self, x, router, top, act, renorm, residual, valid):
        x, router = x.cpu().double(), router.cpu().double()
        logits = x @ router.t()
        p = torch.softmax(logits, 1)
        ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top]
        w = torch.gather(p, 1, ids)
        if renorm:
            w = w / w.sum(1, keepdim=True)
        y = torch.zeros(x.shape[0], self.d, dtype=torch.float64)
        if valid is not None:
            ids[~valid.cpu()] = -1
            w[~valid.cpu()] = 0
        for t in range(x.shape[0]):
            for e, we in zip(ids[t].tolist(), w[t]):
                if e >= 0:
                    g, u, dn = self.dense[e]
                    y[t] += we * ((R.act(x[t] @ g, act) * (x[t] @ u)) @ dn)
        if residual is not None:
            y = y + residual.cpu().double()
        return y, ids, w


def _x(m, k, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g)
    x[:, ::96] *= 10.0
    return (x * torch.exp(torch.randn(m, 1, generator=g) * 0.5)).to(dtype).cuda()


def _router(n, d, dtype, seed):
    return (torch.randn(n, d, generator=torch.Generator().manual_seed(seed)) / d ** 0.5).to(dtype).cuda()


def _check(layer, xt, x, router, top, act="silu", renorm=True, residual=None, valid=None):
    y, ids, w = xt.moe(x, router, layer.experts, top, act=act, renorm=renorm, residual=residual, valid=valid,
                       return_routing=True)
    wy, wi, ww = layer.want(x, router, top, act, renorm, residual, valid)
    assert torch.equal(ids.cpu().long(), wi)
    assert ids.dtype == torch.int32 and y.dtype == x.dtype
    assert float((w.cpu().double() - ww).abs().max()) <= 1e-5
    assert float(R.row_errors(y, wy).max()) <= _tol(x.dtype)
    return y


@pytest.mark.parametrize("rows", (1, 2, 4, 5, 8, 9, 16, 17, 33, 64))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_moe_rows(xt, oracle_mod, rows, dtype):
    """Row counts around the launches' and the lists' groups; more slots than experts and fewer."""
    layer = Layer(xt, oracle_mod, 256, 384, [(4, 4, 4)] * 6, 100)
    x, router = _x(rows, 256, dtype, rows), _router(6, 256, dtype, 1)
    _check(layer, xt, x, router, 2, residual=_x(rows, 256, dtype, 7) if rows % 2 else None)


@pytest.mark.parametrize("code", sorted(R.CODES))
@pytest.mark.parametrize("rows", (3, 20))
def test_moe_mixed_widths(xt, oracle_mod, code, rows):
    """Every width, different in each expert and weight; every codebook; a scale of the weights."""
    Ks = [(2 + e % 6, 2 + (e + 1) % 6, 2 + (e + 3) % 6) for e in range(6)]
    layer = Layer(xt, oracle_mod, 384, 128, Ks, 200, code=code, scale=0.75)
    x, router = _x(rows, 384, torch.float16, rows), _router(6, 384, torch.float32, 2)
    _check(layer, xt, x, router, 6, renorm=False, act="gelu")


@pytest.mark.parametrize("experts,top", [(1, 1), (3, 3), (64, 8), (65, 1), (130, 16), (512, 4)])
def test_moe_experts(xt, oracle_mod, experts, top):
    """Numbers of experts around the router's registers."""
    layer = Layer(xt, oracle_mod, 128, 128, [(3, 3, 3)] * min(experts, 5), 300)
    few = layer.n
    if experts > few:       # the same weights again under other numbers
        idx = [e % few for e in range(experts)]
        ws = layer.experts.weights
        layer.experts = xt.TrellisExperts(*([ws[3 * i + r] for i in idx] for r in range(3)))
        layer.dense = [layer.dense[i] for i in idx]
    x, router = _x(7, 128, torch.bfloat16, 3), _router(experts, 128, torch.bfloat16, 4)
    for act in ("silu", "relu", "none"):
        _check(layer, xt, x, router, top, act=act, renorm=act != "relu")


@pytest.mark.parametrize("rows,k,f,experts,top", [(1, 1152, 640, 9, 8), (2, 640, 1152, 5, 1), (40, 1024, 256, 3, 2)])
def test_moe_sizes(xt, oracle_mod, rows, k, f, experts, top):
    """Summed dimensions split over several workgroups; one expert with more than 16 rows."""
    layer = Layer(xt, oracle_mod, k, f, [(4, 5, 3)] * experts, 400)
    x, router = _x(rows, k, torch.float16, 5), _router(experts, k, torch.float16, 6)
    if rows == 40:
        router[1] += x.float().mean(0).half() * 4      # most rows choose expert 1
    _check(layer, xt, x, router, top)


@pytest.mark.parametrize("rows", (1, 3, 30))
def test_moe_masks(xt, oracle_mod, rows):
    """Rows left out hold NaN; all rows left out; ties; NaN and infinities stay in their rows."""
    layer = Layer(xt, oracle_mod, 256, 128, [(4, 4, 4)] * 5, 500)
    x, router = _x(rows, 256, torch.bfloat16, 8), _router(5, 256, torch.bfloat16, 9)
    res = _x(rows, 256, torch.bfloat16, 10)
    valid = (torch.arange(rows) % 3 != 1).cuda()
    clean = _check(layer, xt, x, router, 2, residual=res, valid=valid)
    hidden = x.clone()
    hidden[~valid] = float("nan")
    got, ids, w = xt.moe(hidden, router, layer.experts, 2, residual=res, valid=valid, return_routing=True)
    assert torch.equal(got, clean) and torch.equal(got[~valid], res[~valid])
    assert bool((ids[~valid] == -1).all()) and bool((w[~valid] == 0).all())
    none = torch.zeros(rows, dtype=torch.bool, device="cuda")
    assert torch.equal(xt.moe(hidden, router, layer.experts, 2, residual=res, valid=none), res)
    assert bool((xt.moe(hidden, router, layer.experts, 2, valid=none) == 0).all())
    assert torch.equal(xt.moe(hidden, router, layer.experts, 2, residual=res, valid=valid), clean)   # and again
    # equal logits: the lowest experts, for zeros of either sign too
    flat = router.clone()
    flat[3], flat[1] = flat[0], flat[0]
    _check(layer, xt, x, flat, 3)
    _, ids, _ = xt.moe(torch.zeros_like(x), router, layer.experts, 2, return_routing=True)
    assert torch.equal(ids.cpu(), torch.tensor([[0, 1]] * rows, dtype=torch.int32))
    if rows > 1:
        bad = x.clone()
        bad[1, 7] = float("nan")
        y = xt.moe(bad, router, layer.experts, 2)
        want = xt.moe(x, router, layer.experts, 2)
        keep = [i for i in range(rows) if i != 1]
        assert torch.equal(y[keep], want[keep]) and bool(torch.isnan(y[1]).all())


def test_moe_layouts_and_repeats(xt, oracle_mod):
    """More than 64 tokens, leading dimensions, rows apart, other streams, replayed graphs."""
    layer = Layer(xt, oracle_mod, 256, 256, [(4, 4, 4)] * 8, 600)
    x, router = _x(130, 256, torch.float16, 11), _router(8, 256, torch.float16, 12)
    want = _check(layer, xt, x, router, 2)
    assert torch.equal(xt.moe(x.view(2, 65, 256), router, layer.experts, 2), want.view(2, 65, 256))
    wide = torch.full((130, 261), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, 3:259] = x
    assert torch.equal(xt.moe(wide[:, 3:259], router, layer.experts, 2), want)
    assert xt.moe(x[:0], router, layer.experts, 2).shape == (0, 256)
    for rows in (2, 20):
        a, b = x[:rows].clone(), x[40:40 + rows].clone()
        wa, wb = (xt.moe(t, router, layer.experts, 2) for t in (a, b))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ga = [xt.moe(a, router, layer.experts, 2) for _ in range(3)]
        gb = [xt.moe(b, router, layer.experts, 2) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(t, wa) for t in ga) and all(torch.equal(t, wb) for t in gb)
        buf = a.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = xt.moe(buf, router, layer.experts, 2)
        for i in range(4):
            buf.copy_(b if i % 2 else a)
            graph.replay()
            assert torch.equal(xt.moe(a, router, layer.experts, 2), wa)
            torch.cuda.synchronize()
            assert torch.equal(y, wb if i % 2 else wa)


def test_moe_refusals(xt):
    w = lambda k, n, code="exl3_mul1": xt.TrellisLinear(*R.random_weight(k, n, 4, 1), 4, code=code)  # noqa: E731
    g, u, dn = w(256, 128), w(256, 128), w(128, 256)
    e = xt.TrellisExperts([g, g], [u, u], [dn, dn])
    x, router = _x(3, 256, torch.float16, 1), _router(2, 256, torch.float16, 2)
    valid = torch.ones(3, dtype=torch.bool, device="cuda")
    for bad in (lambda: xt.TrellisExperts([], [], []), lambda: xt.TrellisExperts([g], [u, u], [dn]),
                lambda: xt.TrellisExperts([g], [dn], [dn]), lambda: xt.TrellisExperts([g], [u], [g]),
                lambda: xt.TrellisExperts([g], [w(256, 128, "exl3_mcg")], [dn]),
                lambda: xt.moe(x.float(), router, e, 1), lambda: xt.moe(x[:, :128], router, e, 1),
                lambda: xt.moe(x, router[:1], e, 1), lambda: xt.moe(x, router.bfloat16(), e, 1),
                lambda: xt.moe(x, router, e, 0), lambda: xt.moe(x, router, e, 3),
                lambda: xt.moe(x, router, e, 1, act="tanh"), lambda: xt.moe(x, router, e, 1, residual=x[:2]),
                lambda: xt.moe(x, router, e, 1, valid=valid[:2]), lambda: xt.moe(x, router, e, 1, valid=valid.int()),
                lambda: xt.moe(x.cpu(), router, e, 1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        xt.moe(x.requires_grad_(), router, e, 1)
