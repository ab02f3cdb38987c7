"""Norms of rows and the residual sum between blocks (trellis_ops.norm, residual_norm) and their gradients, against
the definitions in 64 bits, differentiated there by torch.

Tolerances.  A result is rounded once, by u = roundoff(type) of itself at most; what comes before is fp32 with sums of
up to 32768 values, whose error (2^-24 times the root of their number, 1.1e-5) and that of the vector unit's
exponential and reciprocal (3e-7) stay below 2e-5 of the row's norm.  So a row is held to u + 2e-5 of its norm, a
gradient of an input to u + 4e-5 of its own (its projections are taken off one of 64 directions at least), and an fp32 gradient of a parameter to 4e-5 of its terms' norm, root of the sum of squares over the rows and
channels: a sum over rows adds the rows' own errors, and its chain of additions 2^-24 of the sum each."""
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


def _rows(m, d, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, d, generator=g)
    x[:, ::96] *= 15.0
    return (x * torch.exp(torch.randn(m, 1, generator=g) * spread)).to(dtype).cuda()


def _param(d, dtype, seed, mean):
    return (mean + 0.3 * torch.randn(d, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


def _normed(t, kind, w, b, eps):
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)
    t = t if w is None else t * w
    return t if b is None else t + b


def _gate(g, act):
    return g if act == "none" else torch.sigmoid(g) * (g if act == "silu" else 1.0)


def _want(v, kind, post, act, number, eps, post_eps):
    """(y, h) in 64 bits of a dict of 64-bit tensors."""
    t = v["block"]
    if post:
        t = _normed(t, post, v.get("post_weight"), v.get("post_bias"), post_eps)
    if "gate" in v:
        t = t * _gate(v["gate"], act)
    y = v["residual"] + t * v.get("scale", number)
    return y, _normed(y, kind, v.get("weight"), v.get("bias"), eps) if kind else None


def _off(got, want, terms=None):
    """Largest row's error over its norm, or over that of `terms` where that is larger."""
    got, want = got.detach().cpu().double(), want.detach().cpu().double()
    assert got.shape == want.shape
    norm = want.norm(dim=-1)
    if terms is not None:
        norm = torch.maximum(norm, terms.detach().cpu().double())
    off = (got - want).norm(dim=-1)
    return float(torch.where(off > 0, off / norm.clamp(min=1e-300), off).max())


WIDTHS = (1, 7, 8, 9, 16, 100, 127, 128, 129, 200, 256, 257, 512, 513, 1000, 1024, 1025, 2047, 5120, 8192, 8193, 16385, 32768)


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("kind", ("rms", "layer"))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_norm(xt, d, kind, dtype):
    """Widths around every number of lanes and eights, odd ones among them; parameters in both types or none."""
    for m, pt in ((1, dtype), (17, torch.float32), (5, None)):
        x = _rows(m, d, dtype, m + d)
        w, b = (None, None) if pt is None else (_param(d, pt, 1, 1.0), _param(d, pt, 2, 0.0))
        h = xt.norm(x, w, b, kind=kind, eps=1e-5)
        assert h.dtype == dtype and h.shape == x.shape
        want = _normed(x.double(), kind, None if w is None else w.double(), None if b is None else b.double(), 1e-5)
        # ("layer" of one channel is 0 before the bias)
        assert _off(h, want) <= R.roundoff(dtype) + 2e-5


CASES = [("rms", "rms", "sigmoid", "tensor"), ("layer", "layer", "silu", "tensor"), ("rms", None, "none", 0.3),
         (None, "rms", None, None), ("layer", "rms", None, "tensor"), ("rms", None, None, None),
         (None, None, "sigmoid", "tensor"), (None, "layer", "none", 2.0)]


def _inputs(m, d, dtype, pt, kind, post, act, scale, bias):
    v = {"block": _rows(m, d, dtype, 1), "residual": _rows(m, d, dtype, 2)}
    if act:
        v["gate"] = _rows(m, d, dtype, 3, spread=0.2)
    if scale == "tensor":
        v["scale"] = _param(d, pt, 4, 0.5)
    for there, name, seed in ((kind, "weight", 5), (post, "post_weight", 6)):
        if there:
            v[name] = _param(d, pt, seed, 1.0)
            if bias:
                v[name.replace("weight", "bias")] = _param(d, pt, seed + 4, 0.0)
    return v


def _call(xt, v, kind, post, act, scale, eps=1e-6, post_eps=1e-5):
    v = dict(v)
    if scale != "tensor":
        v["scale"] = scale
    return xt.residual_norm(v.pop("block"), v.pop("residual"), kind=kind, post=post, gate_act=act or "none", eps=eps,
                            post_eps=post_eps, **v)


@pytest.mark.parametrize("kind,post,act,scale", CASES)
@pytest.mark.parametrize("m,d", [(1, 5120), (3, 127), (130, 1000), (33, 2049), (2, 20000)])
@pytest.mark.parametrize("dtype,pt", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
def test_residual_norm(xt, kind, post, act, scale, m, d, dtype, pt):
    v = _inputs(m, d, dtype, pt, kind, post, act, scale, bias=m % 2 == 1)
    y, h = _call(xt, v, kind, post, act, scale)
    number = 1.0 if scale in (None, "tensor") else scale
    wy, wh = _want({n: t.double() for n, t in v.items()}, kind, post, act or "none", number, 1e-6, 1e-5)
    # y is a sum: beside its own rounding the terms' fp32 errors
    assert _off(y, wy, 1e-2 * (wy - v["residual"].double()).norm(dim=-1)) <= R.roundoff(dtype) + 2e-5
    if kind is None:
        assert h is None
    else:
        assert _off(h, wh) <= R.roundoff(dtype) + 2e-5


def test_means_of_ragged_rows(xt):
    """A centred norm after a centred norm with a bias: what lies past a row's end is none of its mean."""
    for d in (9, 127, 130, 513, 1030, 2049, 6150, 13000):
        x = (5.0 + _rows(3, d, torch.float32, d, spread=0.0)).to(torch.float16)
        r = _rows(3, d, torch.float16, 2, spread=0.0)
        pw, pb = _param(d, torch.float32, 3, 1.0), _param(d, torch.float32, 4, 2.0)
        y, h = xt.residual_norm(x, r, kind="layer", post="layer", post_weight=pw, post_bias=pb)
        wy = r.double() + _normed(x.double(), "layer", pw.double(), pb.double(), 1e-6)
        assert _off(y, wy) <= R.roundoff(torch.float16) + 2e-5
        assert _off(h, _normed(wy, "layer", None, None, 1e-6)) <= R.roundoff(torch.float16) + 2e-5


def _gradients(v, douts, kind, post, act, number, eps, post_eps):
    """Gradients in 64 bits."""
    leaves = {n: t.detach().double().requires_grad_() for n, t in v.items()}
    outs = [o for o in _want(leaves, kind, post, act, number, eps, post_eps) if o is not None]
    return dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), [g.double() for g in douts])))


@pytest.mark.parametrize("kind,post,act,scale", CASES)
@pytest.mark.parametrize("m,d", [(1, 128), (5, 5120), (70, 100), (600, 96), (300, 250), (37, 700), (19, 1024), (530, 2049),
                                 (3, 9000), (4, 17408)])
def test_residual_norm_gradient(xt, kind, post, act, scale, m, d):
    """Every tensor's gradient."""
    dtype, pt = (torch.bfloat16, torch.float32) if m % 2 else (torch.float16, torch.float32)
    v = _inputs(m, d, dtype, pt, kind, post, act, scale, bias=True)
    for t in v.values():
        t.requires_grad_()
    outs = [o for o in _call(xt, v, kind, post, act, scale) if o is not None]
    douts = [_rows(m, d, dtype, 20 + i, spread=0.3) for i in range(len(outs))]
    got = dict(zip(v, torch.autograd.grad(outs, list(v.values()), douts)))
    number = 1.0 if scale in (None, "tensor") else scale
    want = _gradients(v, douts, kind, post, act or "none", number, 1e-6, 1e-5)
    u = R.roundoff(dtype)
    for name, g in got.items():
        assert g.dtype == v[name].dtype and g.shape == v[name].shape
        if name in ("block", "residual", "gate"):
            assert _off(g, want[name]) <= u + 4e-5, name
        else:
            terms = want["residual"].norm() if name in ("scale", "post_weight", "post_bias") else douts[-1].double().norm()
            big = max(float(want[name].norm()), float(terms))
            off = float((g.double() - want[name].cuda()).norm())
            assert off <= 4e-5 * big, name


@pytest.mark.parametrize("kind", ("rms", "layer"))
@pytest.mark.parametrize("m,d", [(6, 64), (9, 600), (4, 1500)])
def test_gradient_against_differences(xt, kind, m, d):
    """Every gradient's product with a direction against a difference of the definition in 64 bits (step 1e-6: its
    error is 1e-10 of the function's size).  The gradients are rounded, independently: sqrt(count) roundings."""
    dtype = torch.float16
    v = _inputs(m, d, dtype, torch.float32, kind, "rms", "silu", "tensor", bias=True)
    for t in v.values():
        t.requires_grad_()
    outs = _call(xt, v, kind, "rms", "silu", "tensor")
    douts = [_rows(m, d, dtype, 30 + i, spread=0.2) for i in range(2)]
    got = dict(zip(v, torch.autograd.grad(outs, list(v.values()), douts)))
    base = {n: t.detach().cpu().double() for n, t in v.items()}

    def f(at):
        return float(sum((o * g.cpu().double()).sum() for o, g in zip(_want(at, kind, "rms", "silu", 1.0, 1e-6, 1e-5), douts)))

    for name, t in base.items():
        u = torch.randn(t.shape, generator=torch.Generator().manual_seed(40)).double()
        dif = (f({**base, name: t + 1e-6 * u}) - f({**base, name: t - 1e-6 * u})) / 2e-6
        g = got[name].cpu().double()
        assert abs(float((g * u).sum()) - dif) <= 4 * R.roundoff(dtype) * float((g * u).norm()) + 1e-5 * float(g.norm()) + 1e-4, name


@pytest.mark.parametrize("which", ("y", "h"))
def test_gradient_of_one_result(xt, which):
    """One of the two results unused: its gradient counts as zero.  Frozen parameters get none."""
    m, d = 40, 600
    v = _inputs(m, d, torch.float16, torch.float32, "rms", "rms", "sigmoid", "tensor", bias=False)
    want_of = ("block", "residual", "gate")
    for n in want_of:
        v[n].requires_grad_()
    out = _call(xt, v, "rms", "rms", "sigmoid", "tensor")[which == "h"]
    dout = _rows(m, d, torch.float16, 9, spread=0.2)
    got = torch.autograd.grad(out, [v[n] for n in want_of], dout)
    douts = [dout, torch.zeros_like(dout)] if which == "y" else [torch.zeros_like(dout), dout]
    want = _gradients(v, douts, "rms", "rms", "sigmoid", 1.0, 1e-6, 1e-5)
    for n, g in zip(want_of, got):
        assert _off(g, want[n]) <= R.roundoff(torch.float16) + 4e-5
    assert all(v[n].grad is None and not v[n].requires_grad for n in ("weight", "scale", "post_weight"))


def test_same_result_with_a_gradient_and_in_any_batch(xt):
    for d in (100, 700, 5120, 20000):
        v = _inputs(50, d, torch.bfloat16, torch.float32, "layer", "rms", "silu", "tensor", bias=True)
        y, h = _call(xt, v, "layer", "rms", "silu", "tensor")
        one = {n: t[7:8] if t.dim() == 2 else t for n, t in v.items()}
        y1, h1 = _call(xt, one, "layer", "rms", "silu", "tensor")
        assert torch.equal(y[7:8], y1) and torch.equal(h[7:8], h1)
        v["weight"].requires_grad_()
        y2, h2 = _call(xt, v, "layer", "rms", "silu", "tensor")
        assert torch.equal(y, y2) and torch.equal(h, h2)


def test_layouts(xt):
    """Rows apart, odd addresses, transposed and expanded rows, leading dimensions, no rows, sliced parameters."""
    m, d = 24, 200
    v = _inputs(m, d, torch.float16, torch.float32, "rms", "layer", "none", "tensor", bias=True)
    y, h = _call(xt, v, "rms", "layer", "none", "tensor")
    wide = {}
    for n, t in v.items():
        big = torch.full((*t.shape[:-1], d + 13), float("nan"), dtype=t.dtype, device="cuda")
        big[..., 5:d + 5] = t
        wide[n] = big[..., 5:d + 5]
    wide["weight"] = v["weight"].repeat_interleave(2)[::2]
    for w in (wide, {n: t.t().contiguous().t() if t.dim() == 2 else t for n, t in v.items()}):
        yw, hw = _call(xt, w, "rms", "layer", "none", "tensor")
        assert torch.equal(y, yw) and torch.equal(h, hw)
    lead = {n: t.view(2, 3, 4, d) if t.dim() == 2 else t for n, t in v.items()}
    yl, hl = _call(xt, lead, "rms", "layer", "none", "tensor")
    assert yl.shape == (2, 3, 4, d) and torch.equal(yl.view(m, d), y) and torch.equal(hl.view(m, d), h)
    # a gate shared by all rows
    gate = v["gate"][:1].clone().requires_grad_()
    ge = {**v, "gate": gate.expand(m, d)}
    gf = {**v, "gate": gate.detach().expand(m, d).contiguous().requires_grad_()}
    a, b = _call(xt, ge, "rms", "layer", "none", "tensor"), _call(xt, gf, "rms", "layer", "none", "tensor")
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ga, = torch.autograd.grad(a, gate, (y, h))
    gb, = torch.autograd.grad(b, gf["gate"], (y, h))
    assert torch.equal(ga, gb.sum(0, keepdim=True))
    # no rows
    none = {n: t[:0].detach().requires_grad_() if t.dim() == 2 else t.detach().requires_grad_() for n, t in v.items()}
    out = _call(xt, none, "rms", "layer", "none", "tensor")
    assert out[0].shape == (0, d) and out[1].shape == (0, d)
    grads = torch.autograd.grad([o.sum() for o in out], list(none.values()))
    assert all(g.shape == t.shape and not g.any() for g, t in zip(grads, none.values()))
    assert xt.norm(v["block"][0], v["weight"]).shape == (d,)


def test_magnitudes(xt):
    """Rows of zeros, near the types' ends, and channels that cancel around a large mean."""
    d = 300
    for dtype, sizes in ((torch.bfloat16, (1e15, 1e-15, 0.0)), (torch.float16, (3e4, 1e-3, 0.0))):
        x = _rows(6, d, torch.float32, 3, spread=0.0)
        x = (x / x.abs().max() * torch.tensor([sizes[i % 3] for i in range(6)]).cuda()[:, None]).to(dtype)
        h = xt.norm(x, eps=1e-12)
        want = _normed(x.double(), "rms", None, None, 1e-12)
        floor = 2.0 ** -25 * d ** 0.5 if dtype == torch.float16 else 0.0     # (float16's smallest steps)
        err = (h.double() - want).norm(dim=-1)
        assert bool((err <= (R.roundoff(dtype) + 2e-5) * want.norm(dim=-1) + floor).all())
        assert not h[2::3].any()
    x = (1000.0 + _rows(5, d, torch.float32, 4, spread=0.0)).to(torch.float16)
    want = _normed(x.double(), "layer", None, None, 1e-6)
    # the mean's fp32 error, 2^-23 of 1000, beside deviations of 3
    assert _off(xt.norm(x, kind="layer"), want) <= R.roundoff(torch.float16) + 2e-5 + 1000 * 2.0 ** -22


def test_nonfinite_rows(xt):
    """A NaN or an infinity stays in its row; parameters' gradients hold it."""
    m, d = 40, 100
    for dd in (d, 700, 1500):
        x = _rows(m, dd, torch.bfloat16, 4)
        clean = xt.norm(x)
        bad = x.clone()
        bad[1, 5] = float("nan")
        bad[3, 90] = float("inf")
        h = xt.norm(bad)
        keep = [i for i in range(m) if i not in (1, 3)]
        assert torch.equal(h[keep], clean[keep])
        assert bool(h[1].isnan().all()) and bool(h[3, 90].isnan())
        w = torch.ones(dd, device="cuda", requires_grad=True)
        bad.requires_grad_()
        dx, dw = torch.autograd.grad(xt.norm(bad, w), (bad, w), x)
        assert bool(dx[keep].isfinite().all()) and bool(dw[90].isnan())


def test_far_rows(xt):
    """Rows whose offsets pass 2^32 elements."""
    m, d, step = 3, 384, 2 ** 31
    near = [_rows(m, d, torch.float16, s) for s in range(3)]
    slots = torch.empty(m * step, dtype=torch.float16, device="cuda")
    far = [slots.as_strided((m, d), (step, 1), 1000 * i) for i in range(3)]
    for f, n in zip(far, near):
        f.copy_(n)
    for a, b in zip(xt.residual_norm(*far[:2], gate=far[2]), xt.residual_norm(*near[:2], gate=near[2])):
        assert torch.equal(a, b)
    grads = []
    for t in (far, near):
        leaves = [v.detach().requires_grad_() for v in t]
        grads.append(torch.autograd.grad(xt.residual_norm(*leaves[:2], gate=leaves[2]), leaves, (t[2], t[1])))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.parametrize("m,d", [(3, 100), (300, 1500)])
def test_repeats_streams_and_graphs(xt, m, d):
    """The same bits on every call, on another stream and in a replayed graph, forward and backward."""
    args = ("layer", "rms", "silu", "tensor")
    v, v2 = ({n: t.clone().requires_grad_() for n, t in _inputs(m, d, torch.bfloat16, torch.float32, *args, bias=True).items()}
             for _ in range(2))
    with torch.no_grad():
        for t in (v2["block"], v2["residual"]):
            t.mul_(0.5)
    dy, dh = _rows(m, d, torch.bfloat16, 50), _rows(m, d, torch.bfloat16, 51)

    def step(s):
        outs = _call(xt, s, *args)
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, list(s.values()), (dy, dh)))

    def equal(a, b):
        return all(torch.equal(s, t) for s, t in zip(a, b))

    want, want2 = step(v), step(v2)
    assert not equal(want, want2) and all(equal(step(v), want) for _ in range(4))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = step(v)
    b = step(v2)
    torch.cuda.synchronize()
    assert equal(a, want) and equal(b, want2)
    buf = {n: t.detach().clone().requires_grad_() for n, t in v.items()}
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step(buf)
        with torch.cuda.graph(graph, stream=side):
            got = step(buf)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        with torch.no_grad():
            for n, t in buf.items():
                t.copy_((v2 if i % 2 else v)[n])
        graph.replay()
        assert equal(step(v), want)
        torch.cuda.synchronize()
        assert equal(got, want2 if i % 2 else want)


def test_refusals(xt):
    x, w = _rows(3, 256, torch.float16, 1), torch.ones(256, device="cuda")
    for bad in (lambda: xt.norm(x.float()), lambda: xt.norm(x.cpu()), lambda: xt.norm(x, w[:5]),
                lambda: xt.norm(x, w.double()), lambda: xt.norm(x, w.bfloat16()), lambda: xt.norm(x, kind="batch"),
                lambda: xt.norm(x, kind=None), lambda: xt.norm(x, eps=-1.0), lambda: xt.norm(x, eps=float("nan")),
                lambda: xt.norm(x[:, :0]), lambda: xt.norm(torch.zeros(1, 32769, dtype=x.dtype, device="cuda")),
                lambda: xt.residual_norm(x, None), lambda: xt.residual_norm(x, x[:2]),
                lambda: xt.residual_norm(x, x.bfloat16()), lambda: xt.residual_norm(x, x, gate=x[:1]),
                lambda: xt.residual_norm(x, x, gate=x, gate_act="tanh"), lambda: xt.residual_norm(x, x, post="batch"),
                lambda: xt.residual_norm(x, x, w, kind=None), lambda: xt.residual_norm(x, x, post_weight=w),
                lambda: xt.residual_norm(x, x, scale=w[:3]), lambda: xt.residual_norm(x, x, scale=w[:1])):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("name", ("block", "residual", "gate", "scale", "weight", "post_weight", "bias", "post_bias"))
def test_derivatives_refused(xt, name):
    """No forward mode, no second derivative."""
    import torch.autograd.forward_ad as fad
    args = ("layer", "rms", "silu", "tensor")
    v = _inputs(3, 64, torch.float16, torch.float32, *args, bias=True)
    with fad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        _call(xt, {**v, name: fad.make_dual(v[name], torch.ones_like(v[name]))}, *args)
    v[name].requires_grad_()
    y, h = _call(xt, v, *args)
    g, = torch.autograd.grad((y, h), v[name], (torch.ones_like(y), torch.ones_like(h)), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), v[name])


def test_more_rows_than_a_grid_holds(xt):
    """Each row has the bits it has alone, whatever rows there are: 2^28 of them are more lanes than one launch."""
    m, d = (1 << 28) + 37, 8
    x = torch.empty(m, d, dtype=torch.float16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(3))
    x.requires_grad_()
    w = torch.linspace(-1.0, 2.0, d, device="cuda")
    h = xt.norm(x, w)
    dx, = torch.autograd.grad(h, x, x.detach())
    for at in (0, (1 << 26) - 50, (1 << 27) - 50, m - 100):
        part = x.detach()[at:at + 100].clone().requires_grad_()
        alone = xt.norm(part, w)
        assert torch.equal(h[at:at + 100], alone)
        assert torch.equal(dx[at:at + 100], torch.autograd.grad(alone, part, part.detach())[0])


@pytest.mark.parametrize("d", (100, 120, 250, 7000, 7001))
def test_an_infinite_scale_stays_infinite(xt, d):
    """dp = dy s w' is infinite in the first channel alone, and so is its mean with x^, so that dx elsewhere is
    infinite too, with the sign of -x^ dp x^[first]: nothing past the row's end makes NaN of it."""
    g = torch.Generator("cuda").manual_seed(5)
    x, dy, res = (torch.randn(5, d, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    scale = torch.ones(d, device="cuda")
    scale[0] = float("inf")
    x.requires_grad_()
    y, _ = xt.residual_norm(x, res, kind=None, post="rms", scale=scale)
    dx, = torch.autograd.grad(y, x, dy)
    want = -torch.sign(x.detach() * dy[:, :1] * x.detach()[:, :1])[:, 1:] * float("inf")
    assert torch.equal(dx[:, 1:], want)


@pytest.mark.parametrize("d", (100, 200, 400, 1000, 7000))
def test_a_row_of_infinite_factor(xt, d):
    """The squares of a first row of 1e-30 are zero and its factor infinite (eps 0): the weight's gradient is too,
    and places of a workgroup without a row add no NaN to it."""
    x = torch.ones(3, d, device="cuda", dtype=torch.bfloat16)
    x[0] = 1e-30
    w = torch.ones(d, device="cuda", requires_grad=True)
    dw, = torch.autograd.grad(xt.norm(x, w, eps=0.0), w, torch.ones_like(x))
    assert torch.equal(dw, torch.full_like(dw, float("inf")))
