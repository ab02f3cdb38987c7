"""Gradients of norms and residual sums in every form that is launched apart: plain norms, with and without means and
biases, every number of lanes a row has, more rows than the lanes have at a time, rows wider than the registers; against
the definitions in 64 bits, differentiated there by torch.

Tolerances.  A result is rounded once, by u = roundoff(type) of itself at most.  Before that everything is fp32, with
sums of up to 32768 values of a row, whose chain of additions is off by 2^-24 times the root of their number (1.1e-5),
twice over where a gradient takes two sums: 4e-5 of what is added up.  That is, for an input's gradient, the row before
the projections that take parts of it away (`before` below), and for a parameter's the terms of its sum over the rows,
root of the sum of their squares, where the rows' chain adds 2^-24 of the sum an addition, of which the launches make
at most 130 one behind the other (a group's rows, its workgroup's groups, every 16th part, 16 of those), 8e-6.  Float16
results below 2^-14 are off by half of their smallest step, 2^-25, each."""
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


def _rows(m, d, dtype, seed, spread=0.5):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(m, d, generator=g, device="cuda")
    x[:, ::96] *= 8.0
    return (x * torch.exp(torch.randn(m, 1, generator=g, device="cuda") * spread)).to(dtype)


def _param(d, dtype, seed, mean):
    return (mean + 0.3 * torch.randn(d, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")).to(dtype)


def _hat(t, kind, eps):
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    return t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)


def _times(t, w, b):
    t = t if w is None else t * w
    return t if b is None else t + b


def _rstd(t, kind, eps):
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    return 1 / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)


def _check_rows(got, want, before, dtype, name):
    assert got.dtype == dtype and got.shape == want.shape
    floor = 2.0 ** -25 * want.shape[-1] ** 0.5 if dtype == torch.float16 else 0.0
    off, norm = (got.double() - want).norm(dim=-1), want.norm(dim=-1)
    most = R.roundoff(dtype) * norm + 4e-5 * torch.maximum(norm, before.norm(dim=-1)) + floor
    assert bool((off <= most).all()), (name, float((off / most).max()))


def _check_param(got, want, terms, dtype, name):
    assert got.dtype == dtype and got.shape == want.shape
    floor = 2.0 ** -25 * want.shape[-1] ** 0.5 if dtype == torch.float16 else 0.0
    off, norm = float((got.double() - want).norm()), float(want.norm())
    u = R.roundoff(dtype) if dtype != torch.float32 else 0.0
    assert off <= u * norm + 4e-5 * max(norm, float(terms.norm())) + floor, (name, off / max(norm, 1e-300))


# 16, 32 and 64 lanes a row, workgroups of one to twelve waves, two passes
SHAPES = [(1, 1), (3, 7), (40, 8), (37, 100), (18, 128), (21, 129), (9, 200), (7, 300), (5, 512), (11, 513), (6, 1000),
          (5, 2049), (3, 6144), (4, 6145), (5, 7001), (3, 17408), (2, 32768)]
# rows that a group of lanes comes back for, and a remainder: 16 rows in each of 768 workgroups, 8, 4; workgroups of
# two waves and of twelve; two passes' workgroups, of which 153 and 85 take rows
TURNS = [(12300, 128), (12345, 40), (6200, 200), (3100, 400), (1600, 1000), (300, 6144), (200, 9000), (100, 17408)]
FORMS = [("rms", False, False), ("rms", True, False), ("rms", True, True), ("layer", False, False),
         ("layer", True, False), ("layer", True, True)]


@pytest.mark.parametrize("kind,weight,bias", FORMS)
@pytest.mark.parametrize("m,d", SHAPES + TURNS)
@pytest.mark.parametrize("dtype,pt", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
def test_norm(xt, m, d, kind, weight, bias, dtype, pt):
    """dx, dweight and dbias of the plain norm."""
    x = _rows(m, d, dtype, m + d).requires_grad_()
    w = _param(d, pt, 1, 1.0).requires_grad_() if weight else None
    b = _param(d, pt, 2, 0.0).requires_grad_() if bias else None
    dh = _rows(m, d, dtype, 3, spread=0.3)
    leaves = [t for t in (x, w, b) if t is not None]
    got = torch.autograd.grad(xt.norm(x, w, b, kind=kind, eps=1e-5), leaves, dh)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    xd, wd = wide[0], wide[1] if weight else None
    want = torch.autograd.grad(_times(_hat(xd, kind, 1e-5), wd, wide[2] if bias else None), wide, dh.double())
    with torch.no_grad():
        c = dh.double() if wd is None else dh.double() * wd
        _check_rows(got[0], want[0], c * _rstd(xd, kind, 1e-5), dtype, "x")
        if weight:
            _check_param(got[1], want[1], dh.double() * _hat(xd, kind, 1e-5), pt, "weight")
        if bias:
            _check_param(got[2], want[2], dh.double(), pt, "bias")


@pytest.mark.parametrize("m,d", [(40, 96), (3100, 400), (5, 700), (90, 9000)])
@pytest.mark.parametrize("frozen", ("x", "weight", "bias", "weight and bias", "x and bias", "x and weight"))
def test_some_of_a_norms_gradients(xt, m, d, frozen):
    """Those that are wanted have the bits that they have beside the others: sums or none, with the bias' or without.
    (A frozen bias has no sum, but its place is another kernel's: the same results to their one rounding.)"""
    v = {"x": _rows(m, d, torch.float16, 1), "weight": _param(d, torch.float32, 1, 1.0), "bias": _param(d, torch.float32, 2, 0.0)}
    dh = _rows(m, d, torch.float16, 3, spread=0.3)

    def step(frozen):
        leaves = {n: t.detach().requires_grad_(n not in frozen) for n, t in v.items()}
        want = [n for n in leaves if leaves[n].requires_grad]
        return dict(zip(want, torch.autograd.grad(xt.norm(leaves["x"], leaves["weight"], leaves["bias"]),
                                                  [leaves[n] for n in want], dh)))

    full, some = step(()), step(frozen.split(" and "))
    assert set(some) == set(full) - set(frozen.split(" and "))
    for n, t in some.items():
        if "bias" not in frozen:
            assert torch.equal(t, full[n]), n
        u = R.roundoff(t.dtype) if t.dtype == torch.float16 else 4e-5
        assert float((t - full[n]).double().norm()) <= 2 * u * float(full[n].double().norm()), n


CASES = [("rms", "rms", "sigmoid", "tensor"), ("rms", "rms", None, "tensor"), ("rms", None, "none", 0.3),
         (None, "rms", "silu", None), ("rms", None, None, None), (None, None, "sigmoid", "tensor"),
         ("layer", "rms", "silu", "tensor"), ("rms", "layer", None, 0.5)]


@pytest.mark.parametrize("kind,post,act,scale", CASES)
@pytest.mark.parametrize("m,d", [(37, 100), (9, 200), (7, 300), (5, 1000), (4, 2049), (3, 6144), (5, 7001)] + TURNS)
@pytest.mark.parametrize("bias", (False, True))
def test_residual_norm(xt, m, d, kind, post, act, scale, bias):
    """Every tensor's gradient, with biases and without: "rms" alone has kernels of its own."""
    dtype = torch.bfloat16 if m % 2 else torch.float16
    v = {"block": _rows(m, d, dtype, 1), "residual": _rows(m, d, dtype, 2)}
    if act:
        v["gate"] = _rows(m, d, dtype, 3, spread=0.2)
    if scale == "tensor":
        v["scale"] = _param(d, torch.float32, 4, 0.5)
    for there, name, seed in ((kind, "weight", 5), (post, "post_weight", 6)):
        if there:
            v[name] = _param(d, torch.float32, seed, 1.0)
            if bias:
                v[name.replace("weight", "bias")] = _param(d, torch.float32, seed + 4, 0.0)
    for t in v.values():
        t.requires_grad_()
    number = 1.0 if scale in (None, "tensor") else scale
    args = {n: t for n, t in v.items() if n not in ("block", "residual", "scale")}
    out = xt.residual_norm(v["block"], v["residual"], kind=kind, post=post, gate_act=act or "none", eps=1e-6,
                           post_eps=1e-5, scale=v["scale"] if scale == "tensor" else scale, **args)
    out = [o for o in out if o is not None]
    douts = [_rows(m, d, dtype, 20 + i, spread=0.3) for i in range(len(out))]
    got = dict(zip(v, torch.autograd.grad(out, list(v.values()), douts)))
    w = {n: t.detach().double().requires_grad_() for n, t in v.items()}
    hat = _hat(w["block"], post, 1e-5) if post else w["block"]
    p = _times(hat, w.get("post_weight"), w.get("post_bias"))
    g = w.get("gate")
    f = None if g is None else g if act == "none" else torch.sigmoid(g) * (g if act == "silu" else 1.0)
    q = p if f is None else p * f
    y = w["residual"] + q * w.get("scale", number)
    wout = [y] + ([_times(_hat(y, kind, 1e-6), w.get("weight"), w.get("bias"))] if kind else [])
    want = dict(zip(w, torch.autograd.grad(wout, list(w.values()), [t.double() for t in douts])))
    with torch.no_grad():
        before = douts[0].double()
        if kind:
            before = before.abs() + (_times(douts[1].double(), w.get("weight"), None) * _rstd(y, kind, 1e-6)).abs()
        s = w.get("scale", torch.full((d,), number, dtype=torch.float64, device="cuda"))
        to = s if f is None else s * f                  # what y's gradient comes to p with
        inner = to if not post else to * w["post_weight"] * _rstd(w["block"], post, 1e-5)
        # a row's error in y's gradient is `before`'s, times what each of its places is multiplied with
        size = before.norm(dim=-1, keepdim=True) / d ** 0.5
        most = {"residual": before, "block": (before + size) * inner.abs()}
        terms = {"scale": (before + size) * q, "post_weight": (before + size) * to * hat,
                 "post_bias": (before + size) * to}
        if kind:
            terms.update(weight=douts[1].double() * _hat(y, kind, 1e-6), bias=douts[1].double())
        if g is not None:
            slope = torch.ones_like(g) if act == "none" else torch.sigmoid(g) * (1 - torch.sigmoid(g))
            if act == "silu":
                slope = torch.sigmoid(g) * (1 + g * (1 - torch.sigmoid(g)))
            most["gate"] = (before + size) * (s * p * slope).abs()
        for n, t in got.items():
            if n in most:
                _check_rows(t, want[n], most[n], dtype, n)
            else:
                _check_param(t, want[n], terms[n], torch.float32, n)
