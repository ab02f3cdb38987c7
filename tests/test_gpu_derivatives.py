"""Derivatives that the operators on trellis weights do not have are refused, never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fad

import trellis_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def xt():
    import trellis_ops
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    trellis_ops._hb.lib()
    return trellis_ops


def _half(*shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(len(shape))).half().cuda()


def _calls(xt):
    """Each operator's call by the name of the input that is given."""
    w = xt.TrellisLinear(*R.random_weight(256, 128, 4, 1), 4)
    down = xt.TrellisLinear(*R.random_weight(128, 256, 4, 2), 4)
    e = xt.TrellisExperts([w, w], [w, w], [down, down])
    x, router = _half(3, 256), _half(2, 256)
    return {"linear x": (x, lambda t: xt.linear(t, w)),
            "linear bias": (_half(128), lambda t: xt.linear(x, w, bias=t)),
            "linear residual": (_half(3, 128), lambda t: xt.linear(x, w, residual=t)),
            "moe x": (x, lambda t: xt.moe(t, router, e, 1)),
            "moe router": (router, lambda t: xt.moe(x, t, e, 1)),
            "moe residual": (x, lambda t: xt.moe(x, router, e, 1, residual=t)),
            "input_gram x": (x, lambda t: xt.input_gram(t)),
            "input_gram prev": (_half(256, 256).float(), lambda t: xt.input_gram(x, prev=t)),
            "input_gram out": (_half(256, 256).float(), lambda t: xt.input_gram(x, out=t))}


NAMES = ("linear x", "linear bias", "linear residual", "moe x", "moe router", "moe residual", "input_gram x",
         "input_gram prev", "input_gram out")


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("mode", ("grad", "no_grad"))
def test_forward_mode_is_refused(xt, name, mode):
    value, call = _calls(xt)[name]
    with fad.dual_level(), torch.set_grad_enabled(mode == "grad"):
        dual = fad.make_dual(value, torch.ones_like(value))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)
        call(value)                     # without a tangent, inside the level
    call(value)


def test_forward_mode_over_a_gradient_is_refused(xt):
    w = xt.TrellisLinear(*R.random_weight(256, 128, 4, 1), 4)
    x, dy = _half(3, 256).requires_grad_(), _half(3, 128)
    y = xt.linear(x, w, act="silu")
    with fad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, fad.make_dual(dy, dy), retain_graph=True)
        torch.autograd.grad(y, x, dy)


@pytest.mark.parametrize("name", ("moe x", "moe router", "moe residual", "input_gram x", "input_gram prev",
                                  "input_gram out"))
def test_gradient_is_refused(xt, name):
    value, call = _calls(xt)[name]
    value = value.clone().requires_grad_()
    with pytest.raises(NotImplementedError, match="no gradient"):
        call(value)
    with torch.no_grad():
        call(value)


def test_out_is_an_inplace_write_to_autograd(xt):
    """A backward pass that kept the Gram so far has to find that it changed."""
    x, gram = _half(3, 256), torch.zeros(256, 256, device="cuda")
    scale = torch.ones(256, 256, device="cuda", requires_grad=True)
    loss = (scale * gram).sum()
    before = gram._version
    xt.input_gram(x, prev=gram, out=gram)
    assert gram._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    whole = torch.zeros(2, 256, 256, device="cuda")
    loss = (scale * whole[0]).sum()
    xt.input_gram(x, out=whole[0])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        kept = torch.zeros(256, 256, device="cuda")
        assert xt.input_gram(x, prev=kept, out=kept) is kept
        xt.input_gram(x, prev=gram, out=gram)
    assert torch.equal(kept, xt.input_gram(x, out=kept))
