"""The C entries of the norms, called as a C program does, where the Python functions refuse or never make the call."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

PARAMS = ("weight", "bias", "scale", "post_weight", "post_bias")


@pytest.fixture(scope="module")
def hb():
    import hip_backend
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    hip_backend.lib()
    return hip_backend


def _both(hb, kind, post, params, m, d):
    """y, h and all gradients of a gated residual sum; params: fp32 tensors [d] by name."""
    g = torch.Generator("cuda").manual_seed(m + d)
    x, res, gate, dy, dh = (torch.randn(m, d, generator=g, device="cuda", dtype=torch.float16) for _ in range(5))
    p = hb.NormParams(kind, post, 1, sum(1 << i for i, n in enumerate(PARAMS) if n in params), 1e-6, 1e-6, 0.5,
                      *(params[n].data_ptr() if n in params else None for n in PARAMS))
    out = {n: torch.zeros(m, d, device="cuda", dtype=torch.float16) for n in ("y", "h", "dx", "dres", "dgate")}
    out["dscale"] = torch.zeros(d, device="cuda", dtype=torch.float32 if "scale" in params else torch.float16)
    stats = torch.empty(m, 4, device="cuda")
    stream, at = torch.cuda.current_stream().cuda_stream, {n: t.data_ptr() for n, t in out.items()}
    assert hb.lib().xtq_norm_dev(
        ctypes.byref(p), 1, m, d, x.data_ptr(), d, res.data_ptr(), d, gate.data_ptr(), d, at["y"], d,
        at["h"] if kind else None, d, stats.data_ptr(), stream) == 0
    need = hb.lib().xtq_norm_bwd_ws_bytes(m, d, 1)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    assert hb.lib().xtq_norm_bwd_dev(
        ctypes.byref(p), 1, m, d, x.data_ptr(), d, res.data_ptr(), d, gate.data_ptr(), d, stats.data_ptr(),
        dy.data_ptr(), d, dh.data_ptr() if kind else None, d, at["dx"], at["dres"], at["dgate"],
        (ctypes.c_void_p * 5)(None, None, at["dscale"], None, None), ws.data_ptr(), need, stream) == 0
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("m,d", [(5, 100), (9, 200), (20, 1000), (3, 7000)])
@pytest.mark.parametrize("kind,post,idle", [
    (1, 0, ("post_weight",)), (1, 0, ("post_weight", "post_bias")), (2, 0, ("post_weight", "post_bias")),
    (0, 1, ("weight",)), (0, 2, ("weight", "bias")), (0, 0, ("weight", "bias", "post_weight", "post_bias"))])
def test_parameters_of_a_norm_that_is_not_there(hb, m, d, kind, post, idle):
    """They are read by neither direction, whatever they hold."""
    params = {n: torch.linspace(0.5, 2.0, d, device="cuda") for n in
              ("scale", *(("weight",) if kind else ()), *(("post_weight",) if post else ()))}
    want = _both(hb, kind, post, params, m, d)
    for value in (3.0, float("nan")):
        got = _both(hb, kind, post, {**params, **{n: torch.full((d,), value, device="cuda") for n in idle}}, m, d)
        for n, t in want.items():
            assert torch.equal(got[n], t), (n, value)
