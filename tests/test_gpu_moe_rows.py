"""A mixture layer whose full batch takes more counters than a call has, against its definition in 64 bits."""
import pytest
import torch

from test_gpu_moe import Layer, _check, _router, _x, xt  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", (1, 40, 64, 130))
def test_many_wide_experts(xt, oracle_mod, rows):  # noqa: F811
    layer = Layer(xt, oracle_mod, 128, 3840, [(2, 3, 2)] * 3, 700)
    idx, ws = [e % 3 for e in range(512)], layer.experts.weights
    layer.experts = xt.TrellisExperts(*([ws[3 * i + r] for i in idx] for r in range(3)))
    layer.dense = [layer.dense[i] for i in idx]
    assert xt._moe_rows(512, 16, 128, 3840) < 64
    x, router = _x(rows, 128, torch.bfloat16, 3), _router(512, 128, torch.bfloat16, 4)
    valid = (torch.arange(rows) % 7 != 3).cuda()
    _check(layer, xt, x, router, 16, residual=_x(rows, 128, torch.bfloat16, 5), valid=valid)


def test_one_token_too_many(xt):  # noqa: F811
    """What no call can count is refused before anything runs."""
    layer = type("experts", (), dict(device=torch.device("cuda", 0), d=128, f=1 << 20, n=512, _rows={}))
    x, router = _x(1, 128, torch.float16, 1), _router(512, 128, torch.float16, 2)
    with pytest.raises(ValueError, match="count"):
        xt.moe(x, router, layer, 16)
