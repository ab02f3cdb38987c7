"""The input Gram's accumulation arguments (trellis_ops.input_gram)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def xt():
    import trellis_ops
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    trellis_ops._hb.lib()
    return trellis_ops


def test_prev_across_out_is_refused(xt):
    """Elements of prev that out's rows have been written over already would be read."""
    x, room = torch.randn(3, 256).half().cuda(), torch.zeros(3 * 65536, device="cuda")
    at = lambda i: room[i:i + 65536].view(256, 256)  # noqa: E731
    for i, j in ((0, 256), (4, 0), (65535, 0)):
        with pytest.raises(ValueError, match="apart"):
            xt.input_gram(x, prev=at(i), out=at(j))
    assert torch.equal(xt.input_gram(x, prev=at(65536), out=at(0)), xt.input_gram(x))
