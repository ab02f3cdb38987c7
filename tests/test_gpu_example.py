"""The example that takes a block from calibration to serving (exl3xpu-mixedk_amd/examples/trellis_block.py)."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "exl3xpu-mixedk_amd", "examples"))


def test_trellis_block():
    """K bits a weight leave an error of 2^-K of a Gaussian weight at best; the products of a layer's two or three
    weights add theirs in squares, and twice that is allowed for the code's distance from the bound."""
    import trellis_block
    out = trellis_block.main(["--dim", "256", "--hidden", "384", "--experts", "4", "--tokens", "128"])
    assert out["mixture finite"] and out["padding without experts"] and out["replays equal eager"]
    assert out["dense error"] <= 2 * (4.0 ** -4 + 4.0 ** -3) ** 0.5
    assert out["mixture error"] <= 2 * (2 * 4.0 ** -4 + 4.0 ** -5) ** 0.5
    before, after = out["loss before, after"]
    assert after < before
