"""The gated block between norms in the example (exl3xpu-mixedk_amd/examples/trellis_block.py)."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "exl3xpu-mixedk_amd", "examples"))


def test_gated_block():
    """Three weights' errors in squares, twice that for the code's distance from the bound (as test_gpu_example.py); a
    norm is off by its own rounding, 2^-8 of each value at most, and by that of the sum which it is compared with."""
    import trellis_block
    out = trellis_block.main(["--dim", "256", "--hidden", "384", "--experts", "4", "--tokens", "128"])
    assert out["replays equal eager"]
    assert out["gated error"] <= 2 * (2 * 4.0 ** -4 + 4.0 ** -5) ** 0.5
    assert out["normed error"] <= 2 * 2.0 ** -8
    assert all(0 < g < float("inf") for g in out["norms' gradients"])
