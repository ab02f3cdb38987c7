"""How many tokens of a mixture layer one call takes (trellis_ops._moe_rows): all 64 where the counters allow it, the
most that they allow elsewhere."""
import os
import subprocess

import pytest

from conftest import PKG


@pytest.fixture(scope="module")
def xt():
    if not os.path.exists(os.path.join(PKG, "lib", "libexl3vit.so")):
        subprocess.run(["make", "-s", "-C", PKG], check=True)
    import trellis_ops
    trellis_ops._hb.lib()
    return trellis_ops


@pytest.mark.parametrize("experts,top,d,f", [(8, 2, 256, 384), (64, 8, 2048, 1024), (512, 8, 4096, 4096),
                                             (512, 16, 4096, 4096), (256, 8, 7168, 8192), (512, 16, 128, 1 << 16),
                                             (1, 1, 128, 1 << 20)])
def test_most_rows(xt, experts, top, d, f):
    rows, need = xt._moe_rows(experts, top, d, f), xt._hb.lib().xtq_moe_ws_bytes
    assert 1 <= rows <= 64 and need(rows, experts, top, d, f) > 0
    assert rows == 64 or need(rows + 1, experts, top, d, f) < 0


def test_bounds(xt):
    assert xt._moe_rows(64, 8, 2048, 1024) == 64
    assert xt._moe_rows(512, 8, 4096, 4096) == 63           # 64 would make 512 lists of 32 blocks
    assert xt._moe_rows(512, 16, 128, 1 << 20) == 0
