"""How many registers a lane the norms' and the few rows' gated kernels keep in scratch, on a compile for gfx950 (no GPU
needed): none but those that their comments name, and no more than they say."""
import os
import re
import shutil
import subprocess

import pytest

from conftest import PKG
from test_operators_isa import HIPCC


def _spills(tmp_path, source, defines=()):
    """Kernel: registers in scratch."""
    if not os.path.exists(HIPCC) and not shutil.which("hipcc"):
        pytest.skip("hipcc not available")
    out = str(tmp_path / "out.s")
    subprocess.run([HIPCC if os.path.exists(HIPCC) else "hipcc", "--offload-arch=gfx950", "-O3", "-std=c++17",
                    "-ffp-contract=off", "-fvisibility=hidden", "-fno-gpu-flush-denormals-to-zero", "-Xclang",
                    "-target-feature", "-Xclang", "-packed-fp32-ops", *defines, "--cuda-device-only", "-S",
                    os.path.join(PKG, "csrc", source), "-o", out], check=True, capture_output=True)
    found = re.findall(r"^\s+\.name:\s+(_Z\S+)\n(?:(?!\s+\.name:).*\n)*?\s+\.vgpr_spill_count:\s+(\d+)", open(out).read(), re.M)
    assert found
    return {name: int(n) for name, n in found}


def _held(spills, allowed):
    """allowed: part of a kernel's name, registers."""
    for name, n in spills.items():
        most = max((m for part, m in allowed if re.search(part, name)), default=0)
        assert n <= most, (name, n, most)


def test_norms(tmp_path):
    """Modes: 3 is a workgroup a row; a gradient is of 0 the norm, 1 a residual sum, 2 one with a gate, then its sums and
    whether it has means and biases."""
    _held(_spills(tmp_path, "norm_kernels.hip"), [
        (r"norm_kernelILi\dELi3ELi6E", 65), (r"norm_bwd_kernelILi\dELi3ELi1ELb1ELb1E", 14),
        (r"norm_bwd_kernelILi\dELi3ELi2ELb1ELb1E", 48), (r"norm_bwd_kernelILi\dELi3ELi2ELb1ELb0E", 6)])


def test_few_rows(tmp_path):
    """Groups of 16 rows, whether the rows are transformed here, two terms, runs within blocks.  (One codebook's.)"""
    _held(_spills(tmp_path, "gated_few.hip", ["-DXTQ_GATED_CODE=0"]), [
        (r"gated_few_kernelILi1ELb\dELb\dELb0E", 31), (r"gated_few_kernelILi1ELb1ELb1ELb1E", 3),
        (r"gated_few_kernelILi4ELb0ELb1ELb1E", 70), (r"gated_few_kernelILi4ELb0ELb1ELb0E", 126),
        (r"gated_few_kernelILi4ELb0ELb0ELb0E", 4)])
