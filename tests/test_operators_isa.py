"""What the operators' kernels rely on in their machine code, checked on a compile for gfx950 (no GPU needed).

- few_kernel joins workgroups of all XCDs: parts are stored and read agent-scope (sc1: past the L2 of the own XCD),
  every wave waits for its stores (vmcnt(0)) and meets the others at a barrier before one lane counts the workgroup,
  and no L2 is written back.
- gemm_kernel has loads to LDS in flight while it reads LDS and multiplies: a wait for all of them (vmcnt(0)) between
  a step's barrier and its products would cost two fifths of its rate.  The compiler adds one where it takes a read
  for a possible read of what is still to be written, as with a second LDS object beside the buffers.
"""
import os
import re
import shutil
import subprocess

import pytest

from conftest import PKG

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


def _bodies(tmp_path_factory, source, defines=()):
    if not os.path.exists(HIPCC) and not shutil.which("hipcc"):
        pytest.skip("hipcc not available")
    out = str(tmp_path_factory.mktemp("isa") / "out.s")
    subprocess.run([HIPCC if os.path.exists(HIPCC) else "hipcc", "--offload-arch=gfx950", "-O3", "-std=c++17",
                    "-ffp-contract=off", "-fvisibility=hidden", "-fno-gpu-flush-denormals-to-zero", "-Xclang",
                    "-target-feature", "-Xclang", "-packed-fp32-ops", *defines, "--cuda-device-only", "-S",
                    os.path.join(PKG, "csrc", source), "-o", out], check=True, capture_output=True)
    found = re.finditer(r"^(_Z\S*?_kernel\S*):[^\n]*\n(.*?)^\.Lfunc_end", open(out).read(), re.S | re.M)
    return {m.group(1): [ln.split(";")[0].strip() for ln in m.group(2).split("\n")] for m in found}


@pytest.fixture(scope="module")
def few(tmp_path_factory):
    return _bodies(tmp_path_factory, "few_kernels.hip", ["-DXTQ_FEW_K=4"])


@pytest.fixture(scope="module")
def many(tmp_path_factory):
    return _bodies(tmp_path_factory, "linear_kernels.hip")


def test_few_rows_join(few):
    bodies = {k: v for k, v in few.items() if "few_kernel" in k}
    assert len(bodies) == 15            # three codes; x transformed here, with two terms, and 1, 2, 4 groups apart
    for name, lines in bodies.items():
        assert not any(ln.startswith("buffer_wbl2") for ln in lines), name
        count = [i for i, ln in enumerate(lines) if re.match(r"global_atomic_(add|inc)", ln)]
        assert len(count) == 1, name
        parts = [i for i in range(count[0]) if re.match(r"global_store_dwordx2\s.*\bsc1\b", lines[i])]
        assert parts, name
        between = lines[parts[-1]:count[0]]
        wait = next(i for i, ln in enumerate(between) if "vmcnt(0)" in ln)
        assert any(ln == "s_barrier" for ln in between[wait:]), name
        assert any(re.match(r"global_load_dwordx2\s.*\bsc1\b", ln) for ln in lines[count[0]:]), name


def test_product_loop_waits_for_no_load_to_lds(many):
    bodies = {k: v for k, v in many.items() if "gemm_kernel" in k}
    assert len(bodies) >= 14
    for name, lines in bodies.items():
        products = [i for i, ln in enumerate(lines) if ln.startswith("v_mfma")]
        first, last = products[0], products[-1]
        # from the loop's head (the last label before the first product) to its last product
        head = max(i for i in range(first) if re.match(r"\.LBB\d+_\d+:", lines[i]))
        assert any(ln.startswith("ds_read") for ln in lines[head:first]), name
        assert not any("vmcnt(0)" in ln for ln in lines[head:last]), name
