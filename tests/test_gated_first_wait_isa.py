"""The wait before the first step of the gated projection's product, in its machine code (a compile for gfx950, no GPU
needed): it leaves as many loads under way as a step issues, the youngest, so none of the first step's pieces for LDS
may be among these, or its waves read LDS before it is written."""
import os
import re

from conftest import PKG
from test_operators_isa import _bodies


def _first_wait(lines, pieces, own):
    """Whether the first `pieces` loads to LDS are older than the `own` loads that the first meeting waits for none of."""
    loads = ""
    for ln in lines:
        if re.match(r"(buffer|global|flat)_load", ln):
            loads += "a" if re.match(r"buffer_load_\S+ .*\blds\b", ln) else "b"
        wait = re.match(r"s_waitcnt .*vmcnt\((\d+)\)", ln)
        if wait:
            left = int(wait.group(1))
        if ln == "s_barrier":
            last = [i for i, c in enumerate(loads) if c == "a"][pieces - 1]
            return left <= own and len(loads) - 1 - last >= left
    return False


def test_the_check_sees_a_wrong_order():
    a, b, meet = "buffer_load_dwordx4 v1, s[0:3], 0 offen lds", "global_load_dwordx4 v[0:3], v[4:5], off", ["s_waitcnt vmcnt(3)", "s_barrier"]
    assert _first_wait([a, b, b, a, b, b, *meet], 1, 3)
    assert _first_wait([b, a, b, a, b, *meet], 1, 3)
    assert not _first_wait([b, b, b, b, a, a, *meet], 1, 3)
    assert not _first_wait([b, b, a, b, a, *meet], 1, 3)


def test_first_pieces_are_waited_for(tmp_path_factory):
    bodies = {k: v for k, v in _bodies(tmp_path_factory, "gated_kernels.hip").items() if "gated_gemm_kernel" in k}
    assert len(bodies) == 20
    for name, lines in bodies.items():
        nb, terms, waves = (int(v) for v in re.search(r"ILi\dELi\dELi(\d)ELi(\d)ELi(\d)E", name).groups())
        assert _first_wait(lines, 16 // waves, 16 // waves + nb * terms), name


def test_the_order_is_fixed_in_the_source():
    """Between the first step's loads to LDS and all others lies a fence, so that the order is not the compiler's choice."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(PKG, "csrc", "gated_kernels.hip")).read())
    assert re.search(r"load_a\(s0\);\s*asm volatile\(\"\" ::: \"memory\"\);\s*load_b\(s0, c0\);", text)
