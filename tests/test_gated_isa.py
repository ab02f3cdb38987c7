"""What the gated projection's kernels rely on in their machine code, checked on a compile for gfx950 (no GPU needed).

- gated_gemm_kernel counts its loads: between two meetings of its waves (s_barrier) a wave issues those of one step,
  and waits before the second until no more than these are under way, so that the step before's have arrived.  A wait
  for all of them anywhere in its loop would cost the time of a load in every turn, and so would spilled registers.
- gated_few_kernel of up to 16 rows joins workgroups of all XCDs as few_kernel does: parts stored and read agent-scope
  (sc1), every wave's stores waited for, a barrier, and then one lane counts the workgroup.
"""
import re

import pytest

from test_operators_isa import _bodies


@pytest.fixture(scope="module")
def many(tmp_path_factory):
    return _bodies(tmp_path_factory, "gated_kernels.hip")


@pytest.fixture(scope="module")
def few(tmp_path_factory):
    return _bodies(tmp_path_factory, "gated_few.hip", ["-DXTQ_GATED_CODE=0"])


def test_product_counts_its_loads(many):
    bodies = {k: v for k, v in many.items() if "gated_gemm_kernel" in k}
    assert len(bodies) == 20            # two types; whole and in parts; 2 and 4 groups, 1 and 2 terms, and eight waves
    for name, lines in bodies.items():
        nb, terms, waves = (int(v) for v in re.search(r"ILi\dELi\dELi(\d)ELi(\d)ELi(\d)E", name).groups())
        own = 16 // waves + nb * terms
        steps, loads, products, waits = [], "", 0, []
        for ln in lines:
            assert not ln.startswith("scratch_"), name
            if re.match(r"(buffer|global)_load", ln):
                loads += "a" if re.match(r"buffer_load_\S+ .*\blds\b", ln) else "b"
            products += ln.startswith("v_mfma")
            if ln.startswith("s_waitcnt") and "vmcnt" in ln:
                waits.append(int(re.search(r"vmcnt\((\d+)\)", ln).group(1)))
            if ln == "s_barrier":
                steps.append((loads, products, waits))
                loads, products, waits = "", 0, []
        turn = 2 if nb * terms > 4 else 3
        first = next(i for i, (_, products, _) in enumerate(steps) if products)
        before, loop, rest = steps[first - 1], steps[first:first + turn], steps[first + turn:first + 2 * turn - 1]
        for loads, products, waits in loop:
            assert (loads.count("a"), loads.count("b"), products) == (16 // waves, nb * terms, 8 * nb * terms), name
            assert waits[-1] == own and min(waits) >= own, name
        # what a step leaves under way is younger than the step before's pieces for LDS
        # (nothing follows the last one)
        for one, two in zip([before] + loop + loop[-1:], loop + loop[:1] + rest[:-1]):
            assert two[1] == 8 * nb * terms and two[2][-1] == own, name
            assert len(one[0]) - 1 - one[0].rindex("a") + len(two[0]) >= own, name
        assert [r[1] for r in rest] == [8 * nb * terms] * (turn - 1), name


def test_few_rows_join(few):
    bodies = {k: v for k, v in few.items() if "gated_few_kernelILi1E" in k}
    assert len(bodies) == 8             # x transformed here or apart, one term or two, runs within blocks or over their ends
    for name, lines in bodies.items():
        assert not any(ln.startswith("buffer_wbl2") for ln in lines), name
        count = [i for i, ln in enumerate(lines) if re.match(r"global_atomic_(add|inc)", ln)]
        assert count, name
        for at in count:
            parts = [i for i in range(at) if re.match(r"global_store_dwordx2\s.*\bsc1\b", lines[i])]
            assert parts, name
            between = lines[parts[-1]:at]
            wait = next(i for i, ln in enumerate(between) if "vmcnt(0)" in ln)
            assert any(ln == "s_barrier" for ln in between[wait:]), name
        assert any(re.match(r"global_load_dwordx2\s.*\bsc1\b", ln) for ln in lines[count[0]:]), name
