"""The kernels of two terms join workgroups as those of one do (test_operators_isa.py): parts are stored and read
agent-scope, every wave waits for its stores and meets the others before one lane counts the workgroup."""
import re

import pytest

from test_operators_isa import _bodies


@pytest.fixture(scope="module")
def two(tmp_path_factory):
    return _bodies(tmp_path_factory, "few_kernels.hip", ["-DXTQ_FEW_K=4", "-DXTQ_FEW_TWO"])


def test_join(two):
    bodies = {k: v for k, v in two.items() if "few_kernel" in k}
    assert len(bodies) == 9             # three codes; 1, 2, 4 groups of rows
    for name, lines in bodies.items():
        assert not any(ln.startswith("buffer_wbl2") for ln in lines), name
        count, = [i for i, ln in enumerate(lines) if re.match(r"global_atomic_(add|inc)", ln)]
        parts = [i for i in range(count) if re.match(r"global_store_dwordx2\s.*\bsc1\b", lines[i])]
        between = lines[parts[-1]:count]
        wait = next(i for i, ln in enumerate(between) if "vmcnt(0)" in ln)
        assert "s_barrier" in between[wait:], name
        assert any(re.match(r"global_load_dwordx2\s.*\bsc1\b", ln) for ln in lines[count:]), name
