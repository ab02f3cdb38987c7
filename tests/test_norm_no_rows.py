"""No rows: the norms' C entry has nothing to do, and empty tensors' addresses are NULL."""
import pytest

from test_norm_capi import _norm, _params
from test_operators_capi import hb  # noqa: F401  (the fixture)


@pytest.mark.parametrize("kw", (dict(), dict(kind=0), dict(post=0, post_weight=None), dict(scale=None)))
def test_no_rows_at_null(hb, kw):  # noqa: F811
    assert _norm(hb, _params(hb, **kw), rows=0, x=None, res=None, gate=None, y=None, h=None, stats=None) == 0


def test_what_is_wrong_without_rows_too(hb):  # noqa: F811
    none = dict(rows=0, x=None, res=None, gate=None, y=None, h=None, stats=None)
    for kw, rc in ((dict(kind=3), 15), (dict(post=-1), 15), (dict(gate_act=3), 15)):
        assert _norm(hb, _params(hb, **kw), **none) == rc
    assert _norm(hb, **{**none, "d": 0}) == 6 and _norm(hb, **{**none, "type": 2}) == 15
