"""What the operators' C entries refuse, and say, beside test_operators_capi.py: input_gram takes prev in out's place or
apart from it, not across it.  No pointer here is ever read."""
import pytest

from test_operators_capi import P, _bwd, _gram, _linear, _moe, hb  # noqa: F401  (the fixture)

FAR = 256 * 256 * 4


@pytest.mark.parametrize("off", (4, 1024, FAR - 4, -4, -FAR + 4))
def test_gram_refuses_prev_across_out(hb, off):  # noqa: F811
    assert _gram(hb, out=P + FAR, prev=P + FAR + off, type=0, ws=P, nws=1 << 40) == 12


def test_message_of_sizes(hb):  # noqa: F811
    """Status 6 is what an operator says of its sizes, too: the text names them."""
    assert b"sizes" in hb.lib().xtq_vit_strerror(6)


@pytest.mark.parametrize("kw,rc", [(dict(type=16 | 2), 15), (dict(type=16 | 1, rows=70, nws=100), 14), (dict(type=32), 15)])
def test_fast_types(hb, kw, rc):  # noqa: F811
    """The flag of 11 bits goes with the products' two types alone."""
    assert _linear(hb, **kw) == rc and _bwd(hb, **kw) == rc
    assert _moe(hb, type=16) == 15 and _gram(hb, type=17) == 15
