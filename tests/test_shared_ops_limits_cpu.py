"""Sizes at which the entry points over selected blocks and shared pages stop, refused before they touch a device; every pointer is made up."""
import pytest

from test_shared_ops_cpu import _args, _call


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("n,block", [((1 << 22) + 1, 256), (1 << 23, 256), ((1 << 23) + 1, 256), (1 << 25, 64), (1 << 25, 256)])
def test_listed_tokens(paged, n, block):
    """Places in a list are 32-bit numbers of tokens: a list of more than 2^30 is refused, though its entries are fewer than 2^25."""
    got = _call("blocks", _args("blocks", paged, dict(B=1, Hq=4, n_blocks=n, block=block, page_size=256)))
    assert got[0] == 2 and "listed tokens" in got[1], got


@pytest.mark.parametrize("kw", [dict(B=0), dict(n_new=0), dict(B=0, n_new=0)])
def test_reserve_without_counts(kw):
    """The plan reads the counts of all pages, also where there is nothing to reserve."""
    got = _call("reserve", _args("reserve", False, dict(page_refs=None, **kw)))
    assert got[0] == 1 and "null" in got[1], got
