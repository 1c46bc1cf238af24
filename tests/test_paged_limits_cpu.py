"""Refusals at the limits of what the paged cache's entry points count with, from the host's checks."""
import pytest

from test_paged_cpu import append, attention, read, verify


@pytest.mark.parametrize("call", [append, attention, read])
@pytest.mark.parametrize("page,pages", [(16, 2**26), (256, 2**22)])
def test_page_tables_of_more_than_a_billion_positions(call, page, pages):
    """Positions are rounded up to tiles and pages in 32 bits: tables beyond 2^30 of them are refused. (Calls without new
    tokens, or reading nothing, show what is taken: they end before a launch.)"""
    nothing = dict(count=0) if call is read else {}
    empty = dict(n_tokens=0, max_new=0)
    assert call(cache=dict(page=page), batch=dict(empty, pages_per_seq=pages), **nothing) == "Ok"
    assert call(cache=dict(page=page), batch=dict(empty, pages_per_seq=pages + 1), **nothing) == "ShapeMismatch"
    assert call(cache=dict(page=page), batch=dict(pages_per_seq=2**31 - 1)) == "ShapeMismatch"


def test_no_sequences_need_no_arrays():
    assert verify(seqs=0, target=None, draft=None, ds=0, tokens=None, u=None, acc=None, out=None) == "Ok"
    assert verify(seqs=0, target=None, vocab=0) == "ShapeMismatch"
    assert verify(seqs=1, u=None) == "InvalidArgument"
