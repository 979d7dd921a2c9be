"""The order in which a pool's pages are given (``sgl_amd_mono.moe.pages``), where they do not suffice."""

import pytest

from test_gpu_pages import Both

pytestmark = pytest.mark.gpu


def test_rows_behind_one_that_goes_without():
    """A prompt that the pool does not hold: rows before it and rows that need no page go on, those behind it that need
    one do not; ordered behind them, or in a call of its own, it holds nobody up."""
    b = Both(20, 4, 4, 40, layers=0)
    b.grow([4, 8, 3, 4])  # 1 + 2 + 1 + 1 pages
    b.same()
    b.grow([1, 70, 1, 1])  # the first gets a page, the third has room in its own, the last goes without
    b.same()
    assert b.n == [5, 8, 4, 4] and b.ref.errors == [(3, 1), (3, 3)]
    b.grow([0, 0, 0, 1])
    b.same()
    b.grow([4, 0, 1, 70])  # the prompt behind the others
    b.same()
    assert b.n == [9, 8, 5, 5] and b.ref.errors[2:] == [(3, 3)]


def test_cut_into_a_page_whose_other_holder_goes():
    """Holders count as they were before the call: the row that stays needs a page of its own."""
    b = Both(4, 4, 3, 4, layers=1)
    b.grow([8, 0, 8])
    b.trim([8, 0, 0])
    b.fork([0, 0, -1])  # both hold the first two pages
    b.grow([0, 0, 8])  # the other two
    b.same()
    b.trim([6, 0, 8])
    b.same()
    assert b.n == [8, 0, 8] and b.ref.errors == [(3, 0)]
    b.trim([6, 0, 8])  # it holds them alone now, and needs none
    b.same()
    assert b.n == [6, 0, 8]
