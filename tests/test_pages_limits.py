"""Tables that are wider than the calls on pages take: refused before anything is launched, so that nothing has moved."""
import pytest

from cachegen_b200 import _lib
from test_pages_refusals import copy_job, pages_job


@pytest.mark.parametrize("width", [2 ** 31 - 1024, 2 ** 31 - 1])
def test_rows_that_are_too_wide(width):
    L, given = _lib.lib(), dict(width=width, page_size=1, nrows=1, nnew=1, ntokens=1)
    assert L.cg_fork_pages(pages_job(**given), None, None) == -2 and L.cg_free_pages(pages_job(**given), None) == -2
    assert L.cg_extend_pages(pages_job(**given), None) == -2 and L.cg_compact_pages(pages_job(**given), None, None) == -2


def test_tables_of_too_many_entries():
    L, given = _lib.lib(), dict(width=2 ** 29, page_size=1, nrows=4096, nnew=4096)
    for copy in (None, copy_job(page_size=1)):
        assert L.cg_fork_pages(pages_job(**given), copy, None) == -2 and L.cg_compact_pages(pages_job(**given), copy, None) == -2
