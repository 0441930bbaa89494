"""Tables that are wider than the calls on pages take: refused before anything is launched, so that nothing has moved."""
from cachegen_b200 import _lib
from test_pages_refusals import copy_job, pages_job


def test_tables_of_too_many_entries():
    L, given = _lib.lib(), dict(width=2 ** 29, page_size=1, nrows=4096, nnew=4096)
    for copy in (None, copy_job(page_size=1)):
        assert L.cg_fork_pages(pages_job(**given), copy, None) == -2 and L.cg_compact_pages(pages_job(**given), copy, None) == -2
