"""Cuts inside shared pages: the copy is made before the books change."""
import pytest

from ithaca_b200.cache import KVRequest, SequenceCache
from ithaca_b200.csrc.ops import KernelError


def cache(pages, requests=None):
    return SequenceCache(requests or {0: [KVRequest(2, 16)], 1: [KVRequest(1, 32)]}, max_tokens=64 * pages, max_slots=4, device=None)


def grown(c, n):
    s = c.alloc_slot()
    c.reserve([s], [n])
    c.commit([s], [n])
    return s


def books(c):
    t = c.table
    return ([x.copy().tolist() for x in t.tables], t.length.tolist(), t._reserved.tolist(), [sorted(p._free) for p in t.pools], [p._holders.tolist() for p in t.pools],
            [p.n_shared for p in t.pools])


@pytest.mark.parametrize("pages", [5, 12])
def test_a_cut_whose_copy_fails_changes_nothing(pages, monkeypatch):
    """With pages to spare, and where the only page to be had is one that the cut gives back."""
    c = cache(pages)
    a = grown(c, 200)                                              # three full pages and a begun one
    (b,), = c.fork([(a, 1)])
    assert c.table.pools[0].n_free == pages - 5
    before, asked = books(c), []
    def fail(jobs, src, dst):
        asked.append([list(j) for j in jobs])
        raise KernelError("lost")
    with monkeypatch.context() as m:
        m.setattr(c, "_copy", fail)
        with pytest.raises(KernelError, match="lost"):
            c.truncate(b, 70)
    assert books(c) == before and all(len(j) == 1 for j in asked[0])
    c.table.check_consistent()
    done = []
    monkeypatch.setattr(c, "_copy", lambda jobs, src, dst: done.append([list(j) for j in jobs]))
    c.truncate(b, 70)
    c.table.check_consistent()
    for g in range(2):
        (old, new, rows), = done[0][g]
        assert (old, new, rows) == (c.table.tables[g][a, 1], c.table.tables[g][b, 1], 6) and old != new
        assert (c.table.tables[g][b, 2:] == -1).all() and c.table.tables[g][b, 0] == c.table.tables[g][a, 0]
    assert c.length(b) == 70 and c.length(a) == 200
    c.free_slot(a)
    c.free_slot(b)
    assert all(p.n_free == pages and p.n_shared == 0 for p in c.table.pools)


def test_a_cut_that_needs_no_copy_asks_for_none(monkeypatch):
    c = cache(12)
    a = grown(c, 200)
    (b,), = c.fork([(a, 1)])
    monkeypatch.setattr(c, "_copy", lambda *x: pytest.fail("nothing to copy"))
    c.truncate(b, 128)                                             # at a page's end
    c.truncate(b, 0)
    c.truncate(a, 195)                                             # inside the page that is a's own
    c.table.check_consistent()
