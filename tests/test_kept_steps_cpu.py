"""How many captured steps are kept: books only."""
from ithaca_b200.engine import graph
from ithaca_b200.engine.graph import GraphDecoder


def test_steps_of_sequences_that_share_pages_are_kept_up_to_a_number():
    d = GraphDecoder(None)
    for n in range(300):
        d._keep((n, 4), n)                                       # steps that share nothing: all are kept
        d._keep((8, 4, (1, 4, 1 << n, 1)), n)
    shared = [k for k in d.graphs if len(k) > 2]
    assert len(shared) == graph.SHARED_KEPT == 64 and len(d.graphs) == 364
    assert [k[2][2] for k in shared] == [1 << n for n in range(236, 300)]
    first, last = shared[0], shared[-1]
    d.graphs[first] = d.graphs.pop(first)                       # used again: the next one goes instead
    d._keep((8, 4, (2, 4, 1, 1)), 0)
    assert first in d.graphs and last in d.graphs and shared[1] not in d.graphs
    d._keep((8, 4, (2, 4, 1, 1), None), 1)                      # a second key/value group
    assert len([k for k in d.graphs if len(k) > 2]) == 64
