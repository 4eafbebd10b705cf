"""Captured steps of sequences that share pages come and go: the results stay those of the same tokens in slots of their own."""
import numpy as np
import pytest

import test_beam_gpu
from helpers import REL_CUT, random_ids
from test_beam_gpu import off, rows

pytestmark = pytest.mark.gpu
dirs = test_beam_gpu.dirs


def test_a_step_that_was_dropped_is_captured_again(dirs, monkeypatch):
    from ithaca_b200 import Engine
    from ithaca_b200.csrc import attention_bf16
    from ithaca_b200.engine import graph
    monkeypatch.setattr(graph, "SHARED_KEPT", 2)
    monkeypatch.setattr(attention_bf16, "sharing_pays", lambda *a: True)
    eng = Engine(dirs("wide"), dtype="bfloat16", max_tokens=64 * 200, max_slots=12)
    prompt = random_ids(330, 300, 7)
    a = eng.alloc_slot()
    eng.step([a], [prompt], None)
    slots = [a] + eng.fork_slot(a, 4)
    alone = eng.alloc_slot()
    eng.step([alone], [prompt], None)
    kept = []
    for n, members in enumerate((2, 3, 4, 4, 2, 5, 1, 3, 2)):
        toks = [[(n * 7) % 300]] * members
        got = eng._decoder.step(slots[:members], toks)[0].float().cpu().numpy().copy()
        for s in slots[members:]:                                 # all sequences stay equal
            eng.step([s], toks[:1], None)
        want = np.repeat(rows(eng, [alone], toks[:1]), members, 0)
        assert off(got, want) <= REL_CUT["bfloat16"]
        kept.append(sorted(k[0] for k in eng._decoder.graphs if len(k) > 2))
    assert kept == [[2], [2, 3], [3, 4], [3, 4], [2, 4], [2, 5], [2, 5], [3, 5], [2, 3]]
    assert [k for k in eng._decoder.graphs if len(k) == 2] == [(1, 8)]
    eng.check_status()
