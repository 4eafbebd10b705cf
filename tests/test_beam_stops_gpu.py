"""A search with more beams and stop tokens than one choice gives, through the engine: against the definition over the plain model."""
import pytest

import test_beam_gpu
from helpers import random_ids
from test_beam_gpu import PlainModel
from test_beam_stops_cpu import defined

pytestmark = pytest.mark.gpu
dirs = test_beam_gpu.dirs


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("K,stops", [(16, [125, 111, 57]), (9, [125, 111, 57, 200, 31]), (16, list(range(100, 116)))])
def test_the_search_matches_plain_float32(dirs, K, stops, graphs):
    from ithaca_b200 import Engine
    d = dirs("A")
    eng, plain = Engine(d, dtype="float32", max_tokens=64 * 80, graphs=graphs), PlainModel(d)
    prompts = [random_ids(n, 256, 40 + n) for n in (5, 62)]
    got = eng.beam_search(prompts, beams=K, max_tokens=4, n_best=K, stop_token_ids=stops)
    for p, hyps in zip(prompts, got):
        want = defined(plain, p, K, 4, set(stops))
        assert [(h.tokens, h.stopped) for h in hyps] == [(t, stop) for _, t, stop in want]
        assert [h.score for h in hyps] == pytest.approx([s for s, _, _ in want], abs=1e-3)
    assert eng.cache.table.n_slots_in_use() == 0 and all(p.held() == 0 for p in eng.cache.table.pools)
