"""The search where many stop tokens are likely: beams go on as long as anything can go on."""
import math

import pytest

from ithaca_b200.engine.beam import BeamOptions, beam_loop, joined
from test_beam_cpu import Backend


class Stopping(Backend):
    """Stop tokens are far more likely than the others."""

    def __init__(self, vocab, seed, stops, by=6.0, **kw):
        super().__init__(vocab, seed, **kw)
        self.stops, self.by, self.asked = stops, by, []

    def logp(self, tokens):
        x = super().logp(tokens)
        x = [v + self.by if i in self.stops else v for i, v in enumerate(x)]
        z = math.log(sum(math.exp(v) for v in x))
        return [v - z for v in x]

    def step_and_select(self, slots, tokens, scores, n_out):
        assert n_out <= 32                           # what the kernel gives
        self.asked.append((len(scores), n_out))
        return super().step_and_select(slots, tokens, scores, n_out)


def defined(model, prompt, K, max_tokens, stops):
    """The search by its definition, every candidate of a step looked at: the K best that are no stop tokens go on, stop tokens among the K best of all end."""
    live, done = [(0.0, [])], []
    for length in range(1, max_tokens + 1):
        cand = sorted((-(s + lp), i, v) for i, (s, t) in enumerate(live) for v, lp in enumerate(model.logp(prompt + t)))
        done += [(-s / length, live[i][1], True) for s, i, v in cand[:K] if v in stops]
        done = sorted(done, key=lambda d: -d[0])[:K]
        live = [(-s, live[i][1] + [v]) for s, i, v in cand if v not in stops][:K]
        if not live:
            return done
        if length == max_tokens:
            return sorted(done + [(s / length, t, False) for s, t in live], key=lambda d: -d[0])[:K]
        if len(done) >= K and live[0][0] / length <= done[-1][0]:
            return done
    return done


@pytest.mark.parametrize("K,stops", [(16, (3, 5, 7)), (16, (0, 1)), (8, (2, 4, 6, 8, 10)), (16, tuple(range(16))), (4, tuple(range(20, 40))), (16, (3,)), (4, (1, 2, 3))])
@pytest.mark.parametrize("by", [6.0, 1.0, -1.0])
def test_stop_tokens_do_not_crowd_out_what_goes_on(K, stops, by):
    be = Stopping(60, 9, set(stops), by)
    prompts = [[1, 2], [3], [5, 50, 5]]
    got, st = beam_loop(prompts, BeamOptions(beams=K, max_tokens=5, n_best=K), be, stop_token_ids=stops)
    for p, hyps in zip(prompts, got):
        want = defined(be, p, K, 5, set(stops))
        assert [(h.tokens, h.stopped) for h in hyps] == [(t, stop) for _, t, stop in want]
        assert [h.score for h in hyps] == pytest.approx([s for s, _, _ in want], rel=1e-12)
    assert be.held == {}


def test_few_stop_tokens_are_asked_for_as_before():
    be = Stopping(60, 9, {3})
    beam_loop([[1], [2]], BeamOptions(beams=4, max_tokens=3), be, stop_token_ids=(3,))
    assert be.asked[0] == (2, 8) and all(n == 8 for _, n in be.asked)


def test_choices_of_single_beams_are_joined_in_order():
    lists = [[(-1.0, 0, 4), (-2.0, 0, 9), (-2.0, 0, 3)], [], [(-1.0, 0, 1), (-1.5, 0, 0)]]
    assert joined(lists) == [(-1.0, 0, 4), (-1.0, 2, 1), (-1.5, 2, 0), (-2.0, 0, 9), (-2.0, 0, 3)]


def test_more_stop_tokens_than_choices_are_refused():
    for K, n in ((16, 17), (4, 29), (1, 32)):
        be = Stopping(60, 9, set(range(n)))
        with pytest.raises(ValueError, match="stop tokens"):
            beam_loop([[1]], BeamOptions(beams=K, max_tokens=3), be, stop_token_ids=range(n))
        assert be.held == {} and be.steps == []
        beam_loop([[1]], BeamOptions(beams=K, max_tokens=3), be, stop_token_ids=range(n - 1))
