"""Forked slots and shared pages in the cache's books, who shares pages in a step, and the search's decisions: no device."""
import array
import itertools
import math
import random

import numpy as np
import pytest

from ithaca_b200.cache import CacheError, CacheFull, KVGroupLayout, KVRequest, PagePool, SequenceCache, SlotTable, StateRequest
from ithaca_b200.csrc.ops import KernelError, copy_moves
from ithaca_b200.engine.beam import BeamOptions, beam_loop, ranked
from ithaca_b200.engine.context import find_sharing


# -- pages ---------------------------------------------------------------------------------------------------------------
def test_a_page_is_free_when_its_last_holder_gives_it_back():
    pool = PagePool(3)
    p = pool.take()
    pool.share(p)
    pool.share(p)
    assert pool.holders(p) == 3 and pool.n_shared == 1 and pool.held() == 1 and pool.n_free == 2
    pool.give_back(p)
    assert pool.n_shared == 1
    pool.give_back(p)
    assert pool.n_shared == 0 and pool.n_free == 2
    pool.give_back(p)
    assert pool.n_free == 3
    for bad in (lambda: pool.give_back(p), lambda: pool.share(p), lambda: pool.share(3), lambda: pool.holders(-1)):
        with pytest.raises(CacheError):
            bad()


def test_many_pages_at_once():
    pool = PagePool(6)
    pages = np.array([pool.take() for _ in range(4)], dtype=np.int32)
    pool.share_all(pages[1:3])
    pool.share_all(pages[:0])
    assert pool.n_shared == 2 and [pool.holders(int(p)) for p in pages] == [1, 2, 2, 1]
    pool.give_back_all(pages[[3, 1, 0]])
    assert pool.n_shared == 1 and pool.n_free == 4 and [pool.take(), pool.take()] == [pages[0], pages[3]]        # the last given back comes first
    for bad in (lambda: pool.share_all(np.array([4])), lambda: pool.give_back_all(np.array([1, 5])), lambda: pool.give_back_all(np.array([6])), lambda: pool.share_all(np.array([-1]))):
        before = pool._holders.copy(), list(pool._free), pool.n_shared
        with pytest.raises(CacheError):
            bad()
        assert (pool._holders == before[0]).all() and pool._free == before[1] and pool.n_shared == before[2]


def table(n_pages=12, slots=6, window=None):
    return SlotTable([KVGroupLayout(2, 16, None, (0, 1)), KVGroupLayout(1, 8, window, (2,))], [n_pages, n_pages], slots, 64)


def grow(t, s, n):
    t.reserve(s, n)
    t.commit(s, n)


def test_a_fork_shares_full_pages_and_copies_the_begun_one():
    t = table()
    a = t.alloc_slot()
    grow(t, a, 150)
    made, copies = t.fork([(a, 2)])
    b, c = made[0]
    assert (t.length[[b, c]] == 150).all() and t.pools[0].n_free == 12 - 3 - 2
    for g in range(2):
        row = t.tables[g]
        assert (row[b, :2] == row[a, :2]).all() and (row[c, :2] == row[a, :2]).all() and len({row[a, 2], row[b, 2], row[c, 2]}) == 3
        assert copies[g] == [(row[a, 2], row[b, 2], 22), (row[a, 2], row[c, 2], 22)]
    t.check_consistent()
    grow(t, b, 100)                                                # it goes on in pages of its own
    assert (t.tables[0][b, 2:4] >= 0).all() and t.length[a] == 150
    t.check_consistent()
    t.free_slot(a)
    assert t.pools[0].holders(int(t.tables[0][b, 0])) == 2
    t.check_consistent()
    t.free_slot(c)
    t.free_slot(b)
    assert all(p.n_free == 12 and p.n_shared == 0 for p in t.pools)
    t.check_consistent()


@pytest.mark.parametrize("length", [0, 1, 64, 128])
def test_forks_of_empty_and_of_whole_pages(length):
    t = table()
    a = t.alloc_slot()
    if length:
        grow(t, a, length)
    made, copies = t.fork([(a, 1), (a, 0)])
    assert made == [[made[0][0]], []] and [len(c) for c in copies] == [1 if length % 64 else 0] * 2
    t.check_consistent()
    grow(t, made[0][0], 5)
    grow(t, a, 5)
    t.check_consistent()
    assert t.tables[0][a, length // 64] != t.tables[0][made[0][0], length // 64]


def test_a_fork_is_refused_whole():
    t = table(n_pages=5, slots=4)
    a = t.alloc_slot()
    grow(t, a, 100)
    before = [x.copy() for x in t.tables]
    for wanted, kind in ([(a, 4)], CacheFull), ([(a, -1)], CacheError), ([(3, 1)], CacheError), ([(a, 1), (9, 1)], CacheError):
        with pytest.raises(kind):
            t.fork(wanted)
    b = t.alloc_slot()
    grow(t, b, 128)
    with pytest.raises(CacheFull):                                  # two slots are free, one page is
        t.fork([(a, 2)])
    t.free_slot(b)
    assert all((x == y).all() for x, y in zip(before, t.tables)) and t.n_slots_in_use() == 1
    t.check_consistent()


def test_a_cut_inside_a_shared_page_gives_a_page_of_its_own():
    t = table()
    a = t.alloc_slot()
    grow(t, a, 200)
    (b,), = t.fork([(a, 1)])[0]
    copies = t.truncate(b, 70)
    assert copies[0] == [(t.tables[0][a, 1], t.tables[0][b, 1], 6)] and t.tables[0][b, 1] != t.tables[0][a, 1] and t.tables[0][b, 0] == t.tables[0][a, 0]
    assert (t.tables[0][b, 2:] == -1).all() and t.length[a] == 200
    t.check_consistent()
    grow(t, b, 200)
    t.check_consistent()
    assert not set(t.tables[0][b, 1:5].tolist()) & set(t.tables[0][a, :4].tolist())
    assert t.truncate(a, 128) == [[], []]                           # page 2 and 3 are a's own again: kept for reuse
    assert t.tables[0][a, 2] >= 0
    t.check_consistent()
    t.truncate(a, 0)
    t.truncate(b, 64)
    t.check_consistent()


def test_a_cut_that_needs_a_page_no_longer_there_is_refused():
    t = SlotTable([KVGroupLayout(2, 16, None, (0,))], [3], 4, 64)
    a = t.alloc_slot()
    grow(t, a, 128)
    (b,), = t.fork([(a, 1)])[0]
    grow(t, a, 1)
    with pytest.raises(CacheFull):
        t.truncate(b, 100)
    assert t.length[b] == 128
    t.check_consistent()
    t.truncate(b, 64)
    t.check_consistent()


def test_windows_release_shared_pages_one_holder_at_a_time():
    t = table(window=70)
    a = t.alloc_slot()
    grow(t, a, 130)
    (b,), = t.fork([(a, 1)])[0]
    t.check_consistent()
    for _ in range(100):
        grow(t, b, 1)
    assert t.tables[1][b, 1] == -1 and t.tables[1][a, 1] >= 0
    t.check_consistent()
    for _ in range(100):
        grow(t, a, 1)
    t.check_consistent()
    t.free_slot(a)
    t.free_slot(b)
    assert all(p.n_free == 12 for p in t.pools)


def test_random_traffic_with_forks_keeps_the_books():
    rng = random.Random(0)
    t = SlotTable([KVGroupLayout(2, 16, None, (0,)), KVGroupLayout(1, 32, 100, (1,))], [60, 60], 10, 64)
    live = []
    for step in range(3000):
        r = rng.random()
        try:
            if r < 0.1 or not live:
                live.append(t.alloc_slot())
            elif r < 0.25:
                made, copies = t.fork([(s, rng.randint(0, 2)) for s in rng.sample(live, min(len(live), 2))])
                live += [s for m in made for s in m]
                for g, moves in enumerate(copies):
                    src, dst = {m[0] for m in moves}, [m[1] for m in moves]
                    assert len(set(dst)) == len(dst) and not src & set(dst)
            elif r < 0.4:
                t.free_slot(live.pop(rng.randrange(len(live))))
            elif r < 0.55:
                s = rng.choice(live)
                t.truncate(s, rng.randint(0, int(t.length[s])))
            else:
                s = rng.choice(live)
                n = rng.choice([1, 1, 1, 7, 64, 150])
                if t.length[s] + n < 600:
                    # what is written is this slot's alone
                    t.reserve(s, n)
                    for g, grp in enumerate(t.kv_groups):
                        for c in range(int(t.length[s]) // 64, int(t.length[s] + n - 1) // 64 + 1):
                            assert t.pools[g].holders(int(t.tables[g][s, c])) == 1
                    t.commit(s, n)
        except (CacheFull, CacheError) as e:
            assert isinstance(e, CacheFull) or "released" in str(e)
        t.check_consistent()
    for s in live:
        t.free_slot(s)
    assert all(p.n_free == 60 and p.n_shared == 0 for p in t.pools)


def test_the_cache_forks_without_a_device():
    c = SequenceCache({0: [KVRequest(2, 16)], 1: [StateRequest("s", (3,))]}, max_tokens=640, max_slots=4, device=None)
    a = c.alloc_slot()
    c.reserve([a], [70])
    c.commit([a], [70])
    assert c.fork([(a, 2)]) == [[1, 2]] and c.length(2) == 70
    with pytest.raises(CacheError, match="fixed-size"):
        c.truncate(1, 10)


def test_a_fork_whose_copies_fail_changes_nothing(monkeypatch):
    c = SequenceCache({0: [KVRequest(2, 16)]}, max_tokens=640, max_slots=4, device=None)
    a = c.alloc_slot()
    c.reserve([a], [70])
    c.commit([a], [70])
    free = [p.n_free for p in c.table.pools]
    def fail(*a):
        raise KernelError("lost")
    monkeypatch.setattr(c, "_copy", fail)
    with pytest.raises(KernelError, match="lost"):
        c.fork([(a, 2)])
    assert c.table.n_slots_in_use() == 1 and [p.n_free for p in c.table.pools] == free and c.table.pools[0].n_shared == 0
    c.table.check_consistent()


def test_lists_of_moves_are_checked():
    assert copy_moves([1, 1], (2, 3), [4, 0], 4, 64) == [1, 2, 4, 1, 3, 0] and copy_moves([1, 0], [2, 3], None, 4, 1) == [1, 2, 1, 0, 3, 1]
    assert copy_moves([], [], None, 4, 1) == []
    for bad in (([0], [1, 2], None), ([0], [4], None), ([-1], [1], None), ([0, 1], [2, 2], None), ([0, 1], [1, 2], None), ([3], [3], None), ([0], [1], [65]), ([0], [1], [-1]),
                ([0], [1], [1, 2])):
        with pytest.raises(KernelError):
            copy_moves(*bad, 4, 64)


def test_a_job_of_more_blocks_than_a_launch_has_is_refused_before_anything_runs():
    """On the host: 4 rows' segments of two bytes each in 2^30 entries, or twice as many positions; nothing is read or launched."""
    from ithaca_b200.csrc import ops
    lib = ops._search_lib()
    moves = array.array("i", [0, 1, 1])
    for job in ([16, 1 << 30, 8, 2, 4, 4, 2, 2, 0, 1], [16, 0x7fffffff, 8, 2, 4, 2, 2, 2, 0, 1]):
        j = array.array("q", job)
        assert lib.ik_copy_rows(j.buffer_info()[0], 1, moves.buffer_info()[0], 1, None) == -2
    j = array.array("q", [16, 1 << 31, 8, 2, 4, 4, 2, 2, 0, 1])
    assert lib.ik_copy_rows(j.buffer_info()[0], 1, moves.buffer_info()[0], 1, None) == -1


# -- who shares pages ------------------------------------------------------------------------------------------------------
def rows(*lists):
    n = max(len(x) for x in lists)
    return np.array([list(x) + [-1] * (n - len(x)) for x in lists], dtype=np.int32)


def test_groups_of_neighbours():
    s = find_sharing(rows([1, 2, 3], [1, 2, 4], [1, 2, 5, 6], [9], [7, 8], [7, 10]), [3, 3, 4, 1, 2, 2])
    assert s.starts == [0, 3, 4, 6] and s.pages == [2, 2, 2, 0, 1, 1] and (s.shared_bound, s.own_bound, s.n_groups, s.max_members) == (2, 2, 3, 3)
    assert find_sharing(rows([1], [2], [3]), [1, 1, 1]) is None and find_sharing(rows([1, 2]), [2]) is None
    assert find_sharing(rows([-1, -1], [-1, -1]), [2, 2]) is None                 # no page is no shared page
    assert find_sharing(rows([1, 2, 3], [4, 2, 3]), [3, 3]) is None               # a prefix, not what comes later
    # one page in common to all, many within the pairs: the pairs save more
    s = find_sharing(rows([1, 2, 3, 4, 10], [1, 2, 3, 4, 11], [1, 5, 6, 7, 12], [1, 5, 6, 7, 13]), [5] * 4)
    assert s.starts == [0, 2, 4] and s.pages == [4] * 4
    # the other way round
    s = find_sharing(rows([1, 2, 3, 4, 10], [1, 2, 3, 4, 11], [1, 2, 3, 7, 12], [1, 2, 3, 7, 13]), [5] * 4)
    assert s.starts == [0, 4] and s.pages == [3] * 4 and s.own_bound == 2


def test_a_captured_step_keeps_room_for_other_groups():
    from ithaca_b200.engine.graph import _sharing_shape
    s = find_sharing(rows([1, 2, 3], [1, 2, 4], [1, 2, 5, 6], [9], [7, 8], [7, 10]), [3, 3, 4, 1, 2, 2])
    assert _sharing_shape(s) == (4, 4, 2, 2) and _sharing_shape(None) is None
    s.pad(4)
    assert s.starts == [0, 3, 4, 6, 6] and s.n_groups == 4 and s.max_members == 3 and _sharing_shape(s) == (4, 4, 2, 2)
    s = find_sharing(rows([1, 2], [1, 3], [1, 4]), [2, 2, 2])
    assert _sharing_shape(s) == (1, 3, 1, 1)                                       # never more than there are sequences


def test_long_runs_are_cut_as_well_as_every_way():
    """Many neighbours: against the plain search over every last cut."""
    from ithaca_b200.engine.context import _cut_run
    rng = random.Random(2)
    for _ in range(300):
        c = [rng.randint(1, rng.choice([2, 4, 40])) for _ in range(rng.randint(1, 14)) for _ in range(rng.choice([1, 1, 3]))]
        best = [0]
        for j in range(1, len(c) + 2):
            best.append(max(best[i] + (j - 1 - i) * min(c[i:j - 1], default=0) for i in range(j)))
        groups = _cut_run(c)
        assert [a for a, _, _ in groups] == [0] + [b for _, b, _ in groups][:-1] and groups[-1][1] == len(c) + 1
        assert all(s == min(c[a:b - 1], default=0) for a, b, s in groups) and sum((b - a - 1) * s for a, b, s in groups) == best[-1]
    assert _cut_run([7] * 500) == [(0, 501, 7)] and _cut_run([]) == [(0, 1, 0)]


def test_groups_save_the_most_page_readings():
    def saved(common, starts):
        return sum((b - a - 1) * min(common[a:b - 1]) for a, b in zip(starts, starts[1:]) if b - a > 1)
    rng = random.Random(1)
    for _ in range(200):
        B = rng.randint(2, 7)
        common = [rng.choice([0, 0, 1, 2, 5]) for _ in range(B - 1)]
        t, fresh = [[0] * 6], itertools.count(100)
        t[0] = [next(fresh) for _ in range(6)]
        for c in common:
            t.append(t[-1][:c] + [next(fresh) for _ in range(6 - c)])
        s = find_sharing(np.array(t, dtype=np.int32), [6] * B)
        best = max(saved(common, [0] + list(cut) + [B]) for n in range(B) for cut in itertools.combinations(range(1, B), n))
        assert (saved(common, s.starts) if s else 0) == best
        if s:
            for a, b in zip(s.starts, s.starts[1:]):
                assert all(s.pages[i] <= (min(common[a:b - 1]) if b - a > 1 else 0) for i in range(a, b))


# -- the search ------------------------------------------------------------------------------------------------------------
class Backend:
    """A made-up model over a small vocabulary: the log probabilities behind a sequence are a function of its tokens alone."""

    def __init__(self, vocab, seed, n_slots=64, context_length=1000, ties=False):
        self.vocab, self.seed, self.context_length, self.ties = vocab, seed, context_length, ties
        self.free, self.held, self.steps, self.forks = list(range(n_slots)), {}, [], 0

    def logp(self, tokens):
        r = random.Random(f"{self.seed} {tokens}")
        x = [r.choice([0.0, 1.0]) if self.ties else r.gauss(0, 1.5) for _ in range(self.vocab)]
        top = max(x)
        z = top + math.log(sum(math.exp(v - top) for v in x))
        return [v - z for v in x]

    def free_slots(self): return len(self.free)
    def room_for_beams(self, prompts, grown, beams): return True

    def alloc_slot(self):
        s = self.free.pop()
        self.held[s] = []
        return s

    def free_slot(self, s):
        del self.held[s]
        self.free.append(s)

    def fork_slots(self, wanted):
        assert len({s for s, _ in wanted}) == len(wanted)
        out = []
        for s, n in wanted:
            out.append([self.alloc_slot() for _ in range(n)])
            for new in out[-1]:
                self.held[new] = list(self.held[s])
            self.forks += n
        return out

    def step_and_select(self, slots, tokens, scores, n_out):
        assert len(set(slots)) == len(slots) == sum(len(s) for s in scores)
        self.steps.append([len(s) for s in scores])
        for s, t in zip(slots, tokens):
            self.held[s] += t
        out, at = [], 0
        for sums in scores:
            cand = [(-(c + lp), b, v) for b, c in enumerate(sums) for v, lp in enumerate(self.logp(self.held[slots[at + b]]))]
            out.append([(-s, b, v) for s, b, v in sorted(cand)[:n_out]])
            at += len(sums)
        return out


def reference(model, prompt, K, max_tokens, stops, penalty, early=False):
    """The search by its definition, over whole sequences."""
    live, done = [(0.0, [])], []
    n_out = min(32, K * (1 + len(stops)))
    for length in range(1, max_tokens + 1):
        cand = sorted(((-(s + lp), i, v) for i, (s, t) in enumerate(live) for v, lp in enumerate(model.logp(prompt + t))))[:n_out]
        nxt = []
        for rank, (s, i, v) in enumerate(cand):
            if v in stops:
                if rank < K:
                    done.append((-s / length ** penalty, -s, live[i][1], True))
            elif len(nxt) < K:
                nxt.append((-s, live[i][1] + [v]))
        done = sorted(done, key=lambda d: -d[0])[:K]
        live = nxt
        if not live:
            return done
        if length == max_tokens:
            return sorted(done + [(s / length ** penalty, s, t, False) for s, t in live], key=lambda d: -d[0])[:K]
        if len(done) >= K and (early or live[0][0] / length ** penalty <= done[-1][0]):
            return done
    return done


@pytest.mark.parametrize("K", [1, 2, 4, 7])
@pytest.mark.parametrize("stops,penalty,early", [((), 1.0, False), ((3,), 1.0, False), ((3, 5), 0.0, False), ((0,), 2.0, True), ((1, 2, 3), 0.6, True)])
@pytest.mark.parametrize("vocab", [8, 40])
def test_the_search_is_the_one_that_is_defined(K, stops, penalty, early, vocab):
    be = Backend(vocab, 5)
    prompts = [[1, 2, 3], [4], [5, 6], [7] * 4]
    got, st = beam_loop(prompts, BeamOptions(beams=K, max_tokens=9, length_penalty=penalty, n_best=K, early_stopping=early), be, stop_token_ids=stops)
    for p, hyps in zip(prompts, got):
        want = reference(be, p, K, 9, stops, penalty, early)
        assert [(h.tokens, h.stopped) for h in hyps] == [(t, stop) for _, _, t, stop in want]
        for h, (score, logprob, _, _) in zip(hyps, want):
            assert h.score == pytest.approx(score, rel=1e-12) and h.logprob == pytest.approx(logprob, rel=1e-12)
    assert be.held == {} and st.prompt_tokens == 10 and st.batches == 1


def test_equal_candidates_and_more_requests_than_slots():
    be = Backend(6, 2, n_slots=7, ties=True)
    prompts = [[i] for i in range(5)]
    got, st = beam_loop(prompts, BeamOptions(beams=3, max_tokens=5, n_best=3), be, stop_token_ids=(2,))
    assert st.batches == 3 and be.held == {}
    for p, hyps in zip(prompts, got):
        assert [h.tokens for h in hyps] == [t for _, _, t, _ in reference(be, p, 3, 5, (2,), 1.0)]


def test_fewer_candidates_than_beams():
    """A vocabulary smaller than the number of beams: the first steps have fewer beams than asked for, and requests of unequal counts run side by side."""
    be = Backend(3, 4)
    got, _ = beam_loop([[1], [2, 2]], BeamOptions(beams=8, max_tokens=4, n_best=8), be, stop_token_ids=(0,))
    for p, hyps in zip([[1], [2, 2]], got):
        assert [h.tokens for h in hyps] == [t for _, _, t, _ in reference(be, p, 8, 4, (0,), 1.0)]
    assert be.steps[0] == [1, 1] and be.steps[1] == [2, 2] and be.held == {}


def test_stop_tokens_and_budgets():
    be = Backend(8, 1)
    with_stop = beam_loop([[1]], BeamOptions(beams=4, max_tokens=8, n_best=4, include_stop=True), be, stop_token_ids=(3,))[0][0]
    without = beam_loop([[1]], BeamOptions(beams=4, max_tokens=8, n_best=4), be, stop_token_ids=(3,))[0][0]
    for a, b in zip(with_stop, without):
        assert a.tokens == b.tokens + ([3] if b.stopped else []) and a.score == b.score
    assert beam_loop([[1]], BeamOptions(beams=2, max_tokens=8, stop_token_ids=()), be, stop_token_ids=(3,))[0][0][0].stopped is False
    assert beam_loop([[1], [2]], BeamOptions(max_tokens=0), be)[0] == [[], []]
    short = Backend(8, 1, context_length=4)
    assert [len(h[0].tokens) for h in beam_loop([[1], [1, 2, 3, 4], [1, 2, 3]], BeamOptions(beams=2, max_tokens=8), short)[0] if h] == [3, 1]
    assert short.held == {}


def test_the_search_refuses():
    be = Backend(8, 1)
    for bad in (dict(beams=0), dict(beams=17), dict(n_best=0), dict(n_best=5), dict(length_penalty=-1.0), dict(length_penalty=math.nan), dict(length_penalty=math.inf),
                dict(length_penalty=200.0)):
        with pytest.raises(ValueError):
            beam_loop([[1]], BeamOptions(**bad), be)
    for prompts in ([[]], [[1] * 1001]):
        with pytest.raises(ValueError):
            beam_loop(prompts, BeamOptions(), be)
    with pytest.raises(RuntimeError, match="does not fit"):
        beam_loop([[1]], BeamOptions(beams=4), Backend(8, 1, n_slots=3))
    assert be.held == {}


def test_a_step_that_fails_leaves_no_slot_behind():
    be = Backend(8, 1)
    run = be.step_and_select
    def fail(*a):
        if len(be.steps) == 3:
            raise RuntimeError("lost")
        return run(*a)
    be.step_and_select = fail
    with pytest.raises(RuntimeError, match="lost"):
        beam_loop([[1], [2]], BeamOptions(beams=3, max_tokens=9), be)
    assert be.held == {}


def test_ranks():
    assert ranked(-6.0, 3, 1.0) == -2.0 and ranked(-6.0, 3, 0.0) == -6.0 and ranked(-6.0, 0, 1.0) == -6.0


# heads, kv heads, head size, groups, members, shared, own pages: us of decode, of decode_shared as measured on B200
MEASURED = [(32, 8, 128, 1, 2, 16, 1, 8.6, 10.0), (32, 8, 128, 1, 4, 8, 1, 9.2, 10.4), (32, 8, 128, 1, 4, 48, 1, 16.1, 11.9), (32, 8, 128, 4, 2, 8, 1, 11.2, 10.0),
            (32, 8, 128, 4, 8, 2, 1, 10.8, 11.6), (32, 8, 128, 4, 8, 4, 4, 18.2, 15.9), (32, 8, 128, 4, 8, 2, 4, 15.3, 18.2), (32, 8, 128, 4, 16, 2, 1, 19.1, 15.0),
            (32, 8, 128, 4, 16, 4, 4, 29.5, 32.2), (32, 8, 128, 4, 16, 8, 4, 38.7, 27.8), (32, 8, 128, 16, 4, 48, 4, 127.3, 54.6), (32, 8, 64, 1, 8, 4, 1, 7.6, 9.3),
            (32, 8, 64, 1, 4, 48, 1, 12.6, 9.7), (32, 8, 64, 4, 16, 8, 1, 21.8, 13.7), (32, 8, 64, 16, 8, 16, 4, 65.6, 30.1), (40, 40, 128, 1, 2, 1, 1, 6.7, 8.6),
            (40, 40, 128, 1, 4, 8, 1, 17.0, 10.1), (40, 40, 128, 4, 16, 48, 1, 529.3, 61.8), (40, 40, 128, 16, 8, 16, 4, 458.0, 161.5)]


@pytest.mark.parametrize("nh,nkv,hd,groups,members,shared,own,apart,together", MEASURED)
def test_shared_pages_are_read_once_where_that_was_measured_faster(nh, nkv, hd, groups, members, shared, own, apart, together):
    from ithaca_b200.csrc.attention_bf16 import sharing_pays
    assert sharing_pays(groups * members, groups, members, shared, own, nh, nkv, hd) == (together < apart)


def test_steps_that_are_too_large_for_one_launch_read_their_pages_apart():
    from ithaca_b200.csrc.attention_bf16 import sharing_pays
    assert sharing_pays(1024, 64, 16, 50, 1, 32, 8, 128) and not sharing_pays(1040, 65, 16, 50, 1, 32, 8, 128) and not sharing_pays(1024, 512, 2, 50, 1, 320, 1, 128)
