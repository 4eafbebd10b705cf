"""Captured decode steps of forked sequences: which are kept under who shares pages, and that those run the kernel for shared pages."""
import pytest

import test_beam_gpu
from helpers import REL_CUT, random_ids
from test_beam_gpu import off, rows

pytestmark = pytest.mark.gpu
dirs = test_beam_gpu.dirs


def test_steps_that_read_their_pages_apart_are_kept_as_any_other(dirs):
    """Twelve members of four heads per kv head stand in tiles of more than 32 rows, where shared pages have to be many: one captured step serves the forks
    and sequences of their own, whoever shares how much."""
    from ithaca_b200 import Engine
    eng = Engine(dirs("wide"), dtype="bfloat16", max_tokens=64 * 300, max_slots=24)
    a = eng.alloc_slot()
    eng.step([a], [random_ids(700, 300, 5)], None)
    slots = [a] + eng.fork_slot(a, 11)
    for n in range(3):
        eng._decoder.step(slots, [[(5 * i + n) % 300] for i in range(12)])
    assert [len(key) for key in eng._decoder.graphs] == [2]
    eng._settle()
    for s in slots[6:]:
        eng.free_slot(s)
    b = eng.alloc_slot()
    eng.step([b], [random_ids(640, 300, 6)], None)
    slots = slots[:6] + [b] + eng.fork_slot(b, 5)
    got = eng._decoder.step(slots, [[3]] * 12)[0].float().cpu().numpy()
    assert [len(key) for key in eng._decoder.graphs] == [2]
    alone = [eng.alloc_slot() for _ in range(2)]
    eng.step(alone[:1], [random_ids(700, 300, 5)], None)
    for n in range(3):
        eng.step(alone[:1], [[n % 300]], None)
    eng.step(alone[1:], [random_ids(640, 300, 6)], None)
    want = rows(eng, alone, [[3], [3]])
    assert off(got[[0, 6]], want) <= REL_CUT["bfloat16"]
    eng.check_status()


def test_a_captured_step_runs_the_kernel_for_shared_pages(dirs, monkeypatch):
    """Eager pass and capture call it, with room for more groups than there are; replays call nothing."""
    from ithaca_b200 import Engine
    from ithaca_b200.csrc import attention_bf16
    calls, run = [], attention_bf16.decode_shared
    monkeypatch.setattr(attention_bf16, "decode_shared", lambda *a, **k: (calls.append(a[7:11]), run(*a, **k))[1])
    eng = Engine(dirs("wide"), dtype="bfloat16", max_tokens=64 * 200, max_slots=24)
    slots = []
    for i, n in enumerate((1500, 1400, 1450)):
        a = eng.alloc_slot()
        eng.step([a], [random_ids(n, 300, n)], None)
        slots += [a] + eng.fork_slot(a, 3)
    key = (12, 24, (4, 4, 32, 1))
    for n in range(3):
        calls.clear()
        had = key in eng._decoder.graphs
        eng._decoder.step(slots, [[i] for i in range(12)])
        assert had == (n > 0) and list(eng._decoder.graphs) == [key]
        assert calls == ([] if had else [(4, 4, 32, 1)] * 4)                       # two layers, run and captured
    # eleven of them: another step
    calls.clear()
    eng._decoder.step(slots[:11], [[i] for i in range(11)])
    assert calls == [(4, 4, 32, 1)] * 4 and len(eng._decoder.graphs) == 2
    eng.check_status()


def test_a_profile_of_a_step_of_forked_sequences(dirs, monkeypatch):
    """The kernel is in the table with its calls; bytes count a shared page once."""
    from ithaca_b200 import Engine
    from ithaca_b200.csrc import attention_bf16
    monkeypatch.setattr(attention_bf16, "sharing_pays", lambda *a: True)
    eng = Engine(dirs("wide"), dtype="bfloat16", max_tokens=64 * 100, max_slots=8)
    a = eng.alloc_slot()
    eng.step([a], [random_ids(1930, 300, 5)], None)
    slots = [a] + eng.fork_slot(a, 3)
    logits, table = eng.profile_step(slots, [[5]] * 4)
    (row,) = [r for r in table if r["kernel"].startswith("attention decode shared")]
    keys = 30 * 64 + 4 * (1931 - 30 * 64)                                  # thirty shared pages, each one's own keys
    assert row["calls"] == 2 and row["us"] > 0 and row["bytes"] == 2 * (2 * 4 * 512 * 2 + keys * 2 * 2 * 64 * 2) and row["flops"] == 2 * 4 * 64 * 8 * 4 * 1931
    alone = eng.alloc_slot()
    eng.step([alone], [random_ids(1930, 300, 5)], None)
    assert off(logits.float().cpu().numpy()[:1], rows(eng, [alone], [[5]])) <= REL_CUT["bfloat16"]
