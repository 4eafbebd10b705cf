"""Forked slots, steps whose sequences share pages, and the search over beams through the engine, against plain forms and against the same tokens
fed to slots of their own."""
import math

import numpy as np
import pytest
import torch

import test_gunenex_gpu
import test_mimadra_gpu
import test_tiralix_gpu
import test_vebisun_gpu
import test_vovalorn_gpu
import test_zomipel_gpu
from helpers import REL, REL_CUT, load_plain, random_ids
from plain import llama_plain as P
from test_beam_cpu import reference
from tiny import TINY, make_model_dir

pytestmark = pytest.mark.gpu

WIDE = {    # heads of 64 in groups of 4, a context of several pages
    "architectures": ["LlamaForCausalLM"], "hidden_size": 256, "num_hidden_layers": 2, "num_attention_heads": 8, "num_key_value_heads": 2, "head_dim": 64, "intermediate_size": 256,
    "vocab_size": 300, "rope_theta": 10000.0, "rope_scaling": None, "rms_norm_eps": 1e-5, "max_position_embeddings": 2048, "tie_word_embeddings": False,
    "torch_dtype": "bfloat16", "eos_token_id": 7}


def model_dir(root, name):
    if name in TINY:
        return make_model_dir(root, TINY[name], seed=31)
    if name == "wide":
        return make_model_dir(root, WIDE, seed=32)
    m = {"vebisun": test_vebisun_gpu, "tiralix": test_tiralix_gpu, "mimadra": test_mimadra_gpu, "gunenex": test_gunenex_gpu, "zomipel": test_zomipel_gpu,
         "vovalorn": test_vovalorn_gpu}[name.split()[0]]
    cfg = getattr(m, "CFG_" + (name.split() + ["A"])[1])
    if name.startswith("vebisun"):
        return m._write(str(root), cfg, 3)
    return m._write(str(root), cfg, m.make_tensors(cfg, 3), "beams_" + name.replace(" ", "_"))


@pytest.fixture(scope="module")
def dirs(tmp_path_factory):
    root, made = tmp_path_factory.mktemp("beam_models"), {}
    def get(name):
        if name not in made:
            made[name] = model_dir(root, name)
        return made[name]
    return get


def rows(eng, slots, tokens):
    return eng.step(slots, tokens, "last").float().cpu().numpy()


def off(a, b):
    return float(np.abs(a - b).max() / np.abs(b).max())


MODELS = ["A", "B", "C", "wide", "vebisun", "vebisun B", "tiralix", "tiralix B", "mimadra", "mimadra B", "mimadra C", "gunenex", "gunenex B", "gunenex C", "zomipel", "zomipel B",
          "zomipel C", "vovalorn", "vovalorn B", "vovalorn C"]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", MODELS)
def test_forked_sequences_go_on_as_if_fed_alone(dirs, name, dtype, monkeypatch):
    """A prompt is fed once and forked twice; each of the three goes on with tokens of its own, one at a time and in a run.  Slots that were fed the
    same tokens in the same steps give the same logits to the last bit, as long as the same kernels run (the one for shared pages rounds otherwise,
    and where experts are chosen a rounding may choose others: it is left out here)."""
    from ithaca_b200 import Engine
    from ithaca_b200.csrc import attention_bf16
    monkeypatch.setattr(attention_bf16, "sharing_pays", lambda *a: False)
    eng = Engine(dirs(name), dtype=dtype, max_tokens=64 * 24, max_slots=8)
    V = eng.model.spec.vocab_size
    for length in (1, 64, 83):
        prompt, tails = random_ids(length, V, length), [random_ids(20, V, 90 + i) for i in range(3)]
        a = eng.alloc_slot()
        eng.step([a], [prompt], None)
        slots = [a] + eng.fork_slot(a, 2)
        assert [eng.length(s) for s in slots] == [length] * 3
        alone = [eng.alloc_slot() for _ in range(3)]
        for s in alone:
            eng.step([s], [prompt], None)
        for lo, hi in [(0, 1), (1, 2), (2, 9), (9, 10), (10, 20)]:
            got = rows(eng, slots, [t[lo:hi] for t in tails])
            assert np.array_equal(got, rows(eng, alone, [t[lo:hi] for t in tails]))
        eng.check_status()
        eng.cache.table.check_consistent()
        for s in slots + alone:
            eng.free_slot(s)
        assert all(p.held() == 0 and p.n_shared == 0 for p in eng.cache.table.pools)


@pytest.mark.parametrize("replayed", [False, True])
def test_shared_pages_are_read_once_and_give_the_same(dirs, replayed, monkeypatch):
    """16-bit decode steps of forked sequences run the kernel for shared pages; a step of one sequence alone runs the ordinary one."""
    from ithaca_b200 import Engine
    from ithaca_b200.csrc import attention_bf16
    calls, run = [], attention_bf16.decode_shared
    monkeypatch.setattr(attention_bf16, "decode_shared", lambda *a, **k: (calls.append(a[7:11]), run(*a, **k))[1])
    monkeypatch.setattr(attention_bf16, "sharing_pays", lambda *a: True)
    eng = Engine(dirs("wide"), dtype="bfloat16", max_tokens=64 * 200, max_slots=24)
    prompts = [random_ids(n, 300, n) for n in (330, 700, 64)]
    slots, alone, lens = [], [], []
    for i, p in enumerate(prompts):
        a = eng.alloc_slot()
        eng.step([a], [p], None)
        slots += [a] + eng.fork_slot(a, 3 - i)
        for _ in range(4 - i):
            alone.append(eng.alloc_slot())
            eng.step([alone[-1]], [p], None)
    step = (lambda s, t: eng._decoder.step(s, t)[0].float().cpu().numpy()) if replayed else (lambda s, t: rows(eng, s, t))
    for n in range(70):
        toks = [[(7 * i + 13 * n + n * n) % 300] for i in range(len(slots))]
        if n in (0, 1, 40, 69):
            calls.clear()
            got = step(slots, toks)
            assert calls and all(c[0] == (4 if replayed else 3) and c[1] == 4 for c in calls) or replayed and not calls          # a captured step keeps room for a fourth group
            want = np.concatenate([rows(eng, [s], [t]) for s, t in zip(alone, toks)])
            assert off(got, want) <= REL_CUT["bfloat16"]
        else:
            step(slots, toks)
            rows(eng, alone, toks)
    # a group loses members, another fork joins behind it: other groups, the same sequences
    keep = [0, 2, 4, 5, 7, 8]
    more = eng.fork_slot(slots[5], 2)
    for s in (1, 3, 6):
        eng.free_slot(slots[s])
    live = [slots[0], slots[2], slots[4], slots[5], *more, slots[7], slots[8]]
    of = [alone[0], alone[2], alone[4], alone[5], alone[5], alone[5], alone[7], alone[8]]
    got = step(live, [[5]] * 8)
    want = {s: rows(eng, [s], [[5]]) for s in dict.fromkeys(of)}
    assert off(got, np.concatenate([want[s] for s in of])) <= REL_CUT["bfloat16"]
    eng.check_status()
    eng.cache.table.check_consistent()


def test_a_cut_of_a_forked_sequence_leaves_the_others_alone(dirs):
    from ithaca_b200 import Engine
    for name, dtype in (("A", "float32"), ("wide", "float32"), ("wide", "bfloat16")):
        eng = Engine(dirs(name), dtype=dtype, max_tokens=64 * 30, max_slots=8)
        V = eng.model.spec.vocab_size
        n = 100 if name == "A" else 300
        prompt, other = random_ids(n, V, 1), random_ids(30, V, 2)
        a = eng.alloc_slot()
        eng.step([a], [prompt], None)
        b, c = eng.fork_slot(a, 2)
        for cut in (90, 64, 10):
            eng.truncate(b, cut)
            eng.step([b], [other[:15]], None)                       # writes behind the cut
            eng.cache.table.check_consistent()
        got = rows(eng, [a, c, b], [[3], [3], [4]])
        fresh = [eng.alloc_slot() for _ in range(2)]
        eng.step(fresh, [prompt, prompt[:10]], None)
        eng.step([fresh[1]], [other[:15]], None)
        want = rows(eng, fresh, [[3], [4]])
        limit = 0.0 if dtype == "float32" else REL_CUT[dtype]
        assert off(got[0], want[0]) <= limit and off(got[1], want[0]) <= limit and off(got[2], want[1]) <= limit
        eng.check_status()


def test_forks_are_refused_and_a_refusal_changes_nothing(dirs):
    from ithaca_b200 import Engine
    from ithaca_b200.cache import CacheError, CacheFull
    eng = Engine(dirs("A"), dtype="float32", max_tokens=64 * 3, max_slots=3)
    a = eng.alloc_slot()
    eng.step([a], [[1, 2, 3]], None)
    for slot, n, kind in ((a, 3, CacheFull), (a, -1, CacheError), (2, 1, CacheError), (77, 1, CacheError)):
        with pytest.raises(kind):
            eng.fork_slot(slot, n)
    assert eng.cache.table.n_slots_in_use() == 1 and eng.fork_slot(a, 0) == []
    b, c = eng.fork_slot(a, 2)
    eng.free_slot(a)
    eng.step([b, c], [[4], [5]], "last")
    eng.cache.table.check_consistent()


def test_greedy_generation_in_forked_slots(dirs):
    """The generation loop's steps launched ahead, replayed for sequences that share pages."""
    from ithaca_b200 import Engine
    from ithaca_b200.engine.generate import GenerationOptions
    eng = Engine(dirs("wide"), dtype="bfloat16", max_tokens=64 * 60, max_slots=8)
    prompt = random_ids(200, 300, 5)
    opts = GenerationOptions(max_tokens=40, rep_pen=1.0, stop_token_ids=[])
    a = eng.alloc_slot()
    eng.step([a], [prompt], None)
    slots = [a] + eng.fork_slot(a, 2)
    prompts = [prompt + [7 + i] for i in range(3)]
    got = eng.generate(prompts, opts, resume=[(s, 200) for s in slots])
    for i in range(3):                                              # each token as good as the best by the logits of a slot of its own
        s = eng.alloc_slot()
        lg = eng.step([s], [prompts[i] + got[i][:-1]], [list(range(200, 240))]).float()
        best = lg.max(-1).values
        mine = lg[torch.arange(40), torch.tensor(got[i], device=lg.device)]
        assert float((best - mine).max()) <= 2 * REL["bfloat16"] * float(lg.abs().max())
        eng.free_slot(s)
    eng.cache.table.check_consistent()


# -- the search ------------------------------------------------------------------------------------------------------------
class PlainModel:
    def __init__(self, d):
        self.cfg, self.tensors = load_plain(d)
        self.known = {}

    def logp(self, tokens):
        key = tuple(tokens)
        if key not in self.known:
            self.known[key] = torch.log_softmax(P.logits_whole(list(tokens), self.cfg, self.tensors)[-1].double(), -1).tolist()
        return self.known[key]


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("name,K,stops,penalty", [("A", 3, [], 1.0), ("A", 4, [125, 111, 57, 200], 0.7), ("B", 2, [63], 1.0)])
def test_the_search_matches_plain_float32(dirs, name, K, stops, penalty, graphs):
    from ithaca_b200 import Engine
    d = dirs(name)
    plain = PlainModel(d)
    eng = Engine(d, dtype="float32", max_tokens=64 * 20, graphs=graphs)
    prompts = [random_ids(n, eng.model.spec.vocab_size, 40 + n) for n in (5, 62, 1)]
    got = eng.beam_search(prompts, beams=K, max_tokens=7, length_penalty=penalty, n_best=K, stop_token_ids=stops)
    for p, hyps in zip(prompts, got):
        want = reference(plain, p, K, 7, set(stops), penalty)
        assert [(h.tokens, h.stopped) for h in hyps] == [(t, stop) for _, _, t, stop in want]
        for h, (score, logprob, _, _) in zip(hyps, want):
            assert h.logprob == pytest.approx(logprob, abs=1e-3) and h.score == pytest.approx(score, abs=1e-3)
    assert eng.last_stats.prompt_tokens == 68 and eng.cache.table.n_slots_in_use() == 0
    assert all(p.held() == 0 for p in eng.cache.table.pools)
    # one beam is the greedy choice
    one = eng.beam_search(prompts, beams=1, max_tokens=7, stop_token_ids=[])
    assert [h[0].tokens for h in one] == eng.generate(prompts, max_tokens=7, temp=0.0, rep_pen=1.0, stop_token_ids=[])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["wide", "C", "vebisun", "tiralix", "mimadra", "gunenex", "zomipel", "vovalorn"])
def test_a_hypothesis_has_the_probability_the_model_gives_it(dirs, name, dtype):
    """Over more steps than a page holds, with states and windows: the log probability that the search adds up, beam by beam across forks, is that of the
    tokens fed to a slot of their own; and no request depends on what else is searched."""
    from ithaca_b200 import Engine
    eng = Engine(dirs(name), dtype=dtype, max_tokens=64 * 120, max_slots=40)
    V = eng.model.spec.vocab_size
    room = eng.context_length
    n_new = min(75, room - 45)
    prompts = [random_ids(n, V, 40 + n) for n in (3, 40, 17)]
    got = eng.beam_search(prompts, beams=4, max_tokens=n_new, n_best=4, stop_token_ids=[])
    for p, hyps in zip(prompts, got):
        assert len(hyps) == 4 and all(len(h.tokens) == n_new for h in hyps) and len({tuple(h.tokens) for h in hyps}) == 4
        assert [h.score for h in hyps] == sorted((h.score for h in hyps), reverse=True)
        for h in hyps:
            s = eng.alloc_slot()
            lg = eng.step([s], [p + h.tokens[:-1]], [list(range(len(p) - 1, len(p) + n_new - 1))]).double()
            eng.free_slot(s)
            logp = torch.log_softmax(lg, -1)[torch.arange(n_new), torch.tensor(h.tokens, device=lg.device)].sum().item()
            # a token's log probability is off by at most twice its logits' error
            limit = 2 * REL[dtype] * float(lg.abs().max()) * n_new
            assert abs(logp - h.logprob) <= limit, (logp, h.logprob, limit)
    if dtype == "float32":
        alone = [eng.beam_search([p], beams=4, max_tokens=n_new, n_best=4, stop_token_ids=[])[0] for p in prompts]
        assert [[h.tokens for h in hyps] for hyps in alone] == [[h.tokens for h in hyps] for hyps in got]
    eng.check_status()
    eng.cache.table.check_consistent()
    assert eng.cache.table.n_slots_in_use() == 0 and all(p.held() == 0 for p in eng.cache.table.pools)


def test_a_small_cache_runs_the_requests_in_turn(dirs):
    from ithaca_b200 import Engine
    big = Engine(dirs("A"), dtype="float32", max_tokens=64 * 64)
    small = Engine(dirs("A"), dtype="float32", max_tokens=64 * 8, max_slots=5)
    prompts = [random_ids(n, 256, n) for n in (5, 60, 30, 64)]
    opts = dict(beams=3, max_tokens=20, n_best=3, stop_token_ids=[])
    assert [[h.tokens for h in r] for r in small.beam_search(prompts, **opts)] == [[h.tokens for h in r] for r in big.beam_search(prompts, **opts)]
    assert small.last_stats.batches == 4 and big.last_stats.batches == 1
    with pytest.raises(RuntimeError, match="does not fit"):
        small.beam_search([prompts[0]], beams=6, max_tokens=20)
    with pytest.raises(ValueError):
        small.beam_search([prompts[0]], beams=17)
    assert small.cache.table.n_slots_in_use() == 0


def test_the_command_line_searches(dirs, capsys):
    from ithaca_b200 import Engine
    from ithaca_b200.engine.cli import main
    assert main(["-m", dirs("A"), "-p", "1,2,3", "-p", "9 8", "-n", "6", "--beams", "3", "--dtype", "float32", "--stop-ids", "", "--max-tokens", "1024"]) == 0
    eng = Engine(dirs("A"), dtype="float32", max_tokens=1024)
    want = eng.beam_search([[1, 2, 3], [9, 8]], beams=3, max_tokens=6, stop_token_ids=[])
    assert capsys.readouterr().out.split() == [",".join(map(str, h[0].tokens)) for h in want]


def test_forks_that_share_too_little_step_as_any_others(dirs):
    """No kernel for shared pages would be chosen, so the captured step is the one that sequences of their own use."""
    from ithaca_b200 import Engine
    eng = Engine(dirs("wide"), dtype="bfloat16", max_tokens=64 * 30, max_slots=8)
    a = eng.alloc_slot()
    eng.step([a], [random_ids(70, 300, 5)], None)
    b = eng.fork_slot(a)[0]
    eng._decoder.step([a, b], [[3], [4]])
    assert [len(key) for key in eng._decoder.graphs] == [2]
    eng._settle()
    ids = random_ids(1, 300, 6)
    got = eng._decoder.step([a, b], [ids, ids])[0].float().cpu().numpy()
    alone = [eng.alloc_slot() for _ in range(2)]
    eng._settle()
    eng.step(alone, [random_ids(70, 300, 5)] * 2, None)
    eng.step(alone, [[3], [4]], None)
    assert off(got, rows(eng, alone, [ids, ids])) <= REL_CUT["bfloat16"]
