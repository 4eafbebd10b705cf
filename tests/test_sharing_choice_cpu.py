"""When a decode step of forked sequences is described as one that shares pages: where a layer's kernel will read them once, by its own heads and by the
sizes that the step is kept under."""
from types import SimpleNamespace

import pytest

from ithaca_b200.cache import KVRequest, SequenceCache
from ithaca_b200.engine.graph import _round_up, _sharing_shape
from ithaca_b200.engine.model import DecoderModel
from ithaca_b200.engine.step import Stepper
from ithaca_b200.parts.attention import Attention
from ithaca_b200.parts.parallel import ParallelMixer


def forked(prompt, members, tail, heads, nkv=2, hd=64, window=None):
    """A stepper over a cache in which ``members`` sequences share a prompt and go on by ``tail`` tokens each; the step's tables and pages."""
    cache = SequenceCache({0: [KVRequest(nkv, hd, window)]}, max_tokens=64 * 4000, max_slots=members, device=None)
    a = cache.alloc_slot()
    cache.reserve([a], [prompt])
    cache.commit([a], [prompt])
    slots = [a] + cache.fork([(a, members - 1)])[0]
    cache.reserve(slots, [tail + 1] * members)
    cache.commit(slots, [tail] * members)
    st = Stepper.__new__(Stepper)
    st.cache, st.runtime, st.joint_heads = cache, SimpleNamespace(dtype="bfloat16"), [heads]
    pages = [cache.length(s) // 64 + 1 for s in slots]
    return st, [cache.table.table_rows(0, slots, max(pages))], pages


@pytest.mark.parametrize("round_up", [None, _round_up])
def test_a_step_is_described_as_sharing_where_a_kernel_reads_pages_once(round_up):
    from ithaca_b200.csrc.attention_bf16 import sharing_pays
    seen = set()
    for prompt in (64, 700, 1300, 2600, 6400):
        for members in (2, 5, 12, 16):
            for tail in (1, 200, 900):
                for heads in (2, 8, 16, 32):
                    st, tables, pages = forked(prompt, members, tail, {heads})
                    (f,) = st.sharing(tables, pages, round_up) or [None]
                    shared, own = prompt // 64, max(pages) - prompt // 64
                    n, m = 1, members
                    if round_up is not None:
                        m = min(members, 1 << (members - 1).bit_length())
                        shared, own = 1 << (shared - 1).bit_length(), 1 << (own - 1).bit_length()
                    pays = sharing_pays(members, n, m, shared, own, heads, 2, 64)
                    assert (f is not None) == pays, (prompt, members, tail, heads)
                    if f is not None:
                        assert (f.n_groups, f.max_members, f.shared_bound, f.own_bound) == (n, m, shared, own)
                    seen.add((heads, pays))
    assert len(seen) == 8                                        # both answers for every number of heads


def test_layers_of_other_heads_in_a_group():
    """One that reads shared pages once is enough; none, or no layer that could, and the step is as any other."""
    st, tables, pages = forked(1300, 12, 200, set())
    assert st.sharing(tables, pages, _round_up) == []
    st.joint_heads = [{8}]
    assert st.sharing(tables, pages, _round_up) == []
    st.joint_heads = [{2}]
    (f,) = st.sharing(tables, pages, _round_up)
    assert _sharing_shape(f) == (1, 12, 32, 4)
    st.joint_heads = [{8, 2}]
    assert len(st.sharing(tables, pages, _round_up)) == 1
    st.runtime.dtype = "float32"
    assert st.sharing(tables, pages, _round_up) == []


def test_which_layers_could():
    def layer(**kw):
        a = Attention.__new__(Attention)
        a.window, a.slopes, a.values_are_keys, a.head_dim, a.v_head_dim, a.n_heads = None, None, False, 64, 64, 8
        for k, v in kw.items():
            setattr(a, k, v)
        return a
    assert layer().joint_heads == 8
    for kw in (dict(window=128), dict(slopes=[0.5] * 8), dict(values_are_keys=True), dict(v_head_dim=32)):
        assert layer(**kw).joint_heads == 0
    both = ParallelMixer.__new__(ParallelMixer)
    both.branches = [SimpleNamespace(), layer(n_heads=6)]
    assert both.joint_heads == 6
    model = DecoderModel.__new__(DecoderModel)
    mixers = [layer(), both, layer(window=64), SimpleNamespace()]
    model.layers = [SimpleNamespace(mixer=m) for m in mixers]
    model.spec = SimpleNamespace(schedule=[SimpleNamespace(layer=i, cache=c) for i, c in ((0, 0), (1, 1), (2, 2), (3, 3), (0, 1))])
    assert model.joint_heads() == {0: {8}, 1: {6, 8}}
