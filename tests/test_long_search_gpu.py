"""The sums of a long search: what a token adds does not drown in what is there."""
import pytest
import torch

import test_beam_gpu
from helpers import random_ids

pytestmark = pytest.mark.gpu
dirs = test_beam_gpu.dirs


@pytest.mark.parametrize("graphs", [True, False])
def test_large_sums_keep_what_a_token_adds(dirs, graphs):
    from ithaca_b200 import Engine
    eng = Engine(dirs("A"), dtype="float32", max_tokens=64 * 20, max_slots=12, graphs=graphs)
    prompts = [random_ids(n, 256, n) for n in (70, 20)]
    slots, alone = [], []
    for p in prompts:
        a = eng.alloc_slot()
        eng.step([a], [p], None)
        slots += [a] + eng.fork_slot(a, 2)
        for _ in range(3):
            alone.append(eng.alloc_slot())
            eng.step([alone[-1]], [p], None)
    tokens = [[5], [9], [77], [5], [200], [1]]
    sums = [[-123456.789, -123456.25, -123459.0], [-3.5, -1.25, -2.0]]
    got = eng.step_and_select(slots, tokens, sums, 12)
    logp = torch.log_softmax(eng.step(alone, tokens, "last").double(), -1).cpu().view(2, 3, -1)
    for r in range(2):
        want = (torch.tensor(sums[r], dtype=torch.float64)[:, None] + logp[r]).flatten().sort(descending=True)
        assert [(b, t) for _, b, t in got[r]] == [divmod(int(i), logp.shape[-1]) for i in want.indices[:12]]
        for (s, b, t), w in zip(got[r], want.values.tolist()):
            # the sum of exponentials is good to 50 x 2^-24, a difference of up to 16 is rounded to a float twice
            assert abs(s - w) <= 50 * 2 ** -24 + 2 * 16 * 2 ** -24, (s, w)


def test_a_long_search_adds_up_its_tokens(dirs):
    """Some hundred tokens, the sum against that of the single probabilities in 64 bits."""
    from ithaca_b200 import Engine
    eng = Engine(dirs("wide"), dtype="float32", max_tokens=64 * 80)
    prompt = random_ids(9, 300, 3)
    hyps = eng.beam_search([prompt], beams=3, max_tokens=400, n_best=3, stop_token_ids=[])[0]
    for h in hyps:
        s = eng.alloc_slot()
        lg = eng.step([s], [prompt + h.tokens[:-1]], [list(range(len(prompt) - 1, len(prompt) + 399))]).double()
        eng.free_slot(s)
        logp = torch.log_softmax(lg, -1)[torch.arange(400), torch.tensor(h.tokens, device=lg.device)].sum().item()
        # a step's sum of exponentials and two roundings of differences up to 16; logits of steps and of a prompt differ by a few 2^-20 of their size
        assert abs(h.logprob - logp) <= 400 * (82 * 2 ** -24 + 2 * 4 * 2 ** -20 * float(lg.abs().max())), (h.logprob, logp)
