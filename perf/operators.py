"""The operators of beam search, as cases that can be timed: inputs, one pass, its work, its exact result.

Three operators: the choice of the best continuations over beams and vocabulary (``select``), the copies that a forked sequence
needs, of pages in part or whole and of fixed-size states, in all layers (``fork``), and attention of one new token per sequence where
groups of sequences share their first pages (``attention``).  Sizes are those of the configurations this repository benchmarks
(Llama-3.1-8B, Llama-3.2-1B and Llama-2-13B shapes, and the states of its recurrent mixers) and odd ones in their neighbourhood.

``own`` False: the operators in their plain form, elementary torch operations.  ``own`` True: this library's calls."""
import math
import random

import torch

own = False
DEVICE = "cuda:0"
PAGE = 64


def listed():
    return [
        # one request with four beams: the smallest call of a search, latency only
        {"name": "select 1x4 of 128256", "kind": "select", "requests": 1, "beams": 4, "vocab": 128256, "out": 8, "live": 4, "masked": 0.0},
        # the first choice behind the prompt: one live beam per request, the others have no score yet
        {"name": "select first 8x5 of 32000", "kind": "select", "requests": 8, "beams": 5, "vocab": 32000, "out": 10, "live": 1, "masked": 0.0},
        # a serving batch under a grammar that forbids most tokens, a vocabulary whose rows do not start on 16 bytes
        {"name": "select 16x8 of 50257 masked", "kind": "select", "requests": 16, "beams": 8, "vocab": 50257, "out": 16, "live": 8, "masked": 0.9},
        # the largest batch of wide searches
        {"name": "select 32x16 of 128256", "kind": "select", "requests": 32, "beams": 16, "vocab": 128256, "out": 32, "live": 16, "masked": 0.0},
        # one beam forks: its last page, just begun, in every layer of the 1B shape
        {"name": "fork 1 page 1b", "kind": "fork", "layers": 16, "heads": 8, "k": 64, "v": 64, "dtype": "bfloat16", "parents": 1, "children": 1, "rows_from": 7, "rows_to": 7,
         "state": 0, "state_layers": 0},
        # a step of eight searches of the 8B shape: about half of the beams fork, their last pages filled to different heights
        {"name": "fork 16 pages 8b", "kind": "fork", "layers": 32, "heads": 8, "k": 128, "v": 128, "dtype": "bfloat16", "parents": 16, "children": 1, "rows_from": 1, "rows_to": 64,
         "state": 0, "state_layers": 0},
        # behind the prompt a sequence with matrix states (16 heads of 128 x 128, two positions) and pages becomes four, for six requests
        {"name": "fork 6 prompts with states", "kind": "fork", "layers": 8, "heads": 4, "k": 64, "v": 64, "dtype": "bfloat16", "parents": 6, "children": 3, "rows_from": 20, "rows_to": 64,
         "state": 2 * 16 * 128 * 128, "state_layers": 16},
        # the 32-bit path with value heads of another size and states of an odd size
        {"name": "fork 32-bit odd", "kind": "fork", "layers": 12, "heads": 3, "k": 80, "v": 33, "dtype": "float32", "parents": 9, "children": 2, "rows_from": 1, "rows_to": 64,
         "state": 4099, "state_layers": 12},
        # one request with four beams behind a prompt of 4,096 tokens, one layer of the 8B shape
        {"name": "attention 1x4 8b", "kind": "attention", "heads": 32, "kv": 8, "size": 128, "groups": 1, "members": 4, "ragged": False, "shared_from": 4096, "shared_to": 4096,
         "own_from": 40, "own_to": 40},
        # eight requests with four beams each, prompts of unequal lengths
        {"name": "attention 8x4 8b", "kind": "attention", "heads": 32, "kv": 8, "size": 128, "groups": 8, "members": 4, "ragged": False, "shared_from": 1000, "shared_to": 8000,
         "own_from": 10, "own_to": 200},
        # forked sequences in groups of unequal size (some alone), smaller heads, tails that differ
        {"name": "attention 12x1-8 1b", "kind": "attention", "heads": 32, "kv": 8, "size": 64, "groups": 12, "members": 8, "ragged": True, "shared_from": 100, "shared_to": 4000,
         "own_from": 1, "own_to": 500},
        # a key head per query head, sixteen beams behind long prompts
        {"name": "attention 2x16 13b", "kind": "attention", "heads": 40, "kv": 40, "size": 128, "groups": 2, "members": 16, "ragged": False, "shared_from": 12000, "shared_to": 16000,
         "own_from": 100, "own_to": 100},
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("select", "fork", "attention"))
    if kind == "select":
        beams, vocab = rng.randint(1, 16), log_int(rng, 300, 129000)
        requests = log_int(rng, 1, max(1, min(64, 32 * 16 * 128256 // (beams * vocab))))
        return {"kind": kind, "requests": requests, "beams": beams, "vocab": vocab, "out": rng.randint(beams, 2 * beams),
                "live": rng.choice((1, beams, beams, max(1, beams - 1))), "masked": rng.choice((0.0, 0.0, 0.5, 0.99))}
    if kind == "fork":
        layers, heads, k = log_int(rng, 2, 32), rng.randint(1, 8), rng.choice((64, 128, 80, 16 * rng.randint(1, 8), rng.randint(20, 140)))
        v, state, children = rng.choice((k, k, rng.randint(20, 140))), rng.choice((0, 0, 2 * 16 * 64 * 64, rng.randint(100, 70000))), rng.choice((1, 1, 1, 2, 3, 5))
        parents = log_int(rng, 1, max(1, min(24, 700_000_000 // ((1 + children) * (layers * heads * PAGE * (k + v) * 4 + 64 * state)))))
        return {"kind": kind, "layers": layers, "heads": heads, "k": k, "v": v, "dtype": rng.choice(("bfloat16", "bfloat16", "float32")),
                "parents": parents, "children": children, "rows_from": 1, "rows_to": rng.choice((1, 33, 64, 64)),
                "state": state, "state_layers": rng.randint(1, 16) if state else 0}
    kv = rng.choice((1, 2, 8, 8, 8, 10, 40))
    per = rng.choice((1, 4, 4, 8, 3)) if kv < 40 else 1
    groups, members = log_int(rng, 1, 12), rng.randint(2, 16)
    size, tail = rng.choice((64, 128, 128)), log_int(rng, 2, 600)
    shared = log_int(rng, 64, max(200, min(16000, 2 * 16 * 16000 * 40 // (groups * members * kv * 2), 500_000_000 // (groups * kv * size * 4) - members * tail)))
    return {"kind": kind, "heads": kv * per, "kv": kv, "size": size, "groups": groups, "members": members, "ragged": rng.random() < 0.4,
            "shared_from": max(1, shared // rng.choice((1, 4))), "shared_to": shared, "own_from": 1, "own_to": tail}


# -- inputs ----------------------------------------------------------------------------------------------------------------
def generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    g, r = generator(seed), random.Random(seed)
    state = {"case": case}
    if case["kind"] == "select":
        R, K, V = case["requests"], case["beams"], case["vocab"]
        logits = torch.randn((R * K, V), generator=g, device=DEVICE) * 2.5
        if case["masked"]:
            mask = torch.rand((R, 1, V), generator=g, device=DEVICE) < case["masked"]              # a request's beams stand at the same place of the grammar
            logits.view(R, K, V).masked_fill_(mask, -math.inf)
        scores = torch.rand((R, K), generator=g, device=DEVICE) * -30.0
        scores[:, case["live"]:] = -math.inf
        return {**state, "logits": logits, "scores": scores}
    if case["kind"] == "fork":
        dtype = torch.bfloat16 if case["dtype"] == "bfloat16" else torch.float32
        P, C = case["parents"], case["children"]
        n = P * (C + 1) + 3
        shape = (case["layers"], n, case["heads"], PAGE)
        state["pages"] = [torch.randn(shape + (s,), generator=g, device=DEVICE, dtype=dtype) for s in (case["k"], case["v"])]
        state["states"] = [torch.randn((case["state_layers"], P * (C + 1), case["state"]), generator=g, device=DEVICE)] if case["state"] else []
        # which pages, filled how far, and which slots: what the cache's bookkeeping has in hand
        at, slots = r.sample(range(n), P * (C + 1)), r.sample(range(P * (C + 1)), P * (C + 1))
        rows = [r.randint(case["rows_from"], case["rows_to"]) for _ in range(P)]
        state["moves"] = [(at[p], at[P + p * C + c], rows[p]) for p in range(P) for c in range(C)]
        state["slot_moves"] = [(slots[p], slots[P + p * C + c]) for p in range(P) for c in range(C)]
        return state
    members, shared, lens = layout(case, seed)
    B, kv, size = sum(members), case["kv"], case["size"]
    pages = [-(-n // PAGE) for n in lens]
    total, cols = sum(shared) + sum(p - s for p, s in zip(pages, per_sequence(members, shared))), max(pages)
    order = r.sample(range(total), total)
    table, b = torch.full((B, cols), -1, dtype=torch.int32), 0
    for m, s in zip(members, shared):
        first, order = order[:s], order[s:]
        for _ in range(m):
            rest, order = order[:pages[b] - s], order[pages[b] - s:]
            table[b, :pages[b]] = torch.tensor(first + rest, dtype=torch.int32)
            b += 1
    starts = [0]
    for m in members:
        starts.append(starts[-1] + m)
    return {**state, "q": torch.randn((B, case["heads"] * size), generator=g, device=DEVICE, dtype=torch.bfloat16),
            "k": torch.randn((total, kv, PAGE, size), generator=g, device=DEVICE, dtype=torch.bfloat16) * 1.5,
            "v": torch.randn((total, kv, PAGE, size), generator=g, device=DEVICE, dtype=torch.bfloat16),
            "lens": torch.tensor(lens, dtype=torch.int32, device=DEVICE), "table": table.to(DEVICE), "bound": max(lens),
            "starts": torch.tensor(starts, dtype=torch.int32, device=DEVICE), "shared": torch.tensor(per_sequence(members, shared), dtype=torch.int32, device=DEVICE),
            "n_groups": len(members), "max_members": max(members), "shared_bound": max(shared),
            "own_bound": max(p - s for p, s in zip(pages, per_sequence(members, shared))), "status": torch.zeros(1, dtype=torch.int32, device=DEVICE)}


def layout(case, seed):
    """Members of every group, pages they share, positions of every sequence (its new token among them)."""
    r = random.Random(seed)
    members = [r.randint(1, case["members"]) if case["ragged"] else case["members"] for _ in range(case["groups"])]
    shared, lens = [], []
    for m in members:
        n = r.randint(case["shared_from"], case["shared_to"])
        tail = r.randint(case["own_from"], case["own_to"])
        shared.append(n // PAGE if m > 1 else 0)                                                    # whole pages only; one alone shares nothing
        lens += [n + (r.randint(case["own_from"], case["own_to"]) if case["ragged"] else tail) for _ in range(m)]
    return members, shared, lens


def per_sequence(members, values):
    return [v for m, v in zip(members, values) for _ in range(m)]


# -- one pass --------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return {"select": run_select, "fork": run_fork, "attention": run_attention}[case["kind"]](case, state)


def run_select(case, state):
    logits, scores, n = state["logits"], state["scores"], case["out"]
    if own:
        from ithaca_b200.csrc import ops
        return ops.beam_select(logits, scores, n)
    R, K, V = case["requests"], case["beams"], case["vocab"]
    # in 64 bits: which of two candidates is the better may be a matter of the last bits
    l = logits.double()
    top = l.amax(-1, keepdim=True)
    lse = top + (l - top).exp().sum(-1, keepdim=True).log()
    s = (scores.double().view(R * K, 1) + (l - lse)).view(R, K * V)
    best, at = s.topk(n, dim=1)
    # descending, equal ones by ascending place
    at, order = at.sort(dim=1)
    best, order = best.gather(1, order).sort(dim=1, descending=True, stable=True)
    at = at.gather(1, order)
    none = best == -math.inf
    return best.float(), (at // V).int().masked_fill(none, -1), (at % V).int().masked_fill(none, -1)


def run_fork(case, state):
    if own:
        from ithaca_b200.csrc import ops
        src, dst, rows = zip(*state["moves"])
        jobs = [(t, src, dst, rows) for t in state["pages"]]
        if state["states"]:
            src, dst = zip(*state["slot_moves"])
            jobs += [(t, src, dst, None) for t in state["states"]]
        ops.copy_rows(jobs)
        return state["pages"] + state["states"]
    moves = torch.tensor(state["moves"]).to(DEVICE)
    src, dst, rows = moves.unbind(1)
    filled = (torch.arange(PAGE, device=DEVICE)[None] < rows[:, None])[None, :, None, :, None]
    out = [t.index_copy_(1, dst, torch.where(filled, t[:, src], t[:, dst])) for t in state["pages"]]
    if state["states"]:
        src, dst = torch.tensor(state["slot_moves"]).to(DEVICE).unbind(1)
        out += [t.index_copy_(1, dst, t[:, src]) for t in state["states"]]
    return out


def run_attention(case, state):
    q, k, v, lens, table = state["q"], state["k"], state["v"], state["lens"], state["table"]
    H, G, size = case["heads"], case["kv"], case["size"]
    if own:
        from ithaca_b200.csrc import attention_bf16
        return attention_bf16.decode_shared(q, k, v, lens, table, state["starts"], state["shared"], state["n_groups"], state["max_members"], state["shared_bound"],
                                            state["own_bound"], H, size ** -0.5, state["status"])
    B, cols = table.shape
    at = table.clamp(min=0).long()
    keys = k[at].transpose(2, 3).reshape(B, cols * PAGE, G, size).float()
    values = v[at].transpose(2, 3).reshape(B, cols * PAGE, G, size).float()
    s = torch.einsum("bgrd,bjgd->bgrj", q.view(B, G, H // G, size).float(), keys) * size ** -0.5
    s = s.masked_fill(torch.arange(cols * PAGE, device=DEVICE)[None, None, None] >= lens[:, None, None, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp()
    o = torch.einsum("bgrj,bjgd->bgrd", p, values) / p.sum(-1, keepdim=True)
    return o.reshape(B, H * size).to(torch.bfloat16)


# -- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "select":
        R, K, V = case["requests"], case["beams"], case["vocab"]
        return {"bytes": R * case["live"] * V * 4 + R * K * 4 + R * case["out"] * 12, "flops": R * case["live"] * V * 4}     # a beam without a score has no candidates
    if case["kind"] == "fork":
        size = 2 if case["dtype"] == "bfloat16" else 4
        rows = (case["rows_from"] + case["rows_to"]) / 2
        once = case["layers"] * case["heads"] * rows * (case["k"] + case["v"]) * size + case["state_layers"] * case["state"] * 4
        return {"bytes": case["parents"] * (1 + case["children"]) * once, "flops": 0}
    # the lengths of a case's every seed, on average
    m = (1 + case["members"]) / 2 if case["ragged"] else case["members"]
    shared, tail = (case["shared_from"] + case["shared_to"]) / 2, (case["own_from"] + case["own_to"]) / 2
    positions, pairs = case["groups"] * (shared + m * tail), case["groups"] * m * (shared + tail)
    return {"bytes": positions * case["kv"] * case["size"] * 4 + case["groups"] * m * case["heads"] * case["size"] * 4, "flops": 4 * case["heads"] * case["size"] * pairs}


# -- the results in 64 bits ------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "select":
        R, K, V, n = case["requests"], case["beams"], case["vocab"], case["out"]
        found, where = [], []
        for r in range(R):
            logp = torch.log_softmax(state["logits"][r * K:(r + 1) * K].to(torch.float64), dim=-1)
            s = (logp + state["scores"][r].to(torch.float64)[:, None]).flatten()
            s, at = torch.sort(s, descending=True, stable=True)
            found.append(s[:n])
            where.append(torch.where(s[:n] > -math.inf, at[:n], -1))
        s, at = torch.stack(found), torch.stack(where)
        return s, torch.where(at >= 0, at // V, -1).to(torch.int32), torch.where(at >= 0, at % V, -1).to(torch.int32)
    if case["kind"] == "fork":
        out = [t.to(torch.float64) for t in state["pages"] + state["states"]]
        for t in out[:2]:
            for s, d, n in state["moves"]:
                t[:, d, :, :n] = t[:, s, :, :n]
        for t in out[2:]:
            for s, d in state["slot_moves"]:
                t[:, d] = t[:, s]
        return out
    H, G, size = case["heads"], case["kv"], case["size"]
    rows = []
    for q, n, t in zip(state["q"].to(torch.float64).view(-1, G, H // G, size), state["lens"].tolist(), state["table"].long()):
        at = t[:-(-n // PAGE)]
        k, v = (x[at].to(torch.float64).permute(1, 0, 2, 3).reshape(G, -1, size)[:, :n] for x in (state["k"], state["v"]))
        rows.append(torch.softmax(q @ k.transpose(1, 2) / math.sqrt(size), dim=-1).matmul(v).flatten())
    return torch.stack(rows)
