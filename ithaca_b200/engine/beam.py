"""Search over beams above the step function.

The reference samples one continuation (src/chat.cpp:292-492); a search is this library's own.  Every request keeps up to K beams: continuations of its
prompt with the sum of the log probabilities of their tokens.  A step evaluates every beam's last token and takes, over all beams and the whole vocabulary, the
best continuations; those that end in a stop token become hypotheses, the K best others the next beams.  A prompt is evaluated once, in one slot; a beam that has several
successors is forked (its slot stays with the first), a beam without one gives its slot back.

The loop's decisions use only the ``BeamBackend`` interface, so they are testable without a device.
"""
from __future__ import annotations

import time
from dataclasses import dataclass, field
from typing import Callable, Dict, List, Optional, Protocol, Sequence, Tuple

from .generate import GenStats, budget_for

BEAMS_MOST, CHOICES_MOST = 16, 32          # what the kernel that chooses takes


@dataclass(frozen=True)
class BeamOptions:
    """``beams``: beams per request.  A hypothesis is ranked by its log probability divided by its length (new tokens, the stop token included) to the
    power ``length_penalty``.  A request ends when it has ``beams`` hypotheses and no beam can still rank above the worst of
    them by what it has now (``early_stopping``: as soon as it has them), or at ``max_tokens``, where its beams become hypotheses as they stand.  Beams and
    stop tokens together may be 32 at most."""
    beams: int = 4
    max_tokens: int = 128
    length_penalty: float = 1.0
    n_best: int = 1
    early_stopping: bool = False
    stop_token_ids: Optional[Sequence[int]] = None     # None: the model's own (eos_token_id)
    include_stop: bool = False
    max_batch: Optional[int] = None                    # None: as many as the cache has slots and room for

    def validate(self) -> None:
        if not 1 <= self.beams <= BEAMS_MOST:
            raise ValueError(f"beams must be between 1 and {BEAMS_MOST}, found {self.beams}")
        if not 1 <= self.n_best <= self.beams:
            raise ValueError(f"n_best must be between 1 and the number of beams, found {self.n_best}")
        if not 0 <= self.length_penalty <= 32:                # (a length to a higher power may pass the largest float)
            raise ValueError(f"length_penalty must be between 0 and 32, found {self.length_penalty}")


@dataclass
class Hypothesis:
    tokens: List[int]              # the new tokens
    logprob: float                 # the sum of their log probabilities, the stop token's included
    score: float                   # logprob / length ** length_penalty
    stopped: bool                  # ended in a stop token


class BeamBackend(Protocol):
    context_length: int

    def room_for_beams(self, prompts: Sequence[int], grown: Sequence[int], beams: int) -> bool: ...
    def free_slots(self) -> int: ...
    def alloc_slot(self) -> int: ...
    def free_slot(self, slot: int) -> None: ...
    def fork_slots(self, wanted: Sequence[Tuple[int, int]]) -> List[List[int]]: ...

    def step_and_select(self, slots: Sequence[int], tokens: Sequence[Sequence[int]], scores: Sequence[Sequence[float]],
                        n_out: int) -> List[List[Tuple[float, int, int]]]:
        """Runs one step and returns per request the best (score, beam, token), best first, at most ``n_out``."""


@dataclass
class _Beam:
    slot: int
    tokens: List[int]
    score: float


@dataclass
class _Search:
    request: int
    budget: int
    beams: List[_Beam]
    done: List[Hypothesis] = field(default_factory=list)

    def keep(self, h: Hypothesis, most: int) -> None:
        """Adds a hypothesis; only the best stay, earlier ones before equal later ones."""
        at = len(self.done)
        while at and self.done[at - 1].score < h.score:
            at -= 1
        self.done.insert(at, h)
        del self.done[most:]


def ranked(logprob: float, length: int, penalty: float) -> float:
    return logprob / max(1, length) ** penalty


def joined(choices: Sequence[Sequence[Tuple[float, int, int]]]) -> List[Tuple[float, int, int]]:
    """The choices of beams that were asked one by one, as those of one request: best first, equal ones by beam, of a beam in their order."""
    return sorted(((score, beam, token) for beam, found in enumerate(choices) for score, _, token in found), key=lambda c: -c[0])


def beam_loop(prompts: Sequence[Sequence[int]], options: BeamOptions, backend: BeamBackend, stop_token_ids: Sequence[int] = (),
              clock: Callable[[], float] = time.perf_counter):
    """Returns (hypotheses per request, best first, at most ``n_best``; GenStats)."""
    options.validate()
    o, ctx = options, backend.context_length
    stops = set(o.stop_token_ids if o.stop_token_ids is not None else stop_token_ids)
    for n, p in enumerate(prompts):
        if len(p) == 0:
            raise ValueError(f"request {n}: empty prompt")
        if len(p) > ctx:
            raise ValueError(f"request {n}: the prompt of {len(p)} tokens is longer than the context of {ctx}")
    budgets = [budget_for(len(p), o.max_tokens, ctx) for p in prompts]
    # of so many choices at least K are no stop tokens.  Where the kernel does not give so many, every beam is asked for its own: K of them are no stop tokens, and the best
    # of all beams are among them
    n_out = o.beams * (1 + len(stops))
    apart = n_out > CHOICES_MOST
    if apart:
        n_out = o.beams + len(stops)
        if n_out > CHOICES_MOST:
            raise ValueError(f"{o.beams} beams and {len(stops)} stop tokens: at most {CHOICES_MOST} together are supported")
    results: List[List[Hypothesis]] = [[] for _ in prompts]
    stats = GenStats()
    pending = list(range(len(prompts)))

    def settle(run: _Search, choices) -> Optional[List[Tuple[int, int, float]]]:
        """Takes a step's choices; the next beams as (parent, token, score), or None if the request has ended."""
        nxt: List[Tuple[int, int, float]] = []
        for rank, (score, beam, token) in enumerate(choices):
            if len(nxt) == o.beams:
                break
            tokens = run.beams[beam].tokens
            if token in stops:
                if rank < o.beams:
                    run.keep(Hypothesis(tokens + [token] if o.include_stop else list(tokens), score, ranked(score, len(tokens) + 1, o.length_penalty), True), o.beams)
            else:
                nxt.append((beam, token, score))
        if not nxt:
            return None
        length = len(run.beams[nxt[0][0]].tokens) + 1
        stats.gen_tokens += len(nxt)
        if length >= run.budget:
            for beam, token, score in nxt:
                run.keep(Hypothesis(run.beams[beam].tokens + [token], score, ranked(score, length, o.length_penalty), False), o.beams)
            return None
        if len(run.done) >= o.beams and (o.early_stopping or ranked(nxt[0][2], length, o.length_penalty) <= run.done[-1].score):
            return None
        return nxt

    def advance(running: List[_Search], chosen: List[Optional[List[Tuple[int, int, float]]]]) -> List[_Search]:
        """Gives back the slots of beams without a successor and forks those with several; the requests that go on."""
        still: List[_Search] = []
        waiting: Dict[int, List[_Beam]] = {}                                   # slot to fork: the beams that wait for a copy of it
        for run, nxt in zip(running, chosen):
            old = run.beams
            alive = {beam for beam, _, _ in nxt or ()}
            for i, b in enumerate(old):
                if i not in alive:
                    backend.free_slot(b.slot)
            run.beams = []
            if nxt is None:
                results[run.request] = run.done[:o.n_best]
                continue
            for beam, token, score in nxt:
                mine = _Beam(old[beam].slot if beam in alive else -1, old[beam].tokens + [token], score)
                if beam in alive:
                    alive.remove(beam)                                         # the first successor goes on in its parent's slot
                else:
                    waiting.setdefault(old[beam].slot, []).append(mine)
                run.beams.append(mine)
            still.append(run)
        if waiting:
            for beams, made in zip(waiting.values(), backend.fork_slots([(slot, len(beams)) for slot, beams in waiting.items()])):
                for b, slot in zip(beams, made):
                    b.slot = slot
        return still

    while pending:
        batch: List[int] = []
        for r in pending:
            if (o.max_batch is not None and len(batch) >= o.max_batch) or (len(batch) + 1) * o.beams > backend.free_slots():
                break
            if not backend.room_for_beams([len(prompts[c]) for c in batch + [r]], [len(prompts[c]) + budgets[c] for c in batch + [r]], o.beams):
                break
            batch.append(r)
        if not batch:
            raise RuntimeError(f"request {pending[0]} does not fit the cache even alone ({len(prompts[pending[0]])} prompt tokens + {budgets[pending[0]]} new "
                               f"in {o.beams} beams)")
        pending = pending[len(batch):]
        stats.batches += 1
        running = [_Search(r, budgets[r], []) for r in batch if budgets[r] > 0]
        try:
            for run in running:
                run.beams = [_Beam(backend.alloc_slot(), [], 0.0)]
            first = True
            while running:
                t0 = clock()
                running.sort(key=lambda run: len(run.beams))               # as many beams next to one another; else in their order
                beams = [b for run in running for b in run.beams]
                tokens = [list(prompts[run.request]) for run in running] if first else [[b.tokens[-1]] for b in beams]
                if apart:
                    each = iter(backend.step_and_select([b.slot for b in beams], tokens, [[b.score] for b in beams], n_out))
                    picked = [joined([next(each) for _ in run.beams]) for run in running]
                else:
                    picked = backend.step_and_select([b.slot for b in beams], tokens, [[b.score for b in run.beams] for run in running], n_out)
                running = advance(running, [settle(run, c) for run, c in zip(running, picked)])
                stats.steps += 1
                if first:
                    stats.prefill_seconds += clock() - t0
                    stats.prompt_tokens += sum(len(t) for t in tokens)
                else:
                    stats.decode_seconds += clock() - t0
                first = False
        finally:
            for run in running:
                for b in run.beams:
                    if b.slot >= 0:
                        backend.free_slot(b.slot)
    return results, stats
