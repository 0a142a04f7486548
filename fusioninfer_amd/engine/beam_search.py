"""Search with beams over the engine's forced steps.

Every search keeps its ``width`` best sequences. A step decodes one token of
each (one batch over all searches), and ``ops.beam_select`` gives the best
continuations by cumulative log-probability. The first continuation of a beam
takes its sequence over; each further one gets a sequence of its own that
shares the full cache blocks and receives a copy of the partly filled one and
of the recurrent state, all of a step's copies in one launch for pages and one
for states. Beams without a continuation give their blocks back first, so that
a step needs no more blocks than its beams hold.

A continuation that ends with a stop token is a finished hypothesis if it ranks
before the last beam kept; hypotheses are ordered by cumulative log-probability
over length ** length_penalty.

A cumulative log-probability is rounded to fp32 at every step, as
``beam_select`` takes and gives it: at -1000 by up to 3e-5 a step. Beams nearer
to one another than that may change places, or be equal and go by beam.
"""

from __future__ import annotations

from typing import Dict, List, NamedTuple, Sequence as Seq

import torch

import fusioninfer_amd.ops as ops


class BeamHypothesis(NamedTuple):
    """``score``: ``cumulative_logprob`` over the number of tokens (the stop
    token among them) to the power of the length penalty."""
    token_ids: List[int]
    cumulative_logprob: float
    score: float
    finish_reason: str           # "stop" or "length"


class _Beam(NamedTuple):
    request_id: str
    token_ids: List[int]         # generated; the last one is not decoded yet
    cumulative_logprob: float


class _Search:
    def __init__(self, prompt: List[int], most: int):
        self.prompt = prompt
        self.most = most         # tokens to generate at most
        self.beams: List[_Beam] = []
        self.done: List[BeamHypothesis] = []


class BeamSearcher:
    def __init__(self, engine, width: int, max_tokens: int,
                 stop_token_ids: Seq[int], length_penalty: float):
        self.engine = engine
        self.width = width
        self.max_tokens = max_tokens
        self.stops = frozenset(int(t) for t in stop_token_ids)
        self.penalty = float(length_penalty)
        # up to one continuation of every beam for each stop token ends it
        self.k = min(width * (1 + len(self.stops)), ops.MOST_CHOICES)
        self.pages, self.states = engine.runner.cache_tensors()
        self.ids: List[str] = []  # of live requests

    # ----------------------------------------------------------- scoring
    def _hypothesis(self, tokens, cumulative, reason) -> BeamHypothesis:
        return BeamHypothesis(tokens, cumulative,
                              cumulative / len(tokens) ** self.penalty,
                              reason)

    def _decided(self, s: _Search) -> bool:
        """No beam can still come among the ``width`` best: log-probabilities
        only fall, and a length divides them by no more than the longest (or,
        for a negative penalty, no less than the shortest) to come."""
        if not s.beams:
            return True
        if len(s.done) < self.width:
            return False
        worst = sorted((h.score for h in s.done),
                       reverse=True)[self.width - 1]
        best = max(b.cumulative_logprob for b in s.beams)
        n = s.most if self.penalty >= 0 else len(s.beams[0].token_ids)
        return best / n ** self.penalty <= worst

    # ------------------------------------------------------------ search
    def run(self, prompts: List[List[int]]) -> List[List[BeamHypothesis]]:
        limit = self.engine.cfg.scheduler.max_model_len
        searches = [_Search(p, min(self.max_tokens, limit - len(p)))
                    for p in prompts]
        try:
            logits = self._prefill(searches)
            live = list(searches)
            scores = torch.zeros((len(live), 1), device=logits.device)
            while live:
                self._advance(live, ops.beam_select(logits, scores, self.k))
                live = [s for s in live if s.beams]
                if live:
                    logits, scores = self._decode(live)
        finally:
            self.engine.release_forced(self.ids)
        return [sorted(s.done, key=lambda h: -h.score)[:self.width]
                for s in searches]

    def _prefill(self, searches) -> torch.Tensor:
        """Logits after every prompt, portions of it within a step's token
        budget."""
        budget = self.engine.cfg.scheduler.max_num_batched_tokens
        rows = []
        for s in searches:
            rid = self.engine.next_request_id("beam")
            self.ids.append(rid)
            for at in range(0, len(s.prompt), budget):
                part = s.prompt[at: at + budget]
                last = at + len(part) == len(s.prompt)
                out = self.engine.forced_step(
                    [(rid, part, [len(part) - 1] if last else [])])
            rows.append(out)
            s.beams = [_Beam(rid, [], 0.0)]
        return torch.cat(rows)

    def _advance(self, live, choice) -> None:
        """The next beams of every search, and the copies they need."""
        host = torch.stack([choice.scores.view(torch.int32), choice.parents,
                            choice.tokens]).cpu()
        totals = host[0].view(torch.float32).tolist()
        parents, tokens = host[1].tolist(), host[2].tolist()
        ended: List[str] = []
        forks = []               # (beam's request, request that goes on from it)
        for g, s in enumerate(live):
            old, s.beams = s.beams, []
            for total, p, t in zip(totals[g], parents[g], tokens[g]):
                if p < 0 or len(s.beams) == self.width:
                    break
                generated = old[p].token_ids + [t]
                if t in self.stops:
                    s.done.append(self._hypothesis(generated, total, "stop"))
                else:
                    s.beams.append(_Beam(old[p].request_id, generated, total))
            if s.beams and len(s.beams[0].token_ids) >= s.most:
                s.done += [self._hypothesis(b.token_ids,
                                            b.cumulative_logprob, "length")
                           for b in s.beams]
                s.beams = []
            if self._decided(s):
                s.beams = []
            taken: Dict[str, bool] = {}
            for i, b in enumerate(s.beams):
                if b.request_id in taken:
                    child = self.engine.next_request_id("beam")
                    forks.append((b.request_id, child))
                    s.beams[i] = b._replace(request_id=child)
                taken[b.request_id] = True
            ended += [b.request_id for b in old if b.request_id not in taken]
        gone = set(ended)
        self.ids = [r for r in self.ids if r not in gone]
        self.engine.release_forced(ended)
        self._fork(forks)

    def _fork(self, forks) -> None:
        if not forks:
            return
        pages, slots = [], []
        for parent, child in forks:
            self.ids.append(child)
            page, slot = self.engine.fork_forced(parent, child)
            if page is not None:
                pages.append(page)
            if slot is not None:
                slots.append(slot)
        runner = self.engine.runner
        if pages and self.pages:
            src, dst, filled = zip(*pages)
            t = runner._to_device({"src": (list(src), torch.int32),
                                   "dst": (list(dst), torch.int32),
                                   "filled": (list(filled), torch.int32)})
            ops.copy_blocks_(self.pages, t["src"], t["dst"], t["filled"])
        if slots and self.states:
            src, dst = zip(*slots)
            t = runner._to_device({"src": (list(src), torch.int32),
                                   "dst": (list(dst), torch.int32)})
            ops.copy_blocks_(self.states, t["src"], t["dst"])

    def _decode(self, live):
        """Logits [searches * beams, V] and scores [searches, beams]; a search
        with fewer beams than others repeats a row at a score of -inf."""
        beams = [b for s in live for b in s.beams]
        logits = self.engine.forced_logits(
            [(b.request_id, b.token_ids[-1:], [0]) for b in beams])
        most = max(len(s.beams) for s in live)
        scores, rows, at = [], [], 0
        for s in live:
            n = len(s.beams)
            scores += [b.cumulative_logprob for b in s.beams]
            scores += [float("-inf")] * (most - n)
            rows += list(range(at, at + n)) + [at] * (most - n)
            at += n
        if len(rows) > at:
            logits = logits[self.engine.runner._to_device(
                {"rows": (rows, torch.long)})["rows"]]
        return logits, torch.tensor(
            scores, pin_memory=logits.is_cuda).view(len(live), most).to(
                logits.device, non_blocking=True)
