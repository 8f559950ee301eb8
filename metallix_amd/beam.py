"""Beam search on the device: a batch of requests, several sequences each.

The reference decodes one sequence per request (EngineLoop::decode_now,
crates/app/cli/src/engine_loop.rs:1080-1134); this is the step that stands in
its place for requests that search.  `BeamSearch.step` takes the logits of all
live sequences and queues the selection (mxs_beam_select) and the move of what
each sequence carries (mxs_beam_reorder: the caller's states, the token
histories, the lengths) on the sampler's stream; nothing is read back until
`result`.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional

from .sampler import BeamResult


@dataclass
class Hypothesis:
    """One sequence a search found: its tokens (the end token included when
    it ended), its cumulative log probability and whether it ended."""
    tokens: List[int]
    score: float
    ended: bool


class BeamSearch:
    """groups x beams sequences over one Sampler.  Row g * beams + b of every
    tensor is beam b of group g; a group starts with one live beam, beam 0.
    Ended beams stay in the race with their score.  length_penalty a orders
    the candidates by score * ((5 + length) / 6) ** -a.

    A group whose selection fails has no hypotheses from then on, and status()
    says why; the others go on."""

    def __init__(self, sampler, groups: int, beams: int, max_new: int, *, end_token: Optional[int] = None,
                 length_penalty: float = 0.0):
        torch = sampler.torch
        self.sampler, self.groups, self.beams, self.max_new = sampler, groups, beams, max_new
        self.end_token, self.length_penalty = end_token, float(length_penalty)
        self.steps = 0
        dev = torch.device("cuda", sampler.device)
        rows = groups * beams
        with torch.cuda.stream(sampler.stream):
            self.score = torch.full((groups, beams), float("-inf"), dtype=torch.float64, device=dev)
            self.score[:, 0] = 0.0
            self.ended = torch.zeros((groups, beams), dtype=torch.bool, device=dev)
            self.tokens = torch.full((rows, max_new), -1, dtype=torch.int32, device=dev)
            self.length = torch.zeros((rows, 1), dtype=torch.int32, device=dev)
            e = lambda *s: torch.empty(s, dtype=torch.int32, device=dev)
            # each step's own tokens and statuses
            self._tokens = torch.empty((max_new, groups, beams), dtype=torch.int32, device=dev)
            self._statuses = torch.zeros((max_new + 1, groups), dtype=torch.int32, device=dev)
            self.picked = BeamResult(token=e(groups, beams), beam=e(groups, beams), score=self.score, ended=self.ended,
                                     status=e(groups))
            self._live = None   # the step and which rows' sequences went on after it (attention)
            # the positions of each row's own cache after so many steps, the ended ones' too (attention)
            self._own = torch.arange(max_new + 1, dtype=torch.int32, device=dev).view(-1, 1).repeat(1, rows)
            self._now = None    # a step and its row of them
            self.moved = e(groups)   # (always 0: the parents are the selection's)

    def step(self, logits, states=(), *, lengths=None, length_dim=None, **rule):
        """Queues one step over `logits` [groups * beams, vocab]: picks each
        group's best continuations (`rule`: mask, legal_norm, ... of
        Sampler.beam_select, but not the end token, the ended beams or, with
        a length penalty, the scale, which are the search's), moves `states`
        (tensors of groups * beams rows, the first lengths[g] positions of
        their length_dim) and the search's own rows to them.  Returns the
        rows' next tokens, int32[groups * beams] on the device (-1: no
        sequence; an ended one's end token), a tensor of this step's own that
        later steps leave alone."""
        if self.steps >= self.max_new:
            raise ValueError(f"the search holds {self.max_new} tokens")
        own = {"ended", "end_token"} | ({"scale"} if self.length_penalty else set())
        if own & rule.keys():
            raise ValueError(f"the search itself gives the selection its {' and '.join(sorted(own & rule.keys()))}")
        s, torch = self.sampler, self.sampler.torch
        with torch.cuda.stream(s.stream):
            # (the states and the move are checked before anything is queued)
            dims = list(length_dim) if isinstance(length_dim, (list, tuple)) else [length_dim] * len(states)
            move = s.reorder_launcher([*states, self.tokens, self.length], self.picked.beam, lengths=lengths,
                                      length_dim=[*dims, None, None], status=self.moved)
            if self.end_token is not None:
                rule = dict(rule, ended=self.ended, end_token=self.end_token)
                going = ~self.ended.view(-1, 1)   # (the selection writes over `ended`)
            if self.length_penalty:
                n = torch.where(self.ended, self.length.view(self.groups, self.beams), self.steps + 1)
                rule = dict(rule, scale=((5.0 + n.double()) / 6.0) ** -self.length_penalty)
            p = self.picked
            picked = BeamResult(self._tokens[self.steps], p.beam, p.score, p.ended, self._statuses[self.steps])
            s.beam_select(logits, self.score, self.beams, out=picked, **rule)
            # (the step is accepted: the parents' lengths, which then move with their rows)
            if self.end_token is not None:
                self.length.masked_fill_(going, self.steps + 1)
            else:
                self.length.fill_(self.steps + 1)
            move()
            self.picked, tokens = picked, picked.token.view(-1)
            self.tokens[:, self.steps] = tokens
        self.steps += 1
        return tokens

    def attention(self, q, prefix_keys, prefix_values, keys, values, *, lengths=None, weight=None, **kw):
        """Queues one layer's attention of all sequences after a step
        (Sampler.prefix_attention): q bf16[groups * beams, heads, dim], the
        queries of the tokens that step() returned; prefix_keys and
        prefix_values [groups, kv_heads, positions, dim], the prompts', one for
        each group; keys and values [groups * beams, kv_heads, at least
        max_new, dim], the sequences' own, of which the steps so far have
        filled the first self.steps positions (these move as step's states, the
        prompts' stay).  Own caches that were evicted since hold lengths[r]
        positions, int32[groups * beams] on the device (a state too, as
        [groups * beams, 1]), and need no room for max_new.  weight
        f32[groups * beams, kv_heads, keys' positions] gets the own positions'
        weights added (a state too).  Only rows whose sequence goes on add
        weights: the queries of ended ones and of beams without a sequence say
        nothing of what later tokens need (counted: other rows).  The other
        arguments are prefix_attention's.  Returns out, of q's shape."""
        if self.steps == 0:
            raise ValueError("the first step comes before the sequences have tokens of their own")
        rows = self.groups * self.beams
        for t, name, n, what in ((q, "q", rows, "rows"), (keys, "keys", rows, "rows"), (values, "values", rows, "rows"),
                                 (prefix_keys, "prefix_keys", self.groups, "prompts, one for each group"),
                                 (prefix_values, "prefix_values", self.groups, "prompts, one for each group")):
            if t is None or t.dim() == 0 or t.shape[0] != n:
                raise ValueError(f"{name} must have {n} {what}, not {None if t is None else list(t.shape)}")
        if lengths is None:
            if keys.dim() != 4 or values.dim() != 4 or min(keys.shape[2], values.shape[2]) < self.steps:
                raise ValueError(f"keys and values must hold {self.steps} positions")
            if self._now is None or self._now[0] != self.steps:
                self._now = self.steps, self._own[self.steps]
            lengths = self._now[1]
        with self.sampler.torch.cuda.stream(self.sampler.stream):
            if kw.get("counted") is None and (weight is not None or kw.get("prefix_weight") is not None):
                kw["counted"] = self._counted()
            return self.sampler.prefix_attention(q, prefix_keys, prefix_values, keys, values,
                                                 lengths=lengths, weight=weight, **kw)

    def _counted(self):
        """The rows whose sequence goes on, bool[groups * beams], worked out once
        a step, or in the graph where the call is captured."""
        if self.sampler.torch.cuda.is_current_stream_capturing():
            return ((self.score > float("-inf")) & ~self.ended).view(-1)
        if self._live is None or self._live[0] != self.steps:
            self._live = self.steps, ((self.score > float("-inf")) & ~self.ended).view(-1)
        return self._live[1]

    def status(self) -> List[int]:
        """What first stopped each group (ROW_STATUS), 0 for one that goes on
        (reads back): a NaN or +inf among its logits (-6), no candidate (-3),
        scores or scales that are no numbers (-14)."""
        self.sampler.sync()
        return [next((s for s in steps if s), 0) for steps in zip(*self._statuses.cpu().tolist())]

    def done(self) -> bool:
        """Whether every sequence has ended or is not there (reads back)."""
        self.sampler.sync()
        return bool((self.ended | (self.score == float("-inf")) | self.score.isnan()).all())

    def result(self) -> List[List[Hypothesis]]:
        """Each group's hypotheses, best first (reads back); none for a group
        whose status() is not 0."""
        self.sampler.sync()
        tokens, length = self.tokens.cpu().tolist(), self.length.cpu().view(-1).tolist()
        score, ended = self.score.cpu().tolist(), self.ended.cpu().tolist()
        out = []
        for g in range(self.groups):
            hyps = []
            for b in range(self.beams):
                r = g * self.beams + b
                if score[g][b] > float("-inf"):
                    hyps.append(Hypothesis(tokens[r][: length[r]], score[g][b], ended[g][b]))
            out.append(hyps)
        return out
