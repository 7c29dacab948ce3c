"""Serving loop over a device model of either kind: sessions, portions of prompts, decode batches, sampling.

The unit of work is `Engine.advance`: some sessions take their next tokens, from the cache and state that earlier
steps left.  Sessions with one token each go through one decode pass per WR_BATCH_MAX sessions
(include/wayruntime/wayruntime.h:423); a session with more goes through prefill passes of at most the model's
max_rows rows.  `Engine.step` schedules queued requests on top of it: one portion of a waiting prompt, then one
decode pass over the running requests.
"""
from __future__ import annotations

import itertools
from collections import deque
from dataclasses import dataclass, field

import numpy as np

from .binding import BATCH_MAX, BEAM_MAX_OUT, NO_BEAM


@dataclass
class Sampling:
    """temperature 0: greedy (the lowest id wins a tie, as the reference's arg-max does, src/cli/wayrt.c:805)."""
    temperature: float = 0.0
    top_k: int = 0
    top_p: float = 1.0
    seed: int = 0


class Session:
    """One sequence: its cache and how many tokens it holds."""

    def __init__(self, model, max_ctx: int):
        self.kv = model.kv_create(max_ctx)
        self.max_ctx, self.pos = max_ctx, 0

    def close(self):
        self.kv.close()

    def fork(self) -> "Session":
        """A session that goes on from here; what both hold is kept once, page by page."""
        s = Session.__new__(Session)
        s.kv, s.max_ctx, s.pos = self.kv.fork(self.pos), self.max_ctx, self.pos
        return s


@dataclass
class Hypothesis:
    """A continuation that a beam search has found: its tokens and the sum of their log probabilities."""
    tokens: list
    score: float

    def rank(self, length_penalty: float) -> float:
        return self.score / len(self.tokens) ** length_penalty


@dataclass
class Request:
    prompt: list
    max_new: int
    sampling: Sampling = field(default_factory=Sampling)
    stop: frozenset = frozenset()
    id: int = 0
    output: list = field(default_factory=list)
    done: bool = False
    session: Session | None = None
    _rng: object = None


def sample(logits: np.ndarray, s: Sampling, rng) -> int:
    """One token id from a row of logits."""
    if s.temperature <= 0:
        return int(np.argmax(logits))
    z = logits.astype(np.float64) / s.temperature
    order = np.argsort(-z, kind="stable")
    if s.top_k > 0:
        order = order[:s.top_k]
    p = np.exp(z[order] - z[order[0]])
    p /= p.sum()
    if s.top_p < 1.0:
        keep = int(np.searchsorted(np.cumsum(p), s.top_p) + 1)
        order, p = order[:keep], p[:keep] / p[:keep].sum()
    return int(order[np.searchsorted(np.cumsum(p), rng.random() * p.sum(), side="right").clip(0, len(p) - 1)])


class Engine:
    def __init__(self, model, max_sessions: int = BATCH_MAX, portion: int | None = None):
        self.model = model
        self.max_sessions = max_sessions
        self.portion = min(portion or model.max_rows, model.max_rows)
        self.waiting, self.running = deque(), []
        self._ids = itertools.count()

    # ---- the step function

    def session(self, max_ctx: int) -> Session:
        return Session(self.model, max_ctx)

    def advance(self, sessions, tokens, want=None, argmax=False):
        """Run tokens[i] (a list of ids) on sessions[i].  want[i]: places among them whose logits are returned,
        default the last one; the result is one array [len(want[i]), vocab] per session — or, with argmax, the id of
        the first maximum after each session's last token."""
        want = [[len(t) - 1] for t in tokens] if want is None else want
        out = [None] * len(sessions)
        single = [i for i, t in enumerate(tokens) if len(t) == 1]
        for lo in range(0, len(single), BATCH_MAX):
            self._decode(single[lo:lo + BATCH_MAX], sessions, tokens, want, argmax, out)
        for i, t in enumerate(tokens):
            if len(t) > 1:
                out[i] = self._prefill(sessions[i], t, want[i], argmax)
        return out

    def _decode(self, rows, sessions, tokens, want, argmax, out):
        m = self.model
        asked = [j for j, i in enumerate(rows) if len(want[i])]
        own = {"apart": True} if asked and not argmax and getattr(m, "ROWS_APART", False) else {}
        res = m.forward(m.FWD_DECODE, [sessions[i].kv for i in rows], [sessions[i].pos for i in rows],
                        [tokens[i][0] for i in rows], logits=False if argmax else asked, argmax=argmax, **own)
        for j, i in enumerate(rows):
            sessions[i].pos += 1
            if argmax:
                out[i] = int(res["argmax"][j])
            elif j in asked:
                at = asked.index(j)
                row = res["logits"][at] if own else res["logits"][at:at + 1]
                out[i] = row if len(want[i]) == 1 else row.repeat(len(want[i]), axis=0)
            else:
                out[i] = np.empty((0, m.vocab), np.float32)

    def _prefill(self, s, tokens, want, argmax):
        m, parts = self.model, []
        rows_max = m.max_rows
        order = sorted(set(want))                    # (asked in any order, computed front to back, each once)
        for lo in range(0, len(tokens), rows_max):
            part = tokens[lo:lo + rows_max]
            last = lo + len(part) == len(tokens)
            here = [w - lo for w in order if lo <= w < lo + len(part)]
            if argmax:
                res = m.forward(m.FWD_PREFILL, [s.kv], [s.pos], part, out_from=len(part) - 1, argmax=last)
            elif here:
                first = here[0]
                res = m.forward(m.FWD_PREFILL, [s.kv], [s.pos], part, out_from=first, logits=[w - first for w in here])
                parts.append(res["logits"])
            else:
                res = m.forward(m.FWD_PREFILL, [s.kv], [s.pos], part, out_from=len(part))
            s.pos += len(part)
        if argmax:
            return int(res["argmax"][0])
        if not parts:
            return np.empty((0, m.vocab), np.float32)
        rows = parts[0] if len(parts) == 1 else np.concatenate(parts)
        return rows if order == list(want) else rows[[order.index(w) for w in want]]

    # ---- beam search

    def beam_search(self, prompt, beams: int, max_new: int, stop=frozenset(), length_penalty: float = 1.0) -> list:
        """The best continuations of a prompt, at most `beams`, as Hypothesis, by score / length ** length_penalty.  One ends
        with a stop id or after max_new tokens; the search ends when `beams` have ended and none that goes on ranks above
        the last of them as it stands.  The beams' sessions are forks of the prompt's: its pages are kept once, and a step
        attends to them once for all beams where the model's stack does that (wr_cuda_model_beam_step).  Any number of stop ids: a step that
        may have to pass over more of them than one choice on the device has places for chooses per beam (beams + stop ids at most
        32), beyond that on the host."""
        stop = frozenset(stop)
        if not prompt or max_new < 1:
            raise ValueError("a prompt token and a new one at least")
        if not 1 <= beams <= BATCH_MAX:
            raise ValueError(f"1 to {BATCH_MAX} beams")
        sessions, histories, ended = [self.session(len(prompt) + max_new)], [[]], []
        rank = lambda h: h.rank(length_penalty)  # noqa: E731
        try:
            if len(prompt) > 1:
                self.advance(sessions, [prompt[:-1]], [[]])
            tokens, scores = [prompt[-1]], [0.0]
            while True:
                live = sessions[:len(tokens)]
                found = self._continuations(live, tokens, scores, beams, len(stop))
                for s in live:
                    s.pos += 1
                going = []                               # (score, parent, token), best first
                for place, (score, parent, token) in enumerate(found):
                    if len(going) == beams:
                        break
                    if token not in stop:
                        going.append((score, parent, token))
                    elif place < beams:
                        ended.append(Hypothesis(histories[parent] + [token], score))
                length = len(histories[0]) + 1
                if length == max_new:
                    ended += [Hypothesis(histories[p] + [t], s) for s, p, t in going]
                    break
                ended = sorted(ended, key=rank, reverse=True)[:beams]
                if not going or (len(ended) == beams and rank(ended[-1]) >= going[0][0] / length ** length_penalty):
                    break
                parents = [p for _, p, _ in going]
                self._follow(sessions, parents, beams)
                histories = [histories[p] + [t] for _, p, t in going]
                tokens, scores = [t for _, _, t in going], [s for s, _, _ in going]
        finally:
            for s in sessions:
                s.close()
        return sorted(ended, key=rank, reverse=True)[:beams]

    def _continuations(self, live, tokens, scores, beams, stops):
        """A step of all live beams, and its continuations as (score, parent, token), best first: as far as `beams` that are not among
        `stops` ids lie."""
        m, kvs, at, places = self.model, [s.kv for s in live], [s.pos for s in live], (1 + stops) * beams
        if places <= BEAM_MAX_OUT:
            found = zip(*(x[0].tolist() for x in m.beam_step(kvs, at, tokens, [scores], places)))
            return [c for c in found if c[1] != NO_BEAM]
        # More places than one choice has: from every beam as many as can be among them, put together here.  (Of one beam's, `beams` are none
        # of the stop ids behind which the others lie.)
        each = beams + stops
        if each <= BEAM_MAX_OUT:
            s, b, t = (x.tolist() for x in m.beam_step(kvs, at, tokens, [[x] for x in scores], each))
            found = [(s[p][i], p, t[p][i]) for p in range(len(live)) for i in range(each) if b[p][i] != NO_BEAM]
        else:
            found = []
            for p, row in enumerate(m.forward(m.FWD_DECODE, kvs, at, tokens, logits=True)["logits"]):
                row = row.astype(np.float64)
                top = row.max()
                if not np.isfinite(top):                 # (no continuation, or a logit that is not a number)
                    continue
                total = scores[p] + (row - (top + np.log(np.exp(row - top).sum())))
                least = np.partition(total, -each)[-each] if each < len(total) else -np.inf
                best = np.flatnonzero((total >= least) & (row > -np.inf))
                best = best[np.argsort(-total[best], kind="stable")][:each]
                found += [(float(total[t]), p, int(t)) for t in best]
        found.sort(key=lambda c: -c[0])                  # (stable: equal ones by beam, then token)
        return [(float(np.float32(s)), p, t) for s, p, t in found[:places]]

    def _follow(self, sessions, parents, beams):
        """Sessions [0, len(parents)) go on from those that parents names.  The others wait until there are more beams again."""
        if len(sessions) < beams:                        # (the prompt's session: every beam goes on from it)
            sessions += [sessions[0].fork() for _ in range(1, beams)]
            return
        spare = [i for i in range(beams) if i not in parents]            # (nobody goes on from these: who waits takes them)
        order, at = parents + spare[:beams - len(parents)], [s.pos for s in sessions]
        if order != list(range(beams)):
            self.model.kv_reorder([s.kv for s in sessions], order, at)
            for s, p in zip(sessions, order):
                s.pos = at[p]

    # ---- scheduling

    def submit(self, request: Request) -> Request:
        if not request.prompt:
            raise ValueError("a request needs at least one prompt token")
        request.id = next(self._ids)
        request._rng = np.random.default_rng(request.sampling.seed)
        self.waiting.append(request)
        return request

    def step(self) -> list:
        """One portion of the first waiting prompt (when a session is free), then one token for every running
        request; returns the requests that finished."""
        if self.waiting and len(self.running) < self.max_sessions:
            r = self.waiting[0]
            if r.session is None:
                r.session = self.session(len(r.prompt) + r.max_new)
            s = r.session
            part = r.prompt[s.pos:s.pos + self.portion]
            if s.pos + len(part) < len(r.prompt):
                self.advance([s], [part], [[]])
            else:
                self.waiting.popleft()
                self.running.append(r)
                self._take(r, self._next([r], [part])[0])
        ready = [r for r in self.running if not r.done]
        if ready:
            for r, t in zip(ready, self._next(ready, [[r.output[-1]] for r in ready])):
                self._take(r, t)
        finished = [r for r in self.running if r.done]
        self.running = [r for r in self.running if not r.done]
        for r in finished:
            r.session.close()
            r.session = None
        return finished

    def _next(self, reqs, tokens):
        sessions = [r.session for r in reqs]
        if all(r.sampling.temperature <= 0 for r in reqs):
            return self.advance(sessions, tokens, argmax=True)
        rows = self.advance(sessions, tokens)
        return [sample(row[-1], r.sampling, r._rng) for r, row in zip(reqs, rows)]

    def _take(self, r, token):
        r.output.append(token)
        if len(r.output) >= r.max_new or token in r.stop:
            r.done = True

    def run(self, requests) -> list:
        """Submit, step until all are done, return the requests."""
        for r in requests:
            self.submit(r)
        while self.waiting or self.running:
            self.step()
        return requests
