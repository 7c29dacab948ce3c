"""Host logic of beam search with more stop ids than one choice on the device has places for."""
import numpy as np
import pytest

from test_beam_search_host import FakeModel, plain_search
from wayruntime_b200.engine import Engine


class Stopping(FakeModel):
    """The stop ids are probable: they take many of a step's first places."""

    def __init__(self, vocab, stop, raised):
        super().__init__(vocab)
        self.stop, self.raised, self.passes = sorted(stop), raised, 0

    def logits(self, seen):
        x = super().logits(seen)
        x[self.stop] += np.float32(self.raised)
        return x

    def forward(self, mode, kvs, positions, tokens, out_from=0, *, logits=False, argmax=False):
        if logits is not True:                           # (the prompt)
            return super().forward(mode, kvs, positions, tokens, out_from, logits=logits, argmax=argmax)
        assert mode == self.FWD_DECODE and positions == [len(kv.seen) for kv in kvs]
        self.passes += 1
        for kv, t in zip(kvs, tokens):
            kv.seen.append(t)
        return {"logits": np.stack([self.logits(kv.seen) for kv in kvs])}


def compare(m, prompt, beams, max_new, stop):
    got = Engine(m).beam_search(prompt, beams, max_new, stop)
    want = plain_search(m, prompt, beams, max_new, frozenset(stop), 1.0)
    assert [h.tokens for h in got] == [t for t, _ in want]
    assert np.allclose([h.score for h in got], [s for _, s in want], rtol=0, atol=1e-5)
    assert m.live == 0


@pytest.mark.parametrize("raised", [1.0, 2.0, 4.0])
@pytest.mark.parametrize("beams, stops", [(16, 2), (16, 3), (8, 4), (11, 2), (12, 6), (16, 16)])
def test_stop_ids_take_no_place_from_the_beams_that_go_on(beams, stops, raised):
    for seed in range(5):
        rng = np.random.default_rng([beams, stops, seed])
        stop = [int(t) for t in rng.choice(60, stops, replace=False)]
        m = Stopping(60, stop, raised)
        compare(m, [int(t) for t in rng.integers(0, 60, 3)], beams, 5, stop)
        assert not m.passes


@pytest.mark.parametrize("beams, stops", [(16, 17), (4, 40), (1, 33), (16, 59), (16, 60)])
def test_more_stop_ids_than_a_choice_has_places(beams, stops):
    """(a choice on the host)"""
    for seed in range(2):
        rng = np.random.default_rng([beams, stops, seed])
        stop = [int(t) for t in rng.choice(60, stops, replace=False)]
        m = Stopping(60, stop, 2.0)
        compare(m, [int(t) for t in rng.integers(0, 60, 3)], beams, 5, stop)
        assert m.passes


@pytest.mark.parametrize("beams, stops", [(3, 33), (16, 4)])
def test_rows_that_are_masked_or_not_numbers(beams, stops):
    """A row of -inf or with a NaN or an infinity has no continuations, and the other beams go on without it."""
    class Spoilt(Stopping):
        def logits(self, seen):
            x = super().logits(seen)
            kind = (sum(seen) + len(seen)) % 5 if len(seen) > 2 else 0
            if kind == 1:
                x[:] = -np.inf
            elif kind in (2, 3):
                x[7] = (np.nan, np.inf)[kind - 2]
            elif kind == 4:
                x[::2] = -np.inf
            return x

    stop = list(range(100, 100 + stops))
    m = Spoilt(200, stop, 1.0)
    got = Engine(m).beam_search([1, 2], beams, 5, stop)
    assert got and m.live == 0
    for h in got:                                        # no token of a spoilt row, and the sum of its tokens' log probabilities
        total, seen = 0.0, [1, 2]
        for t in h.tokens:
            x = m.logits(seen).astype(np.float64)
            assert np.isfinite(x.max()) and np.isfinite(x[t])
            total += x[t] - x.max() - np.log(np.exp(x - x.max()).sum())
            seen = seen + [t]
        assert abs(h.score - total) <= 1e-5
