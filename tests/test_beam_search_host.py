"""Host logic of beam search without a device: Engine.beam_search over a fake model, and what the Python calls refuse."""
import itertools

import numpy as np
import pytest

from _plain_beams import choose
from wayruntime_b200 import binding
from wayruntime_b200.engine import Engine, Hypothesis


class FakeModel:
    """Logits that hang on everything a session has seen; sessions are lists of tokens."""
    FWD_DECODE, FWD_PREFILL, max_rows = 0, 1, 8

    def __init__(self, vocab, spread=1.0):
        self.vocab, self.spread, self.live, self.reorders = vocab, spread, 0, []

    def kv_create(self, max_ctx):
        self.live += 1
        return FakeKV(self, [], max_ctx)

    def logits(self, seen):
        rng = np.random.default_rng([hash(tuple(seen)) & 0xFFFFFFFF, len(seen)])
        return (rng.standard_normal(self.vocab) * self.spread).astype(np.float32)

    def forward(self, mode, kvs, positions, tokens, out_from=0, *, logits=False, argmax=False):
        assert positions == [len(kvs[0].seen)]
        kvs[0].seen += tokens
        return {"logits": np.zeros((0, self.vocab), np.float32)}

    def beam_step(self, kvs, positions, tokens, scores, n_out):
        assert len({id(k) for k in kvs}) == len(kvs) == len(positions) == len(tokens)
        for kv, p, t in zip(kvs, positions, tokens):
            assert p == len(kv.seen) < kv.cap
            kv.seen.append(t)
        scores = np.asarray(scores, np.float32)
        s, b, t = choose(np.stack([self.logits(kv.seen) for kv in kvs]).reshape(*scores.shape, -1), scores, n_out)
        return s.astype(np.float32), b, t

    def kv_reorder(self, kvs, parents, rows):
        assert rows == [len(kv.seen) for kv in kvs] and len(parents) == len(kvs)
        self.reorders.append(parents)
        held = [list(kv.seen) for kv in kvs]
        for kv, p in zip(kvs, parents):
            kv.seen = list(held[p])


class FakeKV:
    def __init__(self, model, seen, cap):
        self.model, self.seen, self.cap = model, seen, cap

    def fork(self, n):
        assert n == len(self.seen)
        self.model.live += 1
        return FakeKV(self.model, list(self.seen), self.cap)

    def close(self):
        self.model.live -= 1


def log_probs(model, seen):
    x = model.logits(seen).astype(np.float64)
    return x - x.max() - np.log(np.exp(x - x.max()).sum())


def plain_search(model, prompt, beams, max_new, stop, penalty):
    """The same search over whole sequences."""
    live, ended, n_out = [([], 0.0)], [], (1 + len(stop)) * beams
    for step in range(1, max_new + 1):
        found = sorted(((s + lp, i, t) for i, (h, s) in enumerate(live) for t, lp in enumerate(log_probs(model, prompt + h))),
                       key=lambda c: (-c[0], c[1], c[2]))[:n_out]
        going = []
        for place, (s, i, t) in enumerate(found):
            if len(going) == beams:
                break
            if t not in stop:
                going.append((live[i][0] + [t], s))
            elif place < beams:
                ended.append((live[i][0] + [t], s))
        if step == max_new:
            ended += going
            break
        live = going
        ended = sorted(ended, key=lambda h: -h[1] / len(h[0]) ** penalty)[:beams]
        if not live or len(ended) == beams and ended[-1][1] / len(ended[-1][0]) ** penalty >= live[0][1] / step ** penalty:
            break
    return sorted(ended, key=lambda h: -h[1] / len(h[0]) ** penalty)[:beams]


@pytest.mark.parametrize("beams, vocab, max_new, stop, penalty", [
    (1, 50, 6, [], 1.0), (4, 50, 8, [], 1.0), (4, 50, 8, [3], 1.0), (3, 12, 10, [0, 5], 0.6), (8, 9, 5, [1], 2.0), (16, 40, 4, [], 0.0),
    (5, 3, 6, [2], 1.0), (4, 2, 3, [], 1.0), (6, 4, 7, [0, 1, 2], 1.0), (2, 30, 1, [4], 1.0), (4, 1, 3, [], 1.0), (2, 3, 4, [0, 1, 2], 1.0)])
@pytest.mark.parametrize("prompt", [[7], list(range(20))])
def test_the_search_is_that_over_whole_sequences(beams, vocab, max_new, stop, penalty, prompt):
    m = FakeModel(vocab)
    got = Engine(m).beam_search(prompt, beams, max_new, stop, penalty)
    want = plain_search(m, prompt, beams, max_new, frozenset(stop), penalty)
    assert [h.tokens for h in got] == [t for t, _ in want]
    assert np.allclose([h.score for h in got], [s for _, s in want], rtol=0, atol=1e-5)
    assert m.live == 0


def test_one_beam_is_the_greedy_choice():
    m = FakeModel(30)
    seen, want = [5, 6], []
    for _ in range(6):
        want.append(int(np.argmax(m.logits(seen))))
        seen = seen + want[-1:]
    assert Engine(m).beam_search([5, 6], 1, 6)[0].tokens == want and not m.reorders


def test_sessions_are_closed_when_a_step_fails():
    m = FakeModel(30)
    m.kv_reorder = None
    with pytest.raises(TypeError):
        Engine(m).beam_search([5, 6], 4, 9)
    assert m.live == 0


@pytest.mark.parametrize("prompt, beams, max_new", [([], 2, 3), ([1], 0, 3), ([1], 17, 3), ([1], 2, 0)])
def test_what_a_search_refuses(prompt, beams, max_new):
    with pytest.raises(ValueError):
        Engine(FakeModel(9)).beam_search(prompt, beams, max_new)


def test_ranks():
    h = Hypothesis([1, 2, 3, 4], -6.0)
    assert h.rank(0.0) == -6.0 and h.rank(1.0) == -1.5 and h.rank(0.5) == -3.0


def test_groups_add_up_to_the_sessions():
    g = binding.Groups([(3, 64), (1, 0)])
    assert len(g) == 2 and list(g.sessions) == [3, 1] and list(g.rows) == [64, 0]
    assert binding.Groups.of(g, 4) is g
    with pytest.raises(ValueError):
        binding.Groups.of([(3, 64)], 4)


def test_null_arguments_are_refused_without_a_device():
    import ctypes as C
    from wayruntime_b200 import _build
    _build.build()
    lib = binding.load_library()
    out = C.c_void_p()
    assert lib.wr_cuda_kv_fork(None, None, 0, C.byref(out)) == -4
    assert lib.wr_cuda_kv_reorder(None, 1, None, None, None) == -4
    assert lib.wr_cuda_kv_shared_rows(None, None) == 0
    assert lib.wr_cuda_attn_decode_shared(None, 1, None, 0, None, 1, None, None, None, None, 1, 0.0, 0) == -4
    assert lib.wr_cuda_decode_step_shared(None, 1, None, 0, None, 1, None, None, None, None, None, None, 1, 1e4, 0, 0, 0.0, 0) == -4
    assert lib.wr_cuda_beam_select(None, 1, 1, 1, None, None, 1, None, None, None, 0) == -4
    assert lib.wr_cuda_model_beam_step(None, None, 1, 1, None, None, None, None, 1, None, None, None) == -4


def test_command_line_refuses_temperature_with_beams(capsys):
    from wayruntime_b200 import cli
    with pytest.raises(SystemExit):
        cli.main(["generate", "--model", "x", "--prompt", "1", "--beams", "2", "--temperature", "0.5"])
    assert "--beams" in capsys.readouterr().err
