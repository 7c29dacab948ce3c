"""GPU: beam search with more stop ids than one choice on the device has places for."""
import numpy as np
import pytest

from _plain_beams import choose, choose_error
from test_gpu_beam_search import alone, ctx, dense, prompt_of, tumadra  # noqa: F401 (ctx: a fixture)

pytestmark = pytest.mark.gpu


def plain_search(engine, prompt, beams, max_new, stop):
    """Every hypothesis on a session of its own, all places looked at."""
    live, ended, size = [([], 0.0)], [], len(prompt) + max_new
    n_out, largest = (1 + len(stop)) * beams, 1.0
    rank = lambda h: h[1] / len(h[0])  # noqa: E731
    for step in range(1, max_new + 1):
        rows = np.stack([alone(engine, prompt, h, size) for h, _ in live])
        largest = max(largest, float(np.abs(rows).max()))
        s, b, t = (x[0] for x in choose(rows[None], np.array([[s for _, s in live]]), n_out))
        going = []
        for place in range(n_out):
            if b[place] == 0xFFFFFFFF or len(going) == beams:
                break
            h = (live[b[place]][0] + [int(t[place])], s[place])
            if t[place] not in stop:
                going.append(h)
            elif place < beams:
                ended.append(h)
        if step == max_new:
            ended += going
            break
        live, ended = going, sorted(ended, key=rank, reverse=True)[:beams]
        if not live or len(ended) == beams and rank(ended[-1]) >= live[0][1] / step:
            break
    return sorted(ended, key=rank, reverse=True)[:beams], largest


@pytest.mark.parametrize("build", [dense, tumadra])
@pytest.mark.parametrize("n, beams, stops", [(40, 16, 3), (300, 9, 5), (300, 5, 40)])
def test_search_with_many_stop_ids(ctx, build, n, beams, stops):  # noqa: F811
    from wayruntime_b200.engine import Engine
    m = build(ctx)
    engine, prompt, max_new = Engine(m), prompt_of(n, n, m.vocab), 4
    # the most probable first tokens of the prompt, every other one of them
    first = alone(engine, prompt, [], n + max_new)
    stop = frozenset(int(t) for t in np.argsort(-first, kind="stable")[:2 * stops:2])
    got = engine.beam_search(prompt, beams, max_new, stop)
    want, largest = plain_search(engine, prompt, beams, max_new, stop)
    assert [h.tokens for h in got] == [t for t, _ in want]
    for h, (_, s) in zip(got, want):
        # Each step's total: rounded, its sum within choose_error, and, where attention goes another way (the dense stack's, together), the
        # logit and the sum off by 1e-4 of the largest logit each: 1e-5 of a row's norm in each of two layers' attention (both ways within
        # 5e-6 of 64 bits), which the two factors of a feed-forward and the norms before it and the head double at most each.
        bound = len(h.tokens) * (choose_error(np.array([s]), m.vocab)[0] + (2e-4 * largest if build is dense else 0.0))
        assert abs(h.score - s) <= bound
    m.close()
