"""GPU: beam search through the serving loop on every stack, against a search whose hypotheses each have a session of their
own that is run token by token; and decode passes over sessions that hold pages together."""
import json
import subprocess
import sys

import numpy as np
import pytest

import _nurosun_models as nuro
import _tumadra_models as tuma
from _plain_beams import choose, choose_error
from test_gpu_model_glue import SHAPE, _model, _weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import wayruntime_b200 as wr
    c = wr.Context(0, attn_max_seq=4096)
    yield c
    c.close()


def dense(ctx, layers=2, qk_norm=True, **kw):
    shape = dict(SHAPE, n_layers=layers)
    return _model(ctx, _weights(shape, 700, qk_norm=qk_norm), shape, **kw)


def tumadra(ctx):
    from wayruntime_b200 import models
    cfg = tuma.config([tuma.with_mlp(tuma.mamba(), 40), tuma.with_mlp(tuma.attn(), 40)], loop=(0, 2, 2))
    return models.build(ctx, cfg, tuma.Weights(tuma.weights(cfg, 3)), "float32", 64)


def nurosun(ctx):
    from wayruntime_b200 import models
    cfg = nuro.config([nuro.latent(mlp=nuro.dense(40)), nuro.latent(source=0, mlp=nuro.moe())])
    return models.build(ctx, cfg, nuro.Weights(nuro.weights(cfg, 3)), "float32", 64)


def alone(engine, prompt, tokens, max_ctx):
    """Logits after prompt + tokens on a session of its own, the steps one token at a time."""
    m, s = engine.model, engine.session(max_ctx)
    if len(prompt) > 1:
        engine.advance([s], [prompt[:-1]], [[]])
    for t in prompt[-1:] + tokens:
        row = m.forward(m.FWD_DECODE, [s.kv], [s.pos], [t], logits=True)["logits"][0]
        s.pos += 1
    s.close()
    return row


def plain_search(engine, prompt, beams, max_new, stop):
    live, ended, n_out, size = [([], 0.0)], [], min((1 + len(stop)) * beams, 32), len(prompt) + max_new
    largest = 1.0
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
        rank = lambda h: h[1] / len(h[0])  # noqa: E731
        if step == max_new:
            ended += going
            break
        live, ended = going, sorted(ended, key=rank, reverse=True)[:beams]
        if not live or len(ended) == beams and rank(ended[-1]) >= live[0][1] / step:
            break
    return sorted(ended, key=rank, reverse=True)[:beams], largest


def compare(engine, prompt, beams, max_new, stop=(), rel=0.0):
    """rel: how far a decode step's logits may be off, of their largest, where attention goes another way."""
    got = engine.beam_search(prompt, beams, max_new, stop)
    want, largest = plain_search(engine, prompt, beams, max_new, frozenset(stop))
    assert [h.tokens for h in got] == [t for t, _ in want]
    for h, (_, s) in zip(got, want):
        # each step's total: rounded, its sum within choose_error, and both the logit and the sum off by rel
        bound = len(h.tokens) * (choose_error(np.array([s]), engine.model.vocab)[0] + 2 * rel * largest)
        assert abs(h.score - s) <= bound


def prompt_of(seed, n, vocab):
    return [int(t) for t in np.random.default_rng(seed).integers(0, vocab, n)]


@pytest.mark.parametrize("n, beams, max_new", [(1, 4, 5), (2, 3, 4), (70, 4, 6), (257, 4, 5), (300, 1, 4), (321, 8, 12), (700, 16, 4), (1300, 4, 5)])
def test_dense_stack(ctx, n, beams, max_new):
    from wayruntime_b200.engine import Engine
    m = dense(ctx)
    before = m.launches
    compare(Engine(m), prompt_of(n, n, m.vocab), beams, max_new, rel=1e-4)
    assert m.launches > before
    m.close()


def test_dense_stack_without_head_norms_and_with_stop_ids(ctx):
    from wayruntime_b200.engine import Engine
    m = dense(ctx, qk_norm=False, max_rows=128)
    engine, prompt = Engine(m), prompt_of(5, 330, 1003)
    free = engine.beam_search(prompt, 4, 6)
    stop = {free[0].tokens[2], free[1].tokens[3]}
    compare(engine, prompt, 4, 6, stop, rel=1e-4)
    m.close()


@pytest.mark.parametrize("build", [tumadra, nurosun])
@pytest.mark.parametrize("n, beams, max_new", [(1, 3, 5), (63, 4, 5), (64, 2, 3), (150, 5, 70)])
def test_mixed_stack(ctx, build, n, beams, max_new):
    """(the same kernels whoever holds the pages: the sums of a pass are the same)"""
    from wayruntime_b200.engine import Engine
    m = build(ctx)
    if max_new > 10:                                     # a long search: every hypothesis by itself is too slow, its own sum is checked
        engine, prompt = Engine(m), prompt_of(n, n, m.vocab)
        for h in engine.beam_search(prompt, beams, max_new):
            total, s = 0.0, engine.session(n + max_new)
            engine.advance([s], [prompt[:-1]], [[]])
            for t, following in zip(prompt[-1:] + h.tokens, h.tokens):
                row = m.forward(m.FWD_DECODE, [s.kv], [s.pos], [t], logits=True)["logits"][0].astype(np.float64)
                s.pos += 1
                total += row[following] - row.max() - np.log(np.exp(row - row.max()).sum())
            s.close()
            assert abs(h.score - total) <= max_new * choose_error(np.array([total]), m.vocab)[0]
    else:
        compare(Engine(m), prompt_of(n, n, m.vocab), beams, max_new)
    m.close()


def test_decode_pass_over_families_and_others(ctx):
    """Two families, one of them with a short beginning, and sessions by themselves, in an order that mixes them."""
    m = dense(ctx)
    V = m.vocab

    def started(seed, n):
        kv = m.kv_create(1400)
        toks = prompt_of(seed, n, V)
        for lo in range(0, n, m.max_rows):
            part = toks[lo:lo + m.max_rows]
            m.forward(m.FWD_PREFILL, [kv], [lo], part, out_from=len(part))
        return kv
    a, b, c, d, e = started(1, 400), started(2, 1200), started(3, 90), started(4, 1100), started(5, 30)
    fa, fb, fc = [a.fork(400) for _ in range(2)], b.fork(1200), c.fork(90)
    kvs = [e, fa[0], b, c, fa[1], d, fc, a, fb]
    pos = [30, 400, 1200, 90, 400, 1100, 90, 400, 1200]
    toks = prompt_of(9, 9, V)
    want = [m.forward(m.FWD_DECODE, [kv], [p], [t], hidden=True, logits=True, attn_tap=True) for kv, p, t in zip(kvs, pos, toks)]
    got = m.forward(m.FWD_DECODE, kvs, pos, toks, hidden=True, normed=True, logits=True, argmax=True, attn_tap=True)
    for i, w in enumerate(want):
        for key, mine in (("hidden", got["hidden"][i]), ("logits", got["logits"][i])):
            assert np.abs(mine - w[key][0]).max() <= 1e-4 * max(1.0, np.abs(w[key]).max()), (i, key)
        assert np.abs(got["attn"][:, i] - w["attn"][:, 0]).max() <= 1e-4
        assert got["argmax"][i] == np.argmax(got["logits"][i])
        if i in (0, 3, 5, 6):                            # those that hold nothing long together go the way they went
            assert np.array_equal(got["logits"][i], w["logits"][0])
    for kv in kvs:
        kv.close()
    m.close()


def test_beam_step_chooses_from_the_passs_logits(ctx):
    m = dense(ctx)
    kvs = [m.kv_create(64) for _ in range(6)]
    toks, scores = prompt_of(3, 6, m.vocab), np.array([[-1.0, -2.0, -1.5], [-3.0, -np.inf, -0.5]], np.float32)
    rows = m.forward(m.FWD_DECODE, kvs, [0] * 6, toks, logits=True)["logits"]
    for n_out in (1, 6, 32):
        got = m.beam_step(kvs, [0] * 6, toks, scores, n_out)
        want = choose(rows.reshape(2, 3, -1), scores, n_out)
        assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
        assert (np.abs(got[0] - want[0]) <= choose_error(want[0], m.vocab)).all()
    for kv in kvs:
        kv.close()
    m.close()


@pytest.mark.parametrize("build", [dense, tumadra])
def test_refusals_consume_nothing(ctx, build):
    import wayruntime_b200 as wr
    m = build(ctx)
    kv = m.kv_create(200)
    toks = prompt_of(4, 130, m.vocab)
    for lo in range(0, 130, 64):
        m.forward(m.FWD_PREFILL, [kv], [lo], toks[lo:lo + 64], out_from=len(toks[lo:lo + 64]))
    f = kv.fork(130)
    want = m.forward(m.FWD_DECODE, [kv], [130], [5], logits=True)["logits"]

    def status(call):
        with pytest.raises(wr.WrCudaError) as e:
            call()
        return e.value.status
    one = np.zeros((1, 1), np.float32)
    assert status(lambda: m.beam_step([f], [130], [5], one, 33)) == -8
    assert status(lambda: m.beam_step([f], [130], [5], one, 0)) == -4
    assert status(lambda: m.beam_step([f], [130], [m.vocab], one, 4)) == -4
    assert status(lambda: m.beam_step([f], [200], [5], one, 4)) == -6
    assert status(lambda: m.forward(m.FWD_DECODE, [f], [0], [5])) == -7           # what both hold is not written
    assert status(lambda: m.forward(m.FWD_PREFILL, [f], [0], toks[:3])) == -7
    with pytest.raises(ValueError):
        m.beam_step([f], [130, 131], [5], one, 4)
    if build is tumadra:
        assert status(lambda: kv.fork(64)) == -7                                  # the recurrent state does not stand there
        assert status(lambda: m.kv_reorder([kv, f], [1, 1], [131, 64])) == -7
    assert np.array_equal(m.forward(m.FWD_DECODE, [f], [130], [5], logits=True)["logits"], want)
    kv.close()
    f.close()
    m.close()


def test_command_line(tmp_path, ctx):
    from wayruntime_b200 import checkpoint
    from wayruntime_b200.engine import Engine
    from wayruntime_b200 import models
    cfg = tuma.config([tuma.with_mlp(tuma.mamba(), 40), tuma.with_mlp(tuma.attn(), 40)])
    checkpoint.save(str(tmp_path), cfg, tuma.weights(cfg, 5))
    out = subprocess.run([sys.executable, "-m", "wayruntime_b200.cli", "generate", "--model", str(tmp_path), "--dtype", "float32",
                          "--prompt", "3,1,4,1,5", "--beams", "3", "--max-new", "6"], capture_output=True, text=True, check=True)
    said = json.loads(out.stdout)
    m = models.load(ctx, str(tmp_path), "float32", 2048)
    want = Engine(m).beam_search([3, 1, 4, 1, 5], 3, 6)
    m.close()
    assert said["output"] == want[0].tokens and [b["output"] for b in said["beams"]] == [h.tokens for h in want]
