"""GPU: model passes over sessions that hold pages together: what they refuse, and whom a session's result hangs on."""
import numpy as np
import pytest

from test_gpu_beam_search import ctx, dense, prompt_of  # noqa: F401 (ctx: a fixture)

pytestmark = pytest.mark.gpu


def started(m, seed, n, max_ctx=1400):
    kv, toks = m.kv_create(max_ctx), prompt_of(seed, n, m.vocab)
    for lo in range(0, n, m.max_rows):
        part = toks[lo:lo + m.max_rows]
        m.forward(m.FWD_PREFILL, [kv], [lo], part, out_from=len(part))
    return kv


@pytest.mark.parametrize("n", [30, 400, 1100])
def test_a_session_given_twice_is_refused(ctx, n):  # noqa: F811
    """Short sessions, long ones, members of a family: whichever kinds of rows the pass would divide them into."""
    import wayruntime_b200 as wr
    m = dense(ctx)
    a = started(m, n, n)
    f, other = a.fork(n), started(m, n + 1, 20)
    want = m.forward(m.FWD_DECODE, [a], [n], [7], logits=True)["logits"]
    a.n_kv_heads, a.head_dim = 2, 128
    rows = [a.read_rows(layer, which, 0, n + 1) for layer in range(2) for which in (0, 1)]
    for kvs, pos in (([a, f, a], [n] * 3), ([a, a], [n] * 2), ([a, a, f], [n, n - 1, n]), ([other, a, f, other], [20, n, n, 20]),
                     ([f, other, a, f], [n, 20, n, n])):
        with pytest.raises(wr.WrCudaError) as e:
            m.forward(m.FWD_DECODE, kvs, pos, list(range(3, 3 + len(kvs))), logits=True)
        assert e.value.status == -4
        with pytest.raises(wr.WrCudaError) as e:
            m.beam_step(kvs, pos, list(range(3, 3 + len(kvs))), np.zeros((1, len(kvs)), np.float32), 4)
        assert e.value.status == -4
    assert all(np.array_equal(a.read_rows(layer, which, 0, n + 1), rows[2 * layer + which]) for layer in range(2) for which in (0, 1))
    assert np.array_equal(m.forward(m.FWD_DECODE, [a], [n], [7], logits=True)["logits"], want)
    for kv in (a, f, other):
        kv.close()
    m.close()


def test_a_session_forked_in_other_threads_while_it_goes_on(ctx):  # noqa: F811
    """Calls of a context come from any thread: passes of a session while others fork its beginning, compare and close the forks."""
    import threading
    m = dense(ctx)
    a, toks = started(m, 11, 700), prompt_of(12, 40, 1003)
    want = [m.forward(m.FWD_DECODE, [a], [700 + i], [t], logits=True)["logits"] for i, t in enumerate(toks)]
    bad, over = [], threading.Event()

    def forks(seed):
        rng = np.random.default_rng(seed)
        try:
            while not over.is_set():
                n = int(rng.integers(1, 700))
                f = a.fork(n)
                g = f.fork(n // 2)
                assert a.shared_rows(f) == n // 64 * 64 and g.shared_rows(f) == n // 2 // 64 * 64
                f.close()
                g.close()
        except BaseException as e:      # noqa: BLE001 (told to the thread that asserts)
            bad.append(e)
    ts = [threading.Thread(target=forks, args=(i,)) for i in range(3)]
    for t in ts:
        t.start()
    try:
        for _ in range(3):
            for i, t in enumerate(toks):
                assert np.array_equal(m.forward(m.FWD_DECODE, [a], [700 + i], [t], logits=True)["logits"], want[i])
    finally:
        over.set()
        for t in ts:
            t.join()
    assert not bad
    a.close()
    m.close()


def family_pass(m):
    """A pass over two families, one of them with a short beginning, and sessions by themselves, in an order that mixes them."""
    a, b, c, d, e = started(m, 1, 400), started(m, 2, 1200), started(m, 3, 90), started(m, 4, 1100), started(m, 5, 30)
    fa, fb, fc = [a.fork(400) for _ in range(2)], b.fork(1200), c.fork(90)
    return [e, fa[0], b, c, fa[1], d, fc, a, fb], [30, 400, 1200, 90, 400, 1100, 90, 400, 1200], prompt_of(9, 9, m.vocab)


@pytest.mark.parametrize("qk_norm", [True, False])
def test_a_forks_result_does_not_hang_on_who_shares_the_call(ctx, qk_norm):  # noqa: F811
    """To the bit, as for sessions that share nothing."""
    m = dense(ctx, qk_norm=qk_norm)
    kvs, pos, toks = family_pass(m)

    def run(rows):
        got = m.forward(m.FWD_DECODE, [kvs[i] for i in rows], [pos[i] for i in rows], [toks[i] for i in rows], logits=True, attn_tap=True)
        return {i: (got["logits"][j], got["attn"][:, j]) for j, i in enumerate(rows)}
    alone = {}
    for i in range(9):
        alone.update(run([i]))
    for rows in (list(range(9)), [8, 2, 5], [1, 4, 7], [7, 1], [6, 0, 3, 8, 1]):
        for i, (logits, attn) in run(rows).items():
            assert np.array_equal(logits, alone[i][0]) and np.array_equal(attn, alone[i][1]), (rows, i)
    for kv in kvs:
        kv.close()
    m.close()


def test_together_when_asked(ctx):  # noqa: F811
    """Attention to rounding; asked no longer, the bits are those of before."""
    m = dense(ctx)
    kvs, pos, toks = family_pass(m)

    def run():
        return m.forward(m.FWD_DECODE, kvs, pos, toks, hidden=True, logits=True, argmax=True, attn_tap=True)
    apart = run()
    m.set_together()
    got = run()
    m.set_together(False)
    again = run()
    assert np.array_equal(apart["logits"], again["logits"]) and np.array_equal(apart["attn"], again["attn"])
    # (the first layer's attention has the same queries and keys: F32 sums in two orders, each near 64 bits to 5e-6 of its norm)
    for i in range(9):
        x, y = got["attn"][0, i], apart["attn"][0, i]
        assert np.linalg.norm(x - y) <= 1e-5 * np.linalg.norm(y), i
        assert got["argmax"][i] == np.argmax(got["logits"][i])
    alone = {0, 3, 5, 6}                                 # those that hold nothing long together go the way they went
    assert all(np.array_equal(got["logits"][i], apart["logits"][i]) == (i in alone) for i in range(9))
    for kv in kvs:
        kv.close()
    m.close()


def test_a_beam_step_attends_together(ctx):  # noqa: F811
    """Without being asked: its choice is that from the logits of a pass that was asked to."""
    from _plain_beams import choose, choose_error
    m = dense(ctx)
    a = started(m, 21, 700)
    kvs, pos, toks = [a] + [a.fork(700) for _ in range(3)], [700] * 4, prompt_of(22, 4, m.vocab)
    scores = np.array([[-1.0, -1.5, -1.25, -2.0]], np.float32)
    got = m.beam_step(kvs, pos, toks, scores, 8)
    m.set_together()
    rows = m.forward(m.FWD_DECODE, kvs, pos, toks, logits=True)["logits"]
    want = choose(rows[None], scores, 8)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    assert (np.abs(got[0] - want[0]) <= choose_error(want[0], m.vocab)).all()
    for kv in kvs:
        kv.close()
    m.close()
