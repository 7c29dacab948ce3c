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
