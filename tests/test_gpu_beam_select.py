"""GPU: wr_cuda_beam_select against a 64-bit restatement."""
import numpy as np
import pytest

from _plain_beams import NONE, choose, choose_error

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import wayruntime_b200 as wr
    c = wr.Context(0)
    yield c
    c.close()


def run(ctx, logits, scores, n_out, device=True, offset=0):
    import torch
    groups = logits.shape[0]
    if not device:
        out = np.full((groups, n_out), np.nan, np.float32), np.zeros((groups, n_out), np.uint32), np.zeros((groups, n_out), np.uint32)
        ctx.beam_select(np.ascontiguousarray(logits), np.ascontiguousarray(scores), *out)
        return out
    room = torch.empty(logits.size + offset, dtype=torch.float32, device="cuda")
    lg = room[offset:].view(logits.shape)
    lg.copy_(torch.from_numpy(logits))
    out = (torch.full((groups, n_out), float("nan"), device="cuda"), torch.zeros((groups, n_out), dtype=torch.int32, device="cuda"),
           torch.zeros((groups, n_out), dtype=torch.int32, device="cuda"))
    sc = torch.from_numpy(scores).cuda()
    torch.cuda.synchronize()
    ctx.beam_select(lg, sc, *out)
    ctx.sync()
    s, b, t = (x.cpu().numpy() for x in out)
    return s, b.view(np.uint32), t.view(np.uint32)


def check(got, logits, scores, n_out):
    want = choose(logits, scores, n_out)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    there = want[1] != NONE
    assert np.array_equal(np.isneginf(got[0]), ~there)
    assert (np.abs(got[0][there] - want[0][there]) <= choose_error(want[0], logits.shape[2])[there]).all()


def rows(seed, groups, beams, vocab, spread=2.5):
    rng = np.random.default_rng(seed)
    return ((rng.standard_normal((groups, beams, vocab)) * spread).astype(np.float32),
            (-20 - np.abs(rng.standard_normal((groups, beams)))).astype(np.float32))


@pytest.mark.parametrize("groups, beams, vocab, n_out", [
    (1, 1, 1, 1), (1, 1, 1, 32), (1, 2, 3, 4), (2, 3, 31, 7), (1, 1, 4093, 2), (1, 1, 4096, 8), (3, 2, 4097, 4), (2, 5, 8191, 10),
    (1, 4, 32003, 8), (1, 16, 12289, 32), (4, 4, 50257, 8), (1, 1, 151936, 16), (1, 3, 151936, 17), (40, 8, 1000, 16),
    (130, 16, 515, 32), (1, 16, 65536, 32)])
def test_choice(ctx, groups, beams, vocab, n_out):
    logits, scores = rows(groups * 1000 + vocab, groups, beams, vocab)
    check(run(ctx, logits, scores, n_out), logits, scores, n_out)


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_rows_at_any_alignment(ctx, offset):
    logits, scores = rows(offset, 2, 3, 10001)
    check(run(ctx, logits, scores, 6, offset=offset), logits, scores, 6)


def test_host_buffers(ctx):
    logits, scores = rows(5, 2, 4, 9999)
    check(run(ctx, logits, scores, 8, device=False), logits, scores, 8)


@pytest.mark.parametrize("vocab, n_out", [(5, 8), (6000, 8), (6000, 32), (40000, 3)])
def test_ties_go_to_the_lower_beam_then_the_lower_token(ctx, vocab, n_out):
    logits = np.zeros((2, 3, vocab), np.float32)                   # every candidate of a group is equal
    scores = np.full((2, 3), -1.0, np.float32)
    check(run(ctx, logits, scores, n_out), logits, scores, n_out)
    rng = np.random.default_rng(vocab)                              # few different values, both zeros among them
    logits = rng.choice(np.array([-1.0, -0.0, 0.0, 0.5], np.float32), (2, 3, vocab))
    check(run(ctx, logits, scores, n_out), logits, scores, n_out)


def test_rows_in_ascending_and_descending_order(ctx):
    logits = np.stack([np.linspace(-9, 9, 20000), np.linspace(9, -9, 20000)]).astype(np.float32)[None]
    scores = np.array([[-3.0, -3.0]], np.float32)
    got = run(ctx, logits, scores, 16)
    want = choose(logits, scores, 16)
    assert np.array_equal(got[2], want[2]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("n_out", [4, 20, 32])
def test_the_best_lie_together(ctx, n_out):
    logits, scores = rows(77, 1, 2, 30000)
    logits[0, 1, 12000:12700] += 30                                 # (700 large ones, all in one part of the row)
    check(run(ctx, logits, scores, n_out), logits, scores, n_out)


def test_what_is_masked_ended_or_not_a_number_has_no_continuation(ctx):
    logits, scores = rows(9, 6, 3, 5000)
    logits[0, :, 7:] = -np.inf                                      # seven tokens a beam
    logits[1] = -np.inf                                             # a row that a mask leaves nothing of
    scores[2, 1] = -np.inf                                          # an ended beam
    scores[3] = np.nan
    logits[4, 0, 4999] = np.nan
    logits[4, 1, 0] = np.inf
    scores[5, 0] = np.inf
    logits[2, 0, ::2] = np.finfo(np.float32).min                    # a mask of the type's lowest value
    got = run(ctx, logits, scores, 24)
    check(got, logits, scores, 24)
    assert (got[1][1] == NONE).all() and (got[1][3] == NONE).all() and (got[1][2] != 1).all()
    assert (got[1][0] != NONE).sum() == 21 and set(got[1][4]) == {2}


@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("vocab", [9, 300, 5000, 40000])
@pytest.mark.parametrize("n_out", [1, 8, 32])
def test_rows_without_a_finite_sum_beside_others(ctx, bad, vocab, n_out):
    """One logit of some beams is not finite: their others are no continuations, and take no place from the other beams'."""
    for beams, spoilt in ((2, [0]), (8, [1, 2, 5]), (16, list(range(0, 16, 2))), (16, list(range(1, 16)))):
        logits, scores = rows(60 + beams + vocab, 3, beams, vocab)
        for b in spoilt:
            logits[:, b, (7 * b) % vocab] = bad
        check(run(ctx, logits, scores, n_out), logits, scores, n_out)


def test_an_ended_beams_row_is_not_read(ctx):
    """Its address may be anything the buffer covers; here NaN, which would take every candidate out if it were read."""
    logits, scores = rows(10, 1, 2, 3000)
    logits[0, 0] = np.nan
    scores[0, 0] = -np.inf
    check(run(ctx, logits, scores, 4), logits, scores, 4)


def test_same_bits_every_time(ctx):
    logits, scores = rows(11, 3, 5, 40000)
    first = run(ctx, logits, scores, 10)
    for _ in range(20):
        assert all(np.array_equal(a, b) for a, b in zip(first, run(ctx, logits, scores, 10)))


def test_captured_in_a_graph(ctx):
    import torch
    logits, scores = rows(12, 1, 4, 20011)
    lg, sc = torch.from_numpy(logits).cuda(), torch.from_numpy(scores).cuda()
    out = (torch.zeros((1, 8), device="cuda"), torch.zeros((1, 8), dtype=torch.int32, device="cuda"),
           torch.zeros((1, 8), dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    ctx.beam_select(lg, sc, *out)
    ctx.sync()
    stream, graph = torch.cuda.ExternalStream(ctx.stream), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ctx.beam_select(lg, sc, *out)
    big, small = rows(13, 16, 16, 60000)                            # the scratch grows between capture and launch
    run(ctx, big, small, 32)
    other, _ = rows(14, 1, 4, 20011)
    lg.copy_(torch.from_numpy(other))
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph.replay()
    ctx.sync()
    check((out[0].cpu().numpy(), out[1].cpu().numpy().view(np.uint32), out[2].cpu().numpy().view(np.uint32)), other, scores, 8)


@pytest.mark.parametrize("vocab", [1000, 5000, 16000, 32003])
@pytest.mark.parametrize("apart", [0.0, 3.0, 200.0])
def test_the_widest_choice_of_beams_far_apart(ctx, vocab, apart):
    """16 beams, 32 out: the weakest beam's best is far below what is chosen, and the last part of a row has a few logits only."""
    logits, scores = rows(70, 2, 16, vocab)
    scores -= apart * np.arange(16, dtype=np.float32)
    check(run(ctx, logits, scores, 32), logits, scores, 32)


def test_scores_in_place(ctx):
    import torch
    logits, scores = rows(40, 6, 4, 9000)
    d, s = torch.from_numpy(logits).cuda(), torch.from_numpy(scores).cuda()
    b, t = (torch.empty((6, 4), dtype=torch.int32, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    ctx.beam_select(d, s, s, b, t)
    ctx.sync()
    check((s.cpu().numpy(), b.cpu().numpy().astype(np.uint32), t.cpu().numpy().astype(np.uint32)), logits, scores, 4)


def test_many_rows_and_the_widest_choice(ctx):
    """As many groups as there may be, and 16 beams with 32 places each."""
    import torch
    n = 65535
    for groups, beams, vocab, n_out in ((n, 1, 9, 3), (n // 16, 16, 7, 32)):
        logits, scores = rows(41 + beams, groups, beams, vocab)
        d, s = torch.from_numpy(logits).cuda(), torch.from_numpy(scores).cuda()
        o = torch.empty((groups, n_out), device="cuda"), *(torch.empty((groups, n_out), dtype=torch.int32, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        ctx.beam_select(d, s, *o)
        ctx.sync()
        got = [x.cpu().numpy() for x in o]
        some = [0, 1, 777, groups - 2, groups - 1]
        check((got[0][some], got[1][some].astype(np.uint32), got[2][some].astype(np.uint32)), logits[some], scores[some], n_out)


def test_two_contexts_in_two_threads():
    """Each context has its own stream and scratch; its calls may come from any thread."""
    import threading
    import torch
    import wayruntime_b200 as wr
    cs = [wr.Context(0) for _ in range(2)]
    data = [rows(50 + i, 3, 4, 20000 + i) for i in range(2)]
    bad = []

    def work(i, c):
        try:
            for _ in range(20):
                check(run(c, *data[i], 8), *data[i], 8)
        except BaseException as e:      # noqa: BLE001 (told to the thread that asserts)
            bad.append(e)
    ts = [threading.Thread(target=work, args=(i % 2, cs[i // 2])) for i in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    torch.cuda.synchronize()
    assert not bad
    for c in cs:
        c.close()


def test_refusals(ctx):
    import torch
    import wayruntime_b200 as wr
    both = torch.zeros((2, 2, 10), device="cuda")
    s, b, t = torch.zeros((2, 2), device="cuda"), *(torch.zeros((2, 3), dtype=torch.int32, device="cuda") for _ in range(2))
    o = torch.zeros((2, 3), device="cuda")
    flat = both.view(-1)
    for bad in ((flat[:6].view(2, 3), b, t), (o, flat[34:].view(torch.int32).view(2, 3), t), (o, b, flat[10:16].view(torch.int32).view(2, 3))):
        with pytest.raises(wr.WrCudaError) as e:                     # a result in what is read
            ctx.beam_select(both, s, *bad)
        assert e.value.status == -4
    wide = torch.zeros(8, device="cuda")
    with pytest.raises(wr.WrCudaError) as e:                         # places of other groups' scores
        ctx.beam_select(both, wide[:4].view(2, 2), wide[:6].view(2, 3), b, t)
    assert e.value.status == -4
    logits, scores = rows(1, 1, 2, 10)
    out = lambda n: (np.zeros((1, n), np.float32), np.zeros((1, n), np.uint32), np.zeros((1, n), np.uint32))  # noqa: E731
    for bad_logits, bad_scores, n, status in ((logits, scores, 33, -8), (np.zeros((1, 17, 10), np.float32), np.zeros((1, 17), np.float32), 4, -8),
                                              (np.zeros((1, 2, 0), np.float32), scores, 4, -4)):
        with pytest.raises(wr.WrCudaError) as e:
            ctx.beam_select(bad_logits, bad_scores, *out(n))
        assert e.value.status == status
    with pytest.raises(ValueError):
        ctx.beam_select(logits, scores[:, :1], *out(4))
    with pytest.raises(ValueError):
        ctx.beam_select(logits.astype(np.float64), scores, *out(4))
    lib = ctx._lib
    p = logits.ctypes.data
    assert lib.wr_cuda_beam_select(ctx._h, 70000, 1, 1, p, p, 1, p, p, p, 0) == -8
    assert lib.wr_cuda_beam_select(ctx._h, 1, 1, 1, None, p, 1, p, p, p, 0) == -4
    assert lib.wr_cuda_beam_select(ctx._h, 1, 1, 1, p, p, 1, p, p, p, 2) == -4
