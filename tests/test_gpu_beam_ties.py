"""GPU: beams whose totals are equal, or nearer than an F32 rounding: their order, wherever their rows lie."""
import numpy as np
import pytest

from _plain_beams import choose
from test_gpu_beam_select import ctx, rows, run  # noqa: F401 (ctx: a fixture)

pytestmark = pytest.mark.gpu


def alike(seed, groups, beams, vocab):
    """The same row of logits in all beams of a group."""
    logits, _ = rows(seed, groups, 1, vocab)
    return np.repeat(logits, beams, axis=1)


@pytest.mark.parametrize("vocab", [1001, 4099, 32000, 32001, 32002, 32003, 151937])
@pytest.mark.parametrize("offset", [0, 1])
def test_equal_beams_go_to_the_lower_one(ctx, vocab, offset):  # noqa: F811
    """Rows of an odd vocabulary begin at every place within 16 bytes; their sums are the same to the bit."""
    logits, n_out = alike(vocab, 6, 4, vocab), 16
    scores = np.repeat(-20 - np.arange(6, dtype=np.float32)[:, None] / 7, 4, axis=1)
    score, beam, token = run(ctx, logits, scores, n_out, offset=offset)
    for g in range(6):
        best = np.lexsort((np.arange(vocab), -logits[g, 0]))[:n_out // 4]
        assert np.array_equal(beam[g], np.tile(np.arange(4), n_out // 4))
        assert np.array_equal(token[g], np.repeat(best, 4))
        assert all(len(set(score[g, i:i + 4])) == 1 for i in range(0, n_out, 4))


@pytest.mark.parametrize("vocab", [1001, 32000, 32003])
def test_totals_nearer_than_an_f32_rounding(ctx, vocab):  # noqa: F811
    """Scores of about -0.001 that differ by a step of theirs, 2^-33: totals of -4 and less are the same in F32, not in 64 bits."""
    logits = alike(vocab + 1, 5, 4, vocab)
    steps = np.array([2, 0, 3, 1])                                   # (how far each is above the lowest)
    scores = np.repeat((np.float32(-0.0015) + np.float32(2.0 ** -33) * steps.astype(np.float32))[None], 5, axis=0).astype(np.float32)
    assert all(len(set(row)) == 4 for row in scores)
    score, beam, token = run(ctx, logits, scores, 8)
    want = choose(logits, scores, 8)
    assert np.array_equal(beam, want[1]) and np.array_equal(token, want[2])
    assert np.array_equal(beam, np.tile(np.argsort(-steps), (5, 2)))
    assert all(len(set(score[g, :4])) == 1 for g in range(5))


@pytest.mark.parametrize("vocab", [1000, 4097, 32003, 151936])
@pytest.mark.parametrize("spread", [1.0, 2.5, 6.0])
def test_a_rows_sum(ctx, vocab, spread):  # noqa: F811
    """Totals near zero, so that what is left of them is the error of the row's sum; rows one by one, and many of them in long parts."""
    x, _ = rows(vocab, 1, 4, vocab, spread)
    wide = x[0].astype(np.float64)
    top = wide.max(-1)
    lse = top + np.log(np.exp(wide - top[:, None]).sum(-1))
    scores = (lse - top).astype(np.float32)
    want = scores + (top - lse)
    for repeat, batches in ((1, 1), (160, -(-vocab // 4096))):       # (640 rows: a part is a whole row)
        got = run(ctx, np.tile(x[0], (repeat, 1))[:, None], np.tile(scores, repeat)[:, None], 1)[0].reshape(repeat, 4)
        # A term: ex2.approx 2^-22, its argument rounded twice (|d| e^d <= 0.37, in powers of two 0.54 * 2^-24 each).  Sums: a lane's two
        # accumulators, 8 terms a batch each and one rescaling; then the two, 5 steps across lanes, 8 warps, each of the two maxima's factors 2^-22 and
        # two roundings, the part's sum rounded.  (Parts and the total are added up in 64 bits; the result's own rounding is relative to nearly zero.)
        rel = 2.0 ** -22 + 2 * 0.54 * 2.0 ** -24 + batches * (8 * 2.0 ** -24 + 2.0 ** -22) + (1 + 5 + 8) * 2.0 ** -24 + 3 * (2.0 ** -22 + 2.0 ** -23)
        assert np.abs(got - want).max() <= rel
        assert (got == got[0]).all()
