"""Plain 64-bit forms of beam search's operators, and how far F32 kernels may be from them."""
import numpy as np

NONE = 0xFFFFFFFF


def choose(logits, scores, n_out):
    """The n_out best of every group by score + log softmax: (scores, beams, tokens)."""
    groups, beams, vocab = logits.shape
    out = np.full((groups, n_out), -np.inf), np.full((groups, n_out), NONE, np.uint32), np.full((groups, n_out), NONE, np.uint32)
    for g in range(groups):
        found = []
        for b in range(beams):
            row, s = logits[g, b].astype(np.float64), float(scores[g, b])
            if not np.isfinite(s) or np.isnan(row).any() or np.isposinf(row).any() or np.isneginf(row).all():
                continue
            top = row.max()
            total = s + (row - (top + np.log(np.exp(row - top).sum())))
            # (a row's candidates are in the order of its logits)
            order = np.lexsort((np.arange(vocab), -row))[:n_out]
            found += [(-total[v], b, v) for v in order if row[v] > -np.inf]
        for i, (t, b, v) in enumerate(sorted(found)[:n_out]):
            out[0][g, i], out[1][g, i], out[2][g, i] = -t, b, v
    return out


def choose_error(want, vocab, parts=1):
    """Largest error of an F32 total: its rounding (half a step, 2^-24 of it), and the F32 sum of exponentials.  Of that sum every term
    is within 2^-22 (ex2.approx) + 0.54 * 2^-24 (its argument d log2 e, rounded twice: |d| e^d <= 0.37), a lane adds up to 16 terms a batch
    of 4096 logits one after the other, and 8 joins (5 across lanes, 3 in depth across warps at least; 7 in order) each multiply by an
    ex2 and add."""
    terms = 16 * -(-vocab // 4096)
    rel = 2.0 ** -22 + 2.0 ** -24 + terms * 2.0 ** -24 + (5 + 7) * (2.0 ** -22 + 2 * 2.0 ** -24)
    finite = np.where(np.isfinite(want), np.abs(want), 0)
    return finite * 2.0 ** -24 + 2 * rel


def attend(q, k, v, scale=None):
    """One query row [heads][dim] over keys and values [rows][kv heads][dim] (F16 bits or floats), in 64 bits."""
    q = q.astype(np.float64)
    k, v = (x.view(np.float16).astype(np.float64) if x.dtype == np.uint16 else x.astype(np.float64) for x in (k, v))
    heads, dim = q.shape
    per = heads // k.shape[1]
    scale = scale or dim ** -0.5
    s = np.einsum("hd,rhd->hr", q, np.repeat(k, per, axis=1)) * scale
    m = s.max(axis=1, keepdims=True)
    with np.errstate(invalid="ignore"):
        p = np.exp(s - np.where(np.isneginf(m), 0, m))
    total = p.sum(axis=1, keepdims=True)
    out = np.einsum("hr,rhd->hd", p, np.repeat(v, per, axis=1))
    return np.where(total == 0, 0, out / np.where(total == 0, 1, total))


def attend_error(q, k, v, scale=None):
    """Largest error of an element of attend()'s row by the shared kernel.

    A score: the query's two F16 parts leave 2^-22 of its row's largest value per element; 16 products of 16 terms are added in an F32
    accumulator that rounds towards zero (a step, 2^-23 of the sum of magnitudes at most, each).  A weight 2^x: x rounded
    (2^-24 |x|, and |x| 2^x <= 0.54 against the largest), ex2.approx 2^-22, its two F16 parts 2^-22.  Output: 16 such additions a
    tile, an F32 addition a tile and a chunk (2^-24 each; fewer than 300 together here), a quotient.  Weights go into numerator and
    sum alike."""
    dim = q.shape[-1]
    scale = scale or dim ** -0.5
    k, v = (np.abs(x.view(np.float16).astype(np.float64)) for x in (k, v))
    aq = np.abs(q).astype(np.float64)
    per = q.shape[0] // k.shape[1]
    kk = np.repeat(k, per, axis=1)
    split = 2.0 ** -22 * np.einsum("h,rhd->hr", aq.max(axis=1), kk).max() * scale
    sums = 16 * 2.0 ** -23 * np.einsum("hd,rhd->hr", aq, kk).max() * scale
    weight = split + sums + 2.0 ** -24 + 2 * 2.0 ** -22
    return (2 * weight + 16 * 2.0 ** -23 + 300 * 2.0 ** -24 + 2.0 ** -23) * v.max()
