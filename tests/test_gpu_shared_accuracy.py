"""GPU: what the two F16 parts of queries and weights are for: shared attention as near to 64 bits as F32 arithmetic."""
import numpy as np
import pytest

import _gen
from _cuda_util import port
from _plain_beams import attend
from test_gpu_shared_attention import HD, Family, call, ctx  # noqa: F401 (ctx: a fixture)

pytestmark = pytest.mark.gpu

# Of rows as Family makes them, q and k of unit scale.  A score: two F16 parts leave 2^-22 of the row's largest query element (about 3.5),
# evenly spread, 2^-23 / sqrt(3) * 3.5 as a root mean square, and 128 of them times unit keys times 128^-0.5 add up to the same: 2.4e-7.
# Its 16 steps in the tensor core cut off 2^-23 of a partial sum (of size 1 or 2) each: 16 * 2^-24 * 1.5 = 1.4e-6 on the average.  A weight:
# ex2.approx 2^-22, its parts 2^-22.  Errors of the weights e_i, independent of one another, leave sqrt(sum (w_i e_i v_i)^2), the same share of
# sqrt(sum (w_i v_i)^2), which is the result's size: 2e-6, the F32 sums 2^-24 each besides.  One F16 part alone is off by 2^-12 / sqrt(3) = 1.4e-4.
NORM = 5e-6


def near(got, want, what):
    err, size = np.linalg.norm((got - want).ravel()), np.linalg.norm(want.ravel())
    assert err <= NORM * size, (what, err / size)


def check_norms(got, families, q):
    i = 0
    for f in families:
        for k, v in zip(f.k, f.v):
            near(got[i], attend(q[i], k, v), i)
            i += 1


@pytest.mark.parametrize("prompt, own, hq, hkv", [
    (64, [5, 70], 4, 2), (130, [1, 40], 16, 8),                                     # 16 columns, whole lists
    (2011, [90] * 4, 32, 8), (3000, [200, 5], 8, 1), (20000, [30, 3], 16, 8),       # ... in shares
    (100, [30] * 6, 32, 8), (3000, [64, 1, 300, 7] * 2, 32, 8),                     # 32
    (100, [20] * 16, 32, 8), (2500, [50, 400] * 8, 32, 8), (5000, [9] * 3, 96, 2),  # 64, the last one in two lists
    (0, [700, 1300], 8, 8)])
def test_every_width(ctx, prompt, own, hq, hkv):  # noqa: F811
    f = Family(ctx, 2000 + prompt + hq, prompt, own, hkv)
    q = _gen.normal(2001 + prompt, (len(own), hq, HD))
    check_norms(call(ctx, [f], q, hq), [f], q)
    f.close()


def test_widths_beside_one_another(ctx):  # noqa: F811
    fs = [Family(ctx, 2100, 1500, [60] * 2, 8), Family(ctx, 2140, 1500, [33] * 5, 8), Family(ctx, 2180, 200, [10] * 9, 8)]
    q = _gen.normal(2099, (16, 40, HD))
    check_norms(call(ctx, fs, q, 40), fs, q)
    for f in fs:
        f.close()


@pytest.mark.parametrize("own, hq", [([30] * 2, 32), ([75, 3, 130, 64, 1, 20], 32), ([40] * 14, 32)])
@pytest.mark.parametrize("rope", [True, False])
def test_steps(ctx, own, hq, rope):  # noqa: F811
    import torch
    hkv, n = 8, len(own)
    f = Family(ctx, 2200 + n, 900, own, hkv, max_ctx=1100)
    q, k, v = _gen.normal(2300, (n, hq, HD)), _gen.normal(2301, (n, hkv, HD)), _gen.normal(2302, (n, hkv, HD))
    dq, dk, dv = (torch.from_numpy(x).cuda() for x in (q, k, v))
    out = torch.full_like(dq, float("nan"))
    torch.cuda.synchronize()
    ctx.decode_step_shared(f.kvs, 0, f.lens, [(n, f.rows)], dq, dk, dv, out, hq, theta=5e5, rope=rope)
    ctx.sync()
    got, P = out.cpu().numpy(), port()
    for i in range(n):
        qr, kr = q[i:i + 1], k[i:i + 1]
        if rope:
            _, qr = P.rope(qr, f.lens[i], 5e5, 0)
            _, kr = P.rope(kr, f.lens[i], 5e5, 0)
        near(got[i], attend(qr[0], np.concatenate([f.k[i], P.f32_to_f16(kr)]), np.concatenate([f.v[i], P.f32_to_f16(v[i:i + 1])])), i)
    f.close()


@pytest.mark.parametrize("below", [17.3, 22.4, 25.6, 28.0])
@pytest.mark.parametrize("sessions, hq, hkv, prompt", [(2, 8, 8, 6000), (4, 32, 8, 20000), (6, 32, 8, 6000), (16, 32, 8, 30000), (2, 4, 1, 900)])
def test_one_large_score_before_a_long_flat_tail(ctx, below, sessions, hq, hkv, prompt):  # noqa: F811
    """The tail's weights, 2^-below of the largest, are all alike and their values have one sign: what is lost of them adds up."""
    own = 40
    k = np.zeros((prompt + own, hkv, HD), np.float32)
    v = np.ones_like(k)
    k[0] = 1.0
    v[0] = 0.0                                                       # (what the result holds is the tail's)
    P = port()
    k, v = P.f32_to_f16(k), P.f32_to_f16(v)
    kv = ctx.kv_create(1, hkv, HD, prompt + own)
    kv.write_rows(0, 0, 0, k)
    kv.write_rows(0, 1, 0, v)
    shared = prompt // 64 * 64
    forks = [kv.fork(prompt + own) for _ in range(sessions - 1)]
    # all elements alike, so that a score is 128 equal products
    element = np.float32(below * np.log(2.0) / (HD * HD ** -0.5))
    q = np.full((sessions, hq, HD), element, np.float32)
    out = np.empty_like(q)
    ctx.attn_decode_shared([kv] + forks, 0, [prompt + own] * sessions, [(sessions, shared)], q, out, hq)
    n = prompt + own - 1
    want = attend(q[0], k, v)
    # A weight: 2^-32 of the largest is lost at most where F16 ends, 2^-22 of itself else; its exponent, near -28, is off by 2^-19 by the
    # rounding of its argument and 28 * 2^-21 by the query's; F32 sums of the tail, all of one sign: 16 cut off by 2^-23 a tile, 300 by 2^-24.
    bound = n * 2.0 ** -32 + want.max() * (2.0 ** -22 + 0.7 * (2.0 ** -19 + 28 * 2.0 ** -21) + 16 * 2.0 ** -23 + 300 * 2.0 ** -24)
    err = np.abs(out - want).max()
    assert err <= bound, (err, bound, want.max())
    for x in [kv] + forks:
        x.close()
