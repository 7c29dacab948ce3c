"""GPU: what shared attention loses of small weights."""
import numpy as np
import pytest

from _cuda_util import port
from _plain_beams import attend
from test_gpu_shared_attention import HD, ctx  # noqa: F401 (ctx: a fixture)

pytestmark = pytest.mark.gpu


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
