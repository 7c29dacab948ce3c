"""GPU: a decode step right behind launches that fill the pages it reads: copies of a reordering and of forks, rows written from device memory."""
import numpy as np
import pytest

import _gen
from _cuda_util import port
from _plain_beams import attend, attend_error
from test_gpu_shared_attention import HD, Family, ctx, f16  # noqa: F401 (ctx: a fixture)

pytestmark = pytest.mark.gpu


def check_step(out, q, k, v, keys, values):
    """One step's rows, q not rotated, against 64 bits; keys, values: [session][rows]."""
    P = port()
    for s in range(len(q)):
        a, b = np.concatenate([keys[s], P.f32_to_f16(k[s:s + 1])]), np.concatenate([values[s], P.f32_to_f16(v[s:s + 1])])
        assert np.abs(out[s] - attend(q[s], a, b)).max() <= attend_error(q[s], a, b), s


def rows_of(seed, n, hq, hkv):
    import torch
    x = _gen.normal(seed, (n, hq, HD)), _gen.normal(seed + 1, (n, hkv, HD)), _gen.normal(seed + 2, (n, hkv, HD))
    return x, [torch.from_numpy(y).cuda() for y in x]


@pytest.mark.parametrize("prompt, own", [(130, 900), (0, 2000), (640, 1300)])
def test_reorder_then_step(ctx, prompt, own):  # noqa: F811
    import torch
    hq, hkv = 32, 8
    f = Family(ctx, 40 + prompt, prompt, [own + 7 * i for i in range(4)], hkv, max_ctx=prompt + own + 60)
    at = list(f.lens)
    plans = [[2, 2, 2, 2], [1, 0, 1, 0], [3, 3, 0, 0], [0, 1, 1, 3]]
    inputs = [rows_of(500 + 10 * i, 4, hq, hkv) for i in range(len(plans))]
    outs = torch.full((len(plans), 4, hq, HD), float("nan"), device="cuda")
    torch.cuda.synchronize()
    keys, values, want = f.k, f.v, []
    P = port()
    for i, parents in enumerate(plans):
        (q, k, v), (dq, dk, dv) = inputs[i]
        ctx.kv_reorder(f.kvs, parents, at)
        at = [at[p] for p in parents]
        ctx.decode_step(f.kvs, 0, at, dq, dk, dv, outs[i], hq, rope=False)
        keys, values = [keys[p] for p in parents], [values[p] for p in parents]
        want.append((q, k, v, keys, values))
        at = [n + 1 for n in at]
        keys = [np.concatenate([x, P.f32_to_f16(k[s:s + 1])]) for s, x in enumerate(keys)]
        values = [np.concatenate([x, P.f32_to_f16(v[s:s + 1])]) for s, x in enumerate(values)]
    ctx.sync()
    for i, w in enumerate(want):
        check_step(outs[i].cpu().numpy(), *w)
    f.close()


def test_fork_then_step(ctx):  # noqa: F811
    import torch
    hq, hkv = 32, 8
    f = Family(ctx, 70, 1000, [1023, 0], hkv, max_ctx=2200)
    (q, k, v), (dq, dk, dv) = rows_of(600, 2, hq, hkv)
    out = torch.full((2, hq, HD), float("nan"), device="cuda")
    torch.cuda.synchronize()
    g = f.kvs[0].fork(2023)
    ctx.decode_step([f.kvs[0], g], 0, [2023, 2023], dq, dk, dv, out, hq, rope=False)
    ctx.sync()
    check_step(out.cpu().numpy(), q, k, v, [f.k[0]] * 2, [f.v[0]] * 2)
    g.close()
    f.close()


def test_rows_from_device_memory_then_step(ctx):  # noqa: F811
    import torch
    hq, hkv, n = 32, 8, 3000
    kvs = [ctx.kv_create(1, hkv, HD, n + 1) for _ in range(4)]
    (q, k, v), (dq, dk, dv) = rows_of(700, 4, hq, hkv)
    keys, values = [f16(710 + i, (n, hkv, HD)) for i in range(4)], [f16(720 + i, (n, hkv, HD)) for i in range(4)]
    rows = [[torch.from_numpy(x.view(np.int16)).cuda() for x in y] for y in (keys, values)]
    out = torch.full((4, hq, HD), float("nan"), device="cuda")
    torch.cuda.synchronize()
    for i, kv in enumerate(kvs):
        kv.write_rows(0, 0, 0, rows[0][i])
        kv.write_rows(0, 1, 0, rows[1][i])
    ctx.decode_step(kvs, 0, [n] * 4, dq, dk, dv, out, hq, rope=False)
    ctx.sync()
    check_step(out.cpu().numpy(), q, k, v, keys, values)
    for kv in kvs:
        kv.close()
