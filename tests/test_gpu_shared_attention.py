"""GPU: wr_cuda_attn_decode_shared and wr_cuda_decode_step_shared against a 64-bit restatement."""
import numpy as np
import pytest

import _gen
from _cuda_util import port
from _plain_beams import attend, attend_error

pytestmark = pytest.mark.gpu
HD = 128


@pytest.fixture(scope="module")
def ctx():
    import wayruntime_b200 as wr
    c = wr.Context(0, attn_max_seq=65536)
    yield c
    c.close()


def f16(seed, shape, std=1.0):
    return port().f32_to_f16(_gen.normal(seed, shape, std))


class Family:
    """Sessions behind one prompt: one has taken it, the others are its forks; every one has rows of its own."""

    def __init__(self, ctx, seed, prompt, own, hkv, max_ctx=None, layers=1, std=1.0):
        cap = max_ctx or prompt + max(own) + 1
        self.prompt, self.own = prompt, own
        self.k, self.v = [], []
        pk, pv = f16(seed, (prompt, hkv, HD), std), f16(seed + 1, (prompt, hkv, HD))
        first = ctx.kv_create(layers, hkv, HD, cap)
        if prompt:
            first.write_rows(0, 0, 0, pk)
            first.write_rows(0, 1, 0, pv)
        self.kvs = [first] + [first.fork(prompt) for _ in own[1:]]
        for i, (kv, n) in enumerate(zip(self.kvs, own)):
            k, v = f16(seed + 10 + 2 * i, (n, hkv, HD), std), f16(seed + 11 + 2 * i, (n, hkv, HD))
            if n:
                kv.write_rows(0, 0, prompt, k)
                kv.write_rows(0, 1, prompt, v)
            self.k.append(np.concatenate([pk, k]))
            self.v.append(np.concatenate([pv, v]))
        self.lens = [prompt + n for n in own]
        self.rows = prompt // 64 * 64

    def close(self):
        for kv in self.kvs:
            kv.close()


def call(ctx, families, q, hq, device=True, scale=0.0, rows=None):
    import torch
    kvs = [kv for f in families for kv in f.kvs]
    lens = [n for f in families for n in f.lens]
    groups = [(len(f.kvs), f.rows if rows is None else rows) for f in families]
    if not device:
        out = np.full(q.shape, np.nan, np.float32)
        ctx.attn_decode_shared(kvs, 0, lens, groups, q, out, hq, scale=scale)
        return out
    dq, out = torch.from_numpy(q).cuda(), torch.full(q.shape, float("nan"), device="cuda")
    torch.cuda.synchronize()
    ctx.attn_decode_shared(kvs, 0, lens, groups, dq, out, hq, scale=scale)
    ctx.sync()
    assert np.array_equal(dq.cpu().numpy(), q, equal_nan=True)
    return out.cpu().numpy()


def check(got, families, q, scale=None):
    i = 0
    for f in families:
        for k, v in zip(f.k, f.v):
            want = attend(q[i], k, v, scale)
            err = np.abs(got[i] - want).max()
            assert err <= attend_error(q[i], k, v, scale), (i, err)
            i += 1


@pytest.mark.parametrize("prompt, own, hq, hkv", [
    (64, [0], 1, 1), (64, [1, 0], 2, 1), (0, [1], 8, 8), (1, [0, 5, 1], 4, 2), (63, [1, 2], 16, 8), (65, [0, 63], 16, 8),
    (128, [64, 1, 200], 32, 8), (127, [1, 1, 1, 1], 40, 8), (192, [130, 0, 0, 7], 16, 4), (1000, [33] * 4, 32, 8),
    (2011, [90] * 4, 32, 8), (640, list(range(16)), 32, 8), (500, [75] * 8, 16, 1), (1500, [700, 3] * 8, 64, 8),
    (3001, [10] * 16, 64, 8), (777, [100] * 3, 96, 2), (64, [2000, 1], 8, 8), (8000, [5, 300], 10, 2)])
def test_one_family(ctx, prompt, own, hq, hkv):
    f = Family(ctx, 100 * prompt + hq, prompt, own, hkv)
    q = _gen.normal(prompt + 7, (len(own), hq, HD))
    check(call(ctx, [f], q, hq), [f], q)
    f.close()


def test_several_families_and_sessions_alone(ctx):
    fs = [Family(ctx, 1, 700, [20, 90, 1], 8), Family(ctx, 50, 1300, [64] * 5, 8), Family(ctx, 90, 100, [900], 8), Family(ctx, 120, 30, [3, 4], 8)]
    q = _gen.normal(3, (11, 32, HD))
    got = call(ctx, fs, q, 32)
    check(got, fs, q)
    assert np.array_equal(got, call(ctx, fs, q, 32))                 # the same bits every time
    assert np.array_equal(got, call(ctx, fs, q, 32, device=False))
    for f in fs:
        f.close()


@pytest.mark.parametrize("rows", [0, 64, 640])
def test_fewer_rows_than_are_held_together(ctx, rows):
    f = Family(ctx, 7, 700, [20, 90, 1], 8)
    q = _gen.normal(4, (3, 32, HD))
    check(call(ctx, [f], q, 32, rows=rows), [f], q)
    f.close()


def test_agrees_with_attention_of_each_session(ctx):
    import torch
    f = Family(ctx, 9, 1025, [77, 1, 300, 64], 8)
    q = _gen.normal(5, (4, 40, HD))
    dq = torch.from_numpy(q).cuda()
    out = torch.empty_like(dq)
    torch.cuda.synchronize()
    ctx.attn_decode(f.kvs, 0, f.lens, dq, out, 40)
    ctx.sync()
    got = call(ctx, [f], q, 40)
    bound = max(attend_error(q[i], k, v) for i, (k, v) in enumerate(zip(f.k, f.v)))
    check(out.cpu().numpy(), [f], q)
    assert np.abs(got - out.cpu().numpy()).max() <= 2 * bound
    f.close()


def test_long_prompt(ctx):
    f = Family(ctx, 11, 33000, [20, 300] * 3, 2)
    q = _gen.normal(6, (6, 16, HD))
    got = call(ctx, [f], q, 16)
    check(got, [f], q)
    want = np.stack([attend(q[i], k, v) for i, (k, v) in enumerate(zip(f.k, f.v))])
    # errors of single elements have either sign: together far below their bound
    assert np.linalg.norm(got - want) <= 5e-6 * np.linalg.norm(want)
    f.close()


@pytest.mark.parametrize("scale, std", [(1.0, 1.0), (0.02, 1.0), (0.0884, 30.0), (3.0, 1.0)])
def test_scales_and_scores_that_grow(ctx, scale, std):
    """Scores of some hundreds: the reference moves often, most weights are zero."""
    f = Family(ctx, 13, 1400, [200, 90], 4, std=std)
    q = _gen.normal(8, (2, 16, HD))
    check(call(ctx, [f], q, 16, scale=scale), [f], q, scale)
    f.close()


def test_scores_in_ascending_order(ctx):
    """Every tile's scores are above all before it."""
    n, hkv = 1600, 1
    rng = np.random.default_rng(0)
    base = rng.standard_normal(HD).astype(np.float32)
    k = port().f32_to_f16((np.linspace(0, 6, n)[:, None, None] * base).astype(np.float32))
    v = f16(3, (n, hkv, HD))
    kv = ctx.kv_create(1, hkv, HD, n)
    kv.write_rows(0, 0, 0, k)
    kv.write_rows(0, 1, 0, v)
    other = kv.fork(1536)
    other.write_rows(0, 0, 1536, k[1536:])
    other.write_rows(0, 1, 1536, v[1536:])
    q = np.stack([np.stack([base, -base, base * 0, base * 1e-3])] * 2).astype(np.float32)
    out = np.empty_like(q)
    ctx.attn_decode_shared([kv, other], 0, [n, n - 1], [(2, 1536)], q, out, 4)
    for i, m in enumerate((n, n - 1)):
        want = attend(q[i], k[:m], v[:m])
        assert np.abs(out[i] - want).max() <= attend_error(q[i], k[:m], v[:m])
    kv.close()
    other.close()


@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -20, 2.0 ** 20, 2.0 ** 100])
def test_queries_of_any_size(ctx, size):
    """Queries are held against a power of two of their own row: F16 parts neither overflow nor run out of bits."""
    f = Family(ctx, 15, 300, [20, 1], 2)
    q = (_gen.normal(9, (2, 4, HD)) * np.float32(size)).astype(np.float32)
    scale = float(np.float32(0.1 / size))
    check(call(ctx, [f], q, 4, scale=scale), [f], q, scale)
    f.close()


def test_rows_behind_the_last_one_do_not_matter(ctx):
    """What a page holds behind a session's rows may be NaN or infinite (rows of a step that was taken back)."""
    f = Family(ctx, 17, 200, [20, 90], 2, max_ctx=1024)
    q = _gen.normal(10, (2, 8, HD))
    want = call(ctx, [f], q, 8)
    check(want, [f], q)
    for bits in (0x7E00, 0x7C00, 0xFC00):
        bad = np.full((40, 2, HD), bits, np.uint16)
        for kv, n in zip(f.kvs, f.lens):
            kv.write_rows(0, 0, n, bad)
            kv.write_rows(0, 1, n, bad)
        assert np.array_equal(call(ctx, [f], q, 8), want)
    f.close()


def test_nan_and_infinite_rows_stay_with_their_sessions(ctx):
    f = Family(ctx, 19, 256, [5, 40, 70], 2)
    q = _gen.normal(11, (3, 8, HD))
    want = call(ctx, [f], q, 8)
    bad = q.copy()
    bad[1, 3, 5] = np.nan
    bad[2, 0, 0] = np.inf
    got = call(ctx, [f], bad, 8)
    touched = np.zeros((3, 8), bool)
    touched[1, 3] = touched[2, 0] = True
    assert np.isnan(got[touched]).all() and np.array_equal(got[~touched], want[~touched])
    row = f16(2, (1, 2, HD))
    row[0, 1, 7] = 0x7E00                                           # a NaN key of session 1, kv head 1
    f.kvs[1].write_rows(0, 0, 256 + 3, row)
    got = call(ctx, [f], q, 8)
    assert np.isnan(got[1, 4:]).all() and np.isfinite(got[1, :4]).all()
    assert np.array_equal(got[[0, 2]], want[[0, 2]])
    f.kvs[1].write_rows(0, 0, 256 + 3, f.k[1][256 + 3:256 + 4])
    row[0, 0, 9], row[0, 1, 7] = 0x7C00, 0x3C00                      # an infinite value of session 1, kv head 0
    f.kvs[1].write_rows(0, 1, 256 + 3, row)
    got = call(ctx, [f], q, 8)
    assert np.isposinf(got[1, :4, 9]).all() and np.isfinite(np.delete(got[1, :4], 9, axis=1)).all()
    assert np.array_equal(got[[0, 2]], want[[0, 2]])
    f.close()


def test_a_row_whose_keys_all_score_minus_infinity_is_zeros(ctx):
    n = 70
    k = np.full((n, 1, HD), 0xFC00, np.uint16)                      # -inf
    v = f16(4, (n, 1, HD))
    kv = ctx.kv_create(1, 1, HD, 128)
    kv.write_rows(0, 0, 0, k)
    kv.write_rows(0, 1, 0, v)
    other = kv.fork(64)
    q = np.ones((2, 1, HD), np.float32) * np.float32(1 + 2.0 ** -12)  # (both F16 parts positive)
    out = np.full_like(q, np.nan)
    ctx.attn_decode_shared([kv, other], 0, [n, 64], [(2, 64)], q, out, 1)
    assert np.array_equal(out, np.zeros_like(out))
    kv.close()
    other.close()


@pytest.mark.parametrize("device", [True, False])
@pytest.mark.parametrize("rope, n_rot", [(True, 0), (True, 20), (False, 0)])
def test_step_appends_and_attends(ctx, device, rope, n_rot):
    import torch
    import wayruntime_b200 as wr
    hq, hkv = 16, 4
    fs = [Family(ctx, 21, 450, [30] * 3, hkv, max_ctx=600), Family(ctx, 60, 64, [7, 100], hkv, max_ctx=600)]
    kvs, lens = [kv for f in fs for kv in f.kvs], [n for f in fs for n in f.lens]
    n = len(kvs)
    q, k, v = _gen.normal(1, (n, hq, HD)), _gen.normal(2, (n, hkv, HD)), _gen.normal(3, (n, hkv, HD))
    groups = wr.Groups([(3, 448), (2, 64)])
    out = np.full_like(q, np.nan)
    if device:
        dq, dk, dv, do = (torch.from_numpy(x).cuda() for x in (q, k, v, out))
        torch.cuda.synchronize()
        ctx.decode_step_shared(kvs, 0, lens, groups, dq, dk, dv, do, hq, theta=5e5, n_rot_pairs=n_rot, rope=rope)
        ctx.sync()
        out = do.cpu().numpy()
        assert np.array_equal(dq.cpu().numpy(), q)
    else:
        given = q.copy()
        ctx.decode_step_shared(kvs, 0, lens, groups, given, k, v, out, hq, theta=5e5, n_rot_pairs=n_rot, rope=rope)
        assert np.array_equal(given, q)
    P, i = port(), 0
    for f in fs:
        for j, kv in enumerate(f.kvs):
            qr, kr = q[i:i + 1], k[i:i + 1]
            if rope:
                _, qr = P.rope(qr, lens[i], 5e5, n_rot)
                _, kr = P.rope(kr, lens[i], 5e5, n_rot)
            keys = np.concatenate([f.k[j], P.f32_to_f16(kr)])
            values = np.concatenate([f.v[j], P.f32_to_f16(v[i:i + 1])])
            assert np.array_equal(kv.read_rows(0, 0, 0, lens[i] + 1), keys)
            assert np.array_equal(kv.read_rows(0, 1, 0, lens[i] + 1), values)
            assert np.abs(out[i] - attend(qr[0], keys, values)).max() <= attend_error(qr[0], keys, values)
            i += 1
    for f in fs:
        f.close()


def test_steps_on_the_heels_of_one_another(ctx):
    """Appends, shared attention, a reorder and attention of each session, back to back without a wait."""
    import torch
    hq, hkv = 16, 4
    f = Family(ctx, 23, 300, [10] * 4, hkv, max_ctx=400)
    rows = [[list(x) for x in zip(k, v)] for k, v in zip(f.k, f.v)]
    keys, values = [list(k) for k in f.k], [list(v) for v in f.v]
    q, k, v = (torch.from_numpy(_gen.normal(s, (12, 4, h, HD))).cuda() for s, h in ((1, hq), (2, hkv), (3, hkv)))
    outs = torch.empty((12, 2, 4, hq, HD), device="cuda")
    torch.cuda.synchronize()
    P, at = port(), list(f.lens)
    plan = [[0, 1, 2, 3], [1, 0, 3, 2], [2, 2, 0, 1], [3, 3, 3, 3], [0, 0, 2, 2], [1, 2, 3, 0]] * 2
    want = []
    for i, parents in enumerate(plan):
        ctx.kv_reorder(f.kvs, parents, at)
        ctx.decode_step_shared(f.kvs, 0, at, [(4, 256)], q[i], k[i], v[i], outs[i, 0], hq, rope=False)
        at = [n + 1 for n in at]
        ctx.attn_decode(f.kvs, 0, at, q[i], outs[i, 1], hq)
        keys = [list(keys[p]) + [P.f32_to_f16(k[i, s:s + 1].cpu().numpy())[0]] for s, p in enumerate(parents)]
        values = [list(values[p]) + [P.f32_to_f16(v[i, s:s + 1].cpu().numpy())[0]] for s, p in enumerate(parents)]
        want.append([(np.stack(a), np.stack(b)) for a, b in zip(keys, values)])
    ctx.sync()
    got, qs = outs.cpu().numpy(), q.cpu().numpy()
    for i in range(12):
        for s in range(4):
            a, b = want[i][s]
            for which in (0, 1):
                assert np.abs(got[i, which, s] - attend(qs[i, s], a, b)).max() <= attend_error(qs[i, s], a, b), (i, which, s)
    f.close()


def test_a_session_alone_whose_full_pages_count_as_shared(ctx):
    """What a step has just written is among the next one's shared rows: with the page's last row at 63, 127 ..., the group of the
    next call takes that page in."""
    import torch
    hq, hkv, start, steps = 8, 2, 60, 72
    kv = ctx.kv_create(1, hkv, HD, start + steps)
    keys, values = f16(900, (start, hkv, HD)), f16(901, (start, hkv, HD))
    kv.write_rows(0, 0, 0, keys)
    kv.write_rows(0, 1, 0, values)
    q = [_gen.normal(910 + i, (1, hq, HD)) for i in range(steps)]
    k = [_gen.normal(1010 + i, (1, hkv, HD)) for i in range(steps)]
    v = [_gen.normal(1110 + i, (1, hkv, HD)) for i in range(steps)]
    dq, dk, dv = ([torch.from_numpy(x).cuda() for x in a] for a in (q, k, v))
    out = [torch.full((1, hq, HD), float("nan"), device="cuda") for _ in range(steps)]
    torch.cuda.synchronize()
    for i in range(steps):
        at = start + i
        ctx.decode_step_shared([kv], 0, [at], [(1, at // 64 * 64)], dq[i], dk[i], dv[i], out[i], hq, rope=False)
    ctx.sync()
    P = port()
    for i in range(steps):
        keys = np.concatenate([keys, P.f32_to_f16(k[i])])
        values = np.concatenate([values, P.f32_to_f16(v[i])])
        err = np.abs(out[i].cpu().numpy()[0] - attend(q[i][0], keys, values)).max()
        assert err <= attend_error(q[i][0], keys, values), (i, err)
    kv.close()


def test_a_fork_right_behind_a_step(ctx):
    """The step fills a page, the fork shares it, and the attention behind that reads it as a shared one."""
    import torch
    hq, hkv = 8, 2
    for trial, rows in enumerate((63, 127, 191, 127)):
        kv = ctx.kv_create(1, hkv, HD, 320)
        keys, values = f16(1200 + trial, (rows, hkv, HD)), f16(1210 + trial, (rows, hkv, HD))
        kv.write_rows(0, 0, 0, keys)
        kv.write_rows(0, 1, 0, values)
        q, q2 = _gen.normal(1220 + trial, (1, hq, HD)), _gen.normal(1230 + trial, (3, hq, HD))
        k, v = _gen.normal(1240 + trial, (1, hkv, HD)), _gen.normal(1250 + trial, (1, hkv, HD))
        dq, dq2, dk, dv = (torch.from_numpy(x).cuda() for x in (q, q2, k, v))
        out, out2 = torch.empty((1, hq, HD), device="cuda"), torch.full((3, hq, HD), float("nan"), device="cuda")
        torch.cuda.synchronize()
        ctx.decode_step_shared([kv], 0, [rows], [(1, 0)], dq, dk, dv, out, hq, rope=False)
        forks = [kv.fork(rows + 1) for _ in range(2)]
        ctx.attn_decode_shared([kv] + forks, 0, [rows + 1] * 3, [(3, rows + 1)], dq2, out2, hq)
        ctx.sync()
        P = port()
        keys, values = np.concatenate([keys, P.f32_to_f16(k)]), np.concatenate([values, P.f32_to_f16(v)])
        got = out2.cpu().numpy()
        for s in range(3):
            assert np.abs(got[s] - attend(q2[s], keys, values)).max() <= attend_error(q2[s], keys, values), (trial, s)
        for x in forks + [kv]:
            x.close()


def test_many_query_heads_to_a_kv_head(ctx):
    """More than 64 queries of one session and kv head: they are split into several lists, which all append the same row."""
    import torch
    for hq, hkv in ((96, 1), (130, 1), (144, 2)):
        fam = Family(ctx, 1300 + hq, 130, [3, 70], hkv, max_ctx=256)
        q = _gen.normal(1310 + hq, (2, hq, HD))
        check(call(ctx, [fam], q, hq), [fam], q)
        k, v = _gen.normal(1320 + hq, (2, hkv, HD)), _gen.normal(1330 + hq, (2, hkv, HD))
        dq, dk, dv = (torch.from_numpy(x).cuda() for x in (q, k, v))
        out = torch.full((2, hq, HD), float("nan"), device="cuda")
        torch.cuda.synchronize()
        ctx.decode_step_shared(fam.kvs, 0, fam.lens, [(2, fam.rows)], dq, dk, dv, out, hq, rope=False)
        ctx.sync()
        P = port()
        for i in range(2):
            fam.k[i] = np.concatenate([fam.k[i], P.f32_to_f16(k[i:i + 1])])
            fam.v[i] = np.concatenate([fam.v[i], P.f32_to_f16(v[i:i + 1])])
        check(out.cpu().numpy(), [fam], q)
        fam.close()


@pytest.mark.parametrize("own, rows", [([1] * 16, 64), ([1] * 16, 0), ([40, 1, 200, 64] * 4, 64)])
def test_more_short_lists_than_multiprocessors(ctx, own, rows):
    """16 sessions with 128 query heads to each of 8 kv heads are 256 lists of a tile or two; launch behind launch."""
    import torch
    hq, hkv = 1024, 8
    fam = Family(ctx, 1500, 64, own, hkv)
    q = _gen.normal(1510, (16, hq, HD))
    dq = torch.from_numpy(q).cuda()
    out = torch.full((6, 16, hq, HD), float("nan"), device="cuda")
    torch.cuda.synchronize()
    for o in out:
        ctx.attn_decode_shared(fam.kvs, 0, fam.lens, [(16, rows)], dq, o, hq)
    ctx.sync()
    check(out[0].cpu().numpy(), [fam], q)
    assert all(torch.equal(o, out[0]) for o in out)
    fam.close()


def test_a_wait_that_ran_out_elsewhere_does_not_stay(ctx):
    """An exchange whose peer never answers ends with an error (its wait is short); the calls behind it give the right answer."""
    import torch
    import wayruntime_b200 as wr
    fam = Family(ctx, 1400, 300, [5, 6, 7], 2)
    q = _gen.normal(1410, (3, 8, HD))
    xs = [wr.Exchange(ctx, 2, r, 8, HD) for r in range(2)]
    wr.Exchange.connect_local(xs)
    triples, out = torch.zeros((8, 4 + HD), device="cuda"), torch.zeros((8, HD), device="cuda")
    for _ in range(2):
        check(call(ctx, [fam], q, 8), [fam], q)
        torch.cuda.synchronize()
        ctx.set_wait_limit(200_000)
        xs[0].combine(8, triples, out)                           # (the other one never steps)
        ctx.set_wait_limit(4_000_000_000)
        with pytest.raises(wr.WrCudaError) as e:
            ctx.sync()
        assert e.value.status == -10
    check(call(ctx, [fam], q, 8), [fam], q)
    for x in xs:
        x.close()
    fam.close()


def test_captured_in_a_graph(ctx):
    import torch
    f = Family(ctx, 25, 700, [30, 40], 8)
    q = _gen.normal(12, (2, 16, HD))
    dq, out = torch.from_numpy(q).cuda(), torch.zeros((2, 16, HD), device="cuda")
    torch.cuda.synchronize()
    ctx.attn_decode_shared(f.kvs, 0, f.lens, [(2, 640)], dq, out, 16)
    ctx.sync()
    stream, graph = torch.cuda.ExternalStream(ctx.stream), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for _ in range(3):
            ctx.attn_decode_shared(f.kvs, 0, f.lens, [(2, 640)], dq, out, 16)
    other = Family(ctx, 30, 30000, [100] * 8, 8)                     # the scratch grows between capture and launch
    check(call(ctx, [other], _gen.normal(13, (8, 64, HD)), 64), [other], _gen.normal(13, (8, 64, HD)))
    q2 = _gen.normal(14, (2, 16, HD))
    dq.copy_(torch.from_numpy(q2))
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph.replay()
        graph.replay()
    ctx.sync()
    check(out.cpu().numpy(), [f], q2)
    f.close()
    other.close()


def test_refusals(ctx):
    import torch
    import wayruntime_b200 as wr
    f = Family(ctx, 27, 200, [10, 20], 2)
    q = np.zeros((2, 4, HD), np.float32)
    out = np.zeros_like(q)
    stranger = ctx.kv_create(1, 2, HD, 221)

    def status(kvs, lens, groups, heads=4, layer=0):
        with pytest.raises(wr.WrCudaError) as e:
            ctx.attn_decode_shared(kvs, layer, lens, groups, q, out, heads)
        return e.value.status
    assert status(f.kvs, f.lens, [(2, 100)]) == -4                   # not whole pages
    assert status(f.kvs, f.lens, [(2, 256)]) == -4                   # more than they hold together
    assert status([f.kvs[0], stranger], f.lens, [(2, 64)]) == -4     # not the same pages
    assert status(f.kvs, [100, 210], [(2, 192)]) == -4               # more than one of them attends
    assert status(f.kvs, f.lens, [(2, 192)], heads=3) == -4
    assert status(f.kvs, f.lens, [(2, 192)], layer=1) == -4
    assert status(f.kvs, [0, 5], [(2, 0)]) == -4
    assert status(f.kvs, [500, 5], [(2, 0)]) == -4
    assert status([f.kvs[0], f.kvs[0]], f.lens, [(2, 64)]) == -4
    with pytest.raises(ValueError):
        ctx.attn_decode_shared(f.kvs, 0, f.lens, [(3, 64)], q, out, 4)
    small = ctx.kv_create(1, 2, 64, 100)
    with pytest.raises(wr.WrCudaError) as e:
        ctx.attn_decode_shared([small], 0, [5], [(1, 0)], np.zeros((1, 4, 64), np.float32), np.zeros((1, 4, 64), np.float32), 4)
    assert e.value.status == -3
    one = torch.zeros(2 * 4 * HD + 1, device="cuda")[1:].view(2, 4, HD)
    with pytest.raises(wr.WrCudaError) as e:
        ctx.attn_decode_shared(f.kvs, 0, f.lens, [(2, 192)], one, one, 4)       # rows that 16-byte vectors cannot read
    assert e.value.status == -4
    with pytest.raises(wr.WrCudaError) as e:                          # the row to append lies in a page that both hold
        ctx.decode_step_shared(f.kvs, 0, [100, 215], [(2, 64)], q, np.zeros((2, 2, HD), np.float32), np.zeros((2, 2, HD), np.float32), out, 4)
    assert e.value.status == -7
    both = torch.zeros(3 * 4 * HD, device="cuda")
    dq, k, v = both[:2 * 4 * HD].view(2, 4, HD), torch.zeros((2, 2, HD), device="cuda"), torch.zeros((2, 2, HD), device="cuda")
    far = torch.zeros_like(dq)
    for o in (dq, both[4 * HD:].view(2, 4, HD)):                      # a result in what is read
        with pytest.raises(wr.WrCudaError) as e:
            ctx.attn_decode_shared(f.kvs, 0, f.lens, [(2, 192)], dq, o, 4)
        assert e.value.status == -4
    for kk, vv in ((far.view(-1)[:2 * 2 * HD].view(2, 2, HD), v), (k, far.view(-1)[4 * HD:].view(2, 2, HD))):
        with pytest.raises(wr.WrCudaError) as e:
            ctx.decode_step_shared(f.kvs, 0, f.lens, [(2, 192)], dq, kk, vv, far, 4)
        assert e.value.status == -4
    lib, h = ctx._lib, ctx._handles(f.kvs)
    u = ctx._u32s
    p = q.ctypes.data
    for sizes, rows in (([1], [64]), ([0, 2], [0, 64]), ([3], [64]), ([1, 1, 1], [0, 0, 0])):
        assert lib.wr_cuda_attn_decode_shared(ctx._h, 2, h, 0, u(f.lens), len(sizes), u(sizes), u(rows), p, p, 4, 0.0, 0) == -4
    assert lib.wr_cuda_attn_decode_shared(ctx._h, 2, h, 0, u(f.lens), 1, None, u([64]), p, p, 4, 0.0, 0) == -4
    stranger.close()
    small.close()
    f.close()
