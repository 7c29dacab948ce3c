"""GPU: sessions that go on from one another (wr_cuda_kv_fork, wr_cuda_kv_reorder)."""
import itertools

import numpy as np
import pytest

import _gen

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ctx():
    import wayruntime_b200 as wr
    c = wr.Context(0, attn_max_seq=8192)
    yield c
    c.close()


def bits(seed, n, heads, dim):
    return (_gen.uniform_u32(seed, (n, heads, dim)) & 0x3BFF).astype(np.uint16)      # finite F16 patterns


def write(kv, row0, rows):
    """rows[layer][which]"""
    for layer, pair in enumerate(rows):
        for which, x in enumerate(pair):
            if len(x):
                kv.write_rows(layer, which, row0, np.ascontiguousarray(x))


def holds(kv, want):
    """want[layer][which]: the rows from the first on"""
    return all(np.array_equal(kv.read_rows(layer, which, 0, len(x)), x) for layer, pair in enumerate(want) for which, x in enumerate(pair))


def some(seed, n, layers, heads, dim):
    return [[bits(seed + 2 * i + w, n, heads, dim) for w in (0, 1)] for i in range(layers)]


def joined(a, b):
    return [[np.concatenate([x, y]) for x, y in zip(p, r)] for p, r in zip(a, b)]


def cut(a, n):
    return [[x[:n] for x in p] for p in a]


@pytest.mark.parametrize("dim, heads, layers", [(128, 2, 3), (64, 1, 1), (6, 3, 2), (256, 1, 2)])
@pytest.mark.parametrize("n", [0, 1, 63, 64, 65, 128, 200, 256])
def test_fork_holds_the_first_rows(ctx, dim, heads, layers, n):
    kv = ctx.kv_create(layers, heads, dim, 256)
    have = some(1, 256, layers, heads, dim)
    write(kv, 0, have)
    f = kv.fork(n)
    assert holds(f, cut(have, n)) and f.shared_rows(kv) == kv.shared_rows(f) == n // 64 * 64
    if n < 256:
        mine = some(100, 256 - n, layers, heads, dim)
        write(f, n, mine)
        assert holds(f, joined(cut(have, n), mine)) and holds(kv, have)
        write(kv, n, some(200, 256 - n, layers, heads, dim))         # (the parent's own rows, in pages of its own)
        assert holds(f, joined(cut(have, n), mine))
    kv.close()
    assert holds(f, cut(have, n))                                    # a fork outlives its parent
    f.close()


def test_pages_that_several_hold_are_not_written(ctx):
    import wayruntime_b200 as wr
    kv = ctx.kv_create(1, 2, 128, 512)
    have = some(3, 300, 1, 2, 128)
    write(kv, 0, have)
    f = kv.fork(300)
    x = np.zeros((1, 2, 128), np.float32)
    for s in (kv, f):
        with pytest.raises(wr.WrCudaError) as e:
            s.write_rows(0, 0, 255, bits(1, 1, 2, 128))
        assert e.value.status == -7
        with pytest.raises(wr.WrCudaError) as e:
            ctx.kv_append([s], 0, [100], x, x)
        assert e.value.status == -7
        with pytest.raises(wr.WrCudaError) as e:
            ctx.decode_step([s], 0, [0], np.zeros((1, 2, 128), np.float32), x, x, np.zeros((1, 2, 128), np.float32), 2)
        assert e.value.status == -7
        s.write_rows(0, 0, 256, bits(9, 1, 2, 128))                  # (behind them each may)
    g = f.fork(64)                                                   # holds the first page alone with both
    kv.close()
    with pytest.raises(wr.WrCudaError):
        f.write_rows(0, 0, 63, bits(1, 1, 2, 128))
    f.write_rows(0, 0, 64, bits(2, 2, 2, 128))                       # nobody else holds the second one any more
    g.close()
    f.write_rows(0, 0, 0, bits(1, 1, 2, 128))
    f.close()


def test_pages_go_back_once_and_clean(ctx):
    """Forks of forks, given back in every order: no page is handed out twice, and what comes back is zeros."""
    for order in itertools.permutations(range(4)):
        a = ctx.kv_create(2, 1, 128, 320)
        have = some(5, 320, 2, 1, 128)
        write(a, 0, have)
        b = a.fork(320)
        c = b.fork(130)
        d = a.fork(64)
        kvs = [a, b, c, d]
        lens = [320, 320, 130, 64]
        for i, at in enumerate(order):
            kvs[at].close()
            for rest in order[i + 1:]:
                assert holds(kvs[rest], cut(have, lens[rest]))
        fresh = [ctx.kv_create(2, 1, 128, 320) for _ in range(4)]
        for i, kv in enumerate(fresh):
            assert holds(kv, [[np.zeros((320, 1, 128), np.uint16)] * 2] * 2)
            write(kv, 0, some(50 + i, 320, 2, 1, 128))
        for i, kv in enumerate(fresh):
            assert holds(kv, some(50 + i, 320, 2, 1, 128))
            kv.close()


@pytest.mark.parametrize("prompt, own", [(0, 5), (70, 0), (70, 1), (64, 100), (130, 60), (100, 260)])
@pytest.mark.parametrize("parents", [[0, 1, 2, 3], [3, 2, 1, 0], [1, 2, 3, 0], [2, 2, 2, 2], [0, 0, 3, 3], [1, 1, 0, 0], [3, 0, 0, 0], [1, 0, 1, 0]])
def test_reorder(ctx, prompt, own, parents):
    layers, heads, dim = 2, 2, 128
    first = ctx.kv_create(layers, heads, dim, 448)
    shared = some(7, prompt, layers, heads, dim)
    write(first, 0, shared)
    kvs = [first] + [first.fork(prompt) for _ in range(3)]
    have = []
    for i, kv in enumerate(kvs):
        have.append(joined(shared, some(100 + 10 * i, own + i, layers, heads, dim)))     # (beams of unequal lengths)
        write(kv, prompt, [[x[prompt:] for x in p] for p in have[i]])
    ctx.kv_reorder(kvs, parents, [prompt + own + i for i in range(4)])
    for i, p in enumerate(parents):
        assert holds(kvs[i], have[p]), i
    # each can go on by itself
    for i, p in enumerate(parents):
        write(kvs[i], prompt + own + p, some(300 + i, 3, layers, heads, dim))
    for i, p in enumerate(parents):
        assert holds(kvs[i], joined(have[p], some(300 + i, 3, layers, heads, dim))), i
    for kv in kvs:
        kv.close()


def test_many_layers_of_unlike_pages(ctx):
    """More layers than one launch takes, and sessions that were never forked."""
    layers = 300
    import ctypes as C
    from wayruntime_b200.binding import CacheLayer, KVCache, _check
    desc = (CacheLayer * layers)()
    for i in range(layers):
        desc[i] = CacheLayer(0 if i % 5 == 4 else 1 + i % 2, 128 if i % 3 else 10, 128 if i % 3 else 10, 1, 0)
    kvs = []
    for _ in range(3):
        h = C.c_void_p()
        _check(ctx._lib.wr_cuda_kv_create_layout(ctx._h, layers, desc, 100, C.byref(h)), "create")
        kvs.append(KVCache._of_handle(ctx, h, 100))
    def shape(i):
        return 1 + i % 2, 128 if i % 3 else 10
    def rows(kv, i, w, n):
        kv.n_kv_heads, kv.head_dim = shape(i)
        return kv.read_rows(i, w, 0, n)
    for s, kv in enumerate(kvs):
        for i in range(layers):
            if i % 5 != 4:
                for w in (0, 1):
                    kv.write_rows(i, w, 0, bits(s * 1000 + 2 * i + w, 70, *shape(i)))
    ctx.kv_reorder(kvs, [2, 2, 2], [70, 70, 70])
    for kv in kvs:
        for i in range(layers):
            if i % 5 != 4:
                for w in (0, 1):
                    assert np.array_equal(rows(kv, i, w, 70), bits(2000 + 2 * i + w, 70, *shape(i))), i
    for kv in kvs:
        kv.close()


def test_rows_behind_those_that_go_on_are_left_alone(ctx):
    a, b = (ctx.kv_create(1, 1, 128, 128) for _ in range(2))
    write(a, 0, some(1, 100, 1, 1, 128))
    write(b, 0, some(5, 128, 1, 1, 128))
    ctx.kv_reorder([a, b], [0, 0], [30, 128])
    want = some(5, 128, 1, 1, 128)
    for w in (0, 1):
        want[0][w][:30] = some(1, 100, 1, 1, 128)[0][w][:30]
    assert holds(b, want) and holds(a, some(1, 100, 1, 1, 128))
    a.close()
    b.close()


def test_memory_whose_further_pages_somebody_holds_is_not_taken(ctx):
    """The child of a session with fewer rows could not go on in it: the page behind them is held by another session too."""
    import wayruntime_b200 as wr
    a = ctx.kv_create(2, 2, 128, 300)
    rows = some(300, 200, 2, 2, 128)
    write(a, 0, rows)
    short, other = a.fork(64), a.fork(200)
    with pytest.raises(wr.WrCudaError) as e:
        ctx.kv_reorder([short, a, other], [0, 0, 2], [64, 200, 200])
    assert e.value.status == -7
    for kv, n in ((short, 64), (a, 200), (other, 200)):
        assert holds(kv, cut(rows, n))
    other.close()
    ctx.kv_reorder([short, a], [0, 0], [64, 200])
    more = some(310, 70, 2, 2, 128)
    for kv in (short, a):
        assert holds(kv, cut(rows, 64))
        write(kv, 64, more)
        assert holds(kv, joined(cut(rows, 64), more))
        kv.close()


def test_refusals_change_nothing(ctx):
    import torch
    import wayruntime_b200 as wr
    kvs = [ctx.kv_create(1, 2, 128, 256) for _ in range(2)]
    have = [some(1 + 10 * i, 200, 1, 2, 128) for i in range(2)]
    for kv, x in zip(kvs, have):
        write(kv, 0, x)
    shorter = ctx.kv_create(1, 2, 128, 255)
    wider = ctx.kv_create(1, 1, 128, 256)
    outside = kvs[1].fork(128)

    def status(*args):
        with pytest.raises(wr.WrCudaError) as e:
            ctx.kv_reorder(*args)
        return e.value.status
    assert status(kvs, [0, 2], [200, 200]) == -4
    assert status([kvs[0], kvs[0]], [0, 0], [200, 200]) == -4
    assert status([kvs[0], shorter], [0, 1], [1, 1]) == -4
    assert status([kvs[0], wider], [0, 1], [1, 1]) == -4
    assert status(kvs, [0, 1], [200, 257]) == -6
    assert status(kvs, [0, 0], [200, 200]) == -7                     # what session 1 would copy into is held outside too
    assert status([], [], []) == -4
    with pytest.raises(ValueError):
        ctx.kv_reorder(kvs, [0], [1, 1])
    for n in (257, 1000):
        with pytest.raises(wr.WrCudaError) as e:
            kvs[0].fork(n)
        assert e.value.status == -6
    stream, graph = torch.cuda.ExternalStream(ctx.stream), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        assert status(kvs, [1, 0], [200, 200]) == -7
        with pytest.raises(wr.WrCudaError) as e:
            kvs[0].fork(10)
        assert e.value.status == -7
    assert all(holds(kv, x) for kv, x in zip(kvs, have))
    other = wr.Context(0)
    elsewhere = other.kv_create(1, 2, 128, 256)
    assert status([kvs[0], elsewhere], [0, 1], [1, 1]) == -4
    assert kvs[0].shared_rows(elsewhere) == 0 and kvs[0].shared_rows(kvs[0]) == 0
    ctx.kv_reorder(kvs, [1, 0], [200, 200])                          # (nothing is copied: what is held outside may stay)
    assert holds(kvs[0], have[1]) and holds(kvs[1], have[0]) and outside.shared_rows(kvs[0]) == 128
    for kv in (*kvs, shorter, wider, outside, elsewhere):
        kv.close()
    other.close()
