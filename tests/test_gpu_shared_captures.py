"""GPU: shared attention and beam selection around stream captures."""
import numpy as np
import pytest

import _gen
from _cuda_util import port
from _plain_beams import attend, attend_error
from test_gpu_shared_attention import HD, ctx  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [2048, 4096])
def test_a_captured_call_is_none_that_has_run(ctx, rows):  # noqa: F811
    """Rows are appended, a fork shares them, a call is captured without running, and the same call runs right behind the append."""
    import torch
    hq, hkv = 32, 8
    for trial in range(4):
        kv = ctx.kv_create(1, hkv, HD, rows + 64)
        k, v = _gen.normal(10 + trial, (rows, hkv, HD)), _gen.normal(20 + trial, (rows, hkv, HD))
        q = _gen.normal(30 + trial, (3, hq, HD))
        dq, dk, dv = (torch.from_numpy(x).cuda() for x in (q, k, v))
        out, again = (torch.full((3, hq, HD), float("nan"), device="cuda") for _ in range(2))
        stream, graph = torch.cuda.ExternalStream(ctx.stream), torch.cuda.CUDAGraph()
        warm = ctx.kv_create(1, hkv, HD, rows + 64)                  # (the call's scratch is there before it is captured)
        warms = [warm] + [warm.fork(rows) for _ in range(2)]
        ctx.attn_decode_shared(warms, 0, [rows] * 3, [(3, rows)], dq, out, hq)
        torch.cuda.synchronize()
        ctx.kv_append([kv], 0, [0], dk, dv, rope=False, n_tokens=rows)
        forks = [kv.fork(rows) for _ in range(2)]
        with torch.cuda.graph(graph, stream=stream):
            ctx.attn_decode_shared([kv] + forks, 0, [rows] * 3, [(3, rows)], dq, again, hq)
        ctx.attn_decode_shared([kv] + forks, 0, [rows] * 3, [(3, rows)], dq, out, hq)
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.sync()
        P = port()
        keys, values = P.f32_to_f16(k), P.f32_to_f16(v)
        got = out.cpu().numpy()
        for s in range(3):
            err, bound = np.abs(got[s] - attend(q[s], keys, values)).max(), attend_error(q[s], keys, values)
            assert err <= bound, (trial, s)
        assert torch.equal(out, again)
        del graph
        for x in [kv] + forks + warms:
            x.close()


def test_scratch_does_not_grow_while_a_capture_runs():
    """The call is refused, also where the capture would let memory be allocated; calls before and behind it are right."""
    import torch
    import wayruntime_b200 as wr
    from test_gpu_beam_select import check, rows as logit_rows
    c = wr.Context(0)
    kv = c.kv_create(1, 8, HD, 2048)
    fork = kv.fork(1024)                                             # (rows of zeros: their lengths alone matter)
    q, out = torch.zeros((2, 1024, HD), device="cuda"), torch.zeros((2, 1024, HD), device="cuda")

    def beams(seed, groups, n, vocab, n_out):
        logits, scores = logit_rows(seed, groups, n, vocab)
        o = (torch.zeros((groups, n_out), device="cuda"), *(torch.zeros((groups, n_out), dtype=torch.int32, device="cuda") for _ in range(2)))
        return logits, scores, torch.from_numpy(logits).cuda(), torch.from_numpy(scores).cuda(), o

    def right(b):
        c.sync()
        check((b[4][0].cpu().numpy(), b[4][1].cpu().numpy().view(np.uint32), b[4][2].cpu().numpy().view(np.uint32)), b[0], b[1], b[4][0].shape[1])

    def refused(call):
        with pytest.raises(wr.WrCudaError) as e:
            call()
        assert e.value.status == -7
    small, large = beams(1, 1, 4, 20011, 8), beams(2, 2600, 16, 300, 32)     # (10.6 MB of scratch, more than a context begins with)
    stream = torch.cuda.ExternalStream(c.stream)
    empty = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(empty, stream=stream, capture_error_mode="relaxed"):
        refused(lambda: c.beam_select(small[2], small[3], *small[4]))
        refused(lambda: c.attn_decode_shared([kv, fork], 0, [1024, 1024], [(2, 1024)], q, out, 1024))
    c.beam_select(small[2], small[3], *small[4])
    right(small)
    graph = torch.cuda.CUDAGraph()
    small[4][1].zero_()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
        refused(lambda: c.beam_select(large[2], large[3], *large[4]))
        c.beam_select(small[2], small[3], *small[4])
    c.beam_select(large[2], large[3], *large[4])
    right(large)
    with torch.cuda.stream(stream):
        graph.replay()
    right(small)
    del graph, empty
    for x in (kv, fork):
        x.close()
    c.close()
