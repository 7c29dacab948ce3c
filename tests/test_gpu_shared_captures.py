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
