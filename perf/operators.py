"""Beam search's operators, and batches that share a prompt, as cases that can be timed and checked.

Three things are called.  `beam_select`: the best continuations of every request over its beams and the vocabulary, from rows
of logits.  `attn_decode_shared`: one new token's attention for sessions whose first rows are the same pages of the cache.
`kv_reorder` with `decode_step_shared` for every layer: the caches follow the chosen beams, the new rows are appended, attention.

A case is a dict: "kind" says which of these, the rest are sizes.  Where `own` is false `run` computes the same in elementary
torch operations; `exact` restates it in 64 bits.
"""
import math
import random
import zlib

import torch

own = False

HEAD_DIM = 128
PAGE = 64                            # rows of a page: what sessions share is whole pages


def listed():
    select = {"kind": "select", "masked": False}
    attend = {"kind": "attend", "groups": 1, "heads": 32, "kv_heads": 8}
    step = {"kind": "step", "heads": 16, "kv_heads": 8}
    return [
        # the first step of a search: one prompt's last row, twice as many continuations as beams
        dict(select, name="select_first", requests=1, beams=1, vocab=32003, n_out=8),
        # one request's four beams over a large vocabulary
        dict(select, name="select_4_beams", requests=1, beams=4, vocab=151936, n_out=8),
        # a full decode batch: four requests of four beams
        dict(select, name="select_batch_16", requests=4, beams=4, vocab=151936, n_out=8),
        # many requests of eight beams whose vocabulary a grammar has masked
        dict(select, name="select_masked_256", requests=32, beams=8, vocab=65536, n_out=16, masked=True),
        # two short beams of a chat with a small model
        dict(attend, name="attend_short", sessions=2, prompt=150, gen_lo=1, gen_hi=20, heads=16),
        # four beams over a prompt of an odd length
        dict(attend, name="attend_4_beams", sessions=4, prompt=2011, gen_lo=90, gen_hi=90),
        # four requests with different long prompts, four beams each, five query heads to a key head
        dict(attend, name="attend_4x4", groups=4, sessions=4, prompt=4096, gen_lo=128, gen_hi=128, heads=40),
        # sixteen conversations of unequal lengths behind one system prompt
        dict(attend, name="attend_system_prompt", sessions=16, prompt=6000, gen_lo=50, gen_hi=1500),
        # sixteen answers to one question about a long document
        dict(attend, name="attend_document", sessions=16, prompt=32768, gen_lo=20, gen_hi=300),
        # one step of a search through all layers of a small model: half of the beams go on, twice each
        dict(step, name="step_4_beams", layers=28, sessions=4, prompt=500, gen_lo=75, gen_hi=75, kept=2),
        # a wide search far into its answers: sixteen beams, six of them end
        dict(step, name="step_16_beams", layers=8, sessions=16, prompt=3000, gen_lo=700, gen_hi=700, kept=10, heads=32),
    ]


def spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["select", "attend", "attend", "step"])
    if kind == "select":
        beams, vocab = rng.choice([1, 2, 3, 4, 5, 8, 16]), spread(rng, 1000, 151936)
        most = max(1, 16_000_000 // (beams * vocab))
        return {"kind": kind, "requests": min(most, spread(rng, 1, 64)), "beams": beams, "vocab": vocab,
                "n_out": rng.choice([beams, 2 * beams, 2 * beams]), "masked": rng.random() < 0.3}
    kv = rng.choice([1, 2, 4, 8, 8])
    heads = kv * rng.choice([1, 2, 2, 4, 4, 5, 8])
    if kind == "attend":
        groups = rng.choice([1, 1, 1, 2, 3, 4])
        sessions, prompt, top = spread(rng, 1, 16 // groups), spread(rng, 1, 32768 // groups), spread(rng, 1, 2000)
        return {"kind": kind, "groups": groups, "sessions": sessions, "prompt": prompt, "gen_lo": max(1, top // rng.choice([1, 2, 8])),
                "gen_hi": top, "heads": heads, "kv_heads": kv}
    sessions, prompt, gen = spread(rng, 2, 16), spread(rng, 1, 4000), spread(rng, 1, 800)
    most = max(1, 60_000 // (prompt + sessions * gen))
    return {"kind": kind, "layers": min(most, spread(rng, 1, 28)), "sessions": sessions, "prompt": prompt, "gen_lo": gen, "gen_hi": gen,
            "kept": rng.randint(1, sessions), "heads": heads, "kv_heads": kv}


# ---- inputs

def normal(shape, *what, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(zlib.crc32(repr(what).encode()))
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale)


def logit_rows(case, seed):
    """Logits as a language model's head gives them; a grammar leaves about one token in eight."""
    shape = (case["requests"], case["beams"], case["vocab"])
    x = normal(shape, "logits", seed, scale=2.5)
    if case["masked"]:
        x.masked_fill_(normal(shape, "mask", seed) < 1.15, -math.inf)
    return x


def beam_scores(case, seed):
    """Sums of log probabilities so far: beams of one request lie within a few units of each other."""
    return -20.0 - normal((case["requests"], case["beams"]), "scores", seed).abs() * (1.5 if case["beams"] > 1 else 0.0)


def lengths(case, seed):
    """Rows that each session holds beyond the prompt, [group][session]."""
    r = random.Random(seed)
    return [[r.randint(case["gen_lo"], case["gen_hi"]) for _ in range(case["sessions"])] for _ in range(case.get("groups", 1))]


def parents(case, seed):
    """For every beam the one that it goes on from: `kept` of them do, in an order that scores give."""
    r = random.Random(zlib.crc32(repr(("parents", seed)).encode()))
    alive = r.sample(range(case["sessions"]), case["kept"])
    return r.sample(alive + [r.choice(alive) for _ in range(case["sessions"] - case["kept"])], case["sessions"])


def cache_rows(case, seed):
    """F16 keys (of unit scale, as after the head norm) and values of every layer: the prompt's [layers][2][groups][rows][kv
    heads][head dim], and what follows it, [layers][2][groups][sessions][rows][kv heads][head dim]."""
    layers, groups, kv = case.get("layers", 1), case.get("groups", 1), case["kv_heads"]
    most = case["gen_hi"] + (1 if case["kind"] == "step" else 0)       # (a step's own row is there, empty)
    own_rows = torch.empty((layers, 2, groups, case["sessions"], most, kv, HEAD_DIM), dtype=torch.float16, device="cuda")
    shared = torch.empty((layers, 2, groups, case["prompt"], kv, HEAD_DIM), dtype=torch.float16, device="cuda")
    for i in range(layers):
        for which, scale in ((0, 1.0), (1, 0.64)):
            shared[i, which] = normal(shared.shape[2:], "prompt", seed, i, which, scale=scale)
            own_rows[i, which] = normal(own_rows.shape[2:], "gen", seed, i, which, scale=scale)
    return shared, own_rows


def new_rows(case, seed):
    """F32 rows of every layer as projections, norms and rotation leave them: queries, keys, values."""
    n = case.get("groups", 1) * case["sessions"]
    shape = lambda h: (case.get("layers", 1), n, h, HEAD_DIM)  # noqa: E731
    return [normal(shape(h), name, seed, scale=s) for name, h, s in
            (("q", case["heads"], 1.0), ("k", case["kv_heads"], 1.0), ("v", case["kv_heads"], 0.64))]


_CONTEXT = []


def context():
    """The process's one device context, as a program keeps it."""
    import wayruntime_b200 as wr
    if not _CONTEXT:
        _CONTEXT.append(wr.Context(0, attn_max_seq=65536))
    return _CONTEXT[0]


def sessions_of(case, shared, own_rows, lens):
    """The sessions as a search has them: one that has taken the prompt, the others forked from it, their own rows behind it."""
    ctx, kvs, prompt = context(), [], case["prompt"]
    torch.cuda.synchronize()
    for g, of_group in enumerate(lens):
        first = ctx.kv_create(shared.shape[0], case["kv_heads"], HEAD_DIM, prompt + max(of_group) + 1)
        for i in range(shared.shape[0]):
            for which in (0, 1):
                first.write_rows(i, which, 0, shared[i, which, g])
        family = [first] + [first.fork(prompt) for _ in of_group[1:]]
        for s, (kv, n) in enumerate(zip(family, of_group)):
            for i in range(shared.shape[0]):
                for which in (0, 1):
                    kv.write_rows(i, which, prompt, own_rows[i, which, g, s, :n])
        kvs += family
    ctx.sync()
    return kvs


def prepare(case, seed):
    if case["kind"] == "select":
        shape = (case["requests"], case["n_out"])
        return {"case": case, "logits": logit_rows(case, seed), "scores": beam_scores(case, seed),
                "out": [torch.zeros(shape, device="cuda"), torch.zeros(shape, dtype=torch.int32, device="cuda"),
                        torch.zeros(shape, dtype=torch.int32, device="cuda")]}
    lens = lengths(case, seed)
    shared, own_rows = cache_rows(case, seed)
    q, k, v = new_rows(case, seed)
    state = {"case": case, "q": q, "k": k, "v": v, "out": torch.zeros_like(q)}
    if case["kind"] == "step":
        state["parents"] = parents(case, seed)
    if own:
        import wayruntime_b200 as wr
        kvs = sessions_of(case, shared, own_rows, lens)
        rows = case["prompt"] // PAGE * PAGE
        state["kvs"] = wr.Batch(kvs)
        state["lens"] = wr.Batch.u32([case["prompt"] + n for g in lens for n in g])
        state["groups"] = wr.Groups([(case["sessions"], rows)] * len(lens))
    else:
        state["shared"], state["rows"] = shared, own_rows
        state["lens"] = torch.tensor(lens, device="cuda")
        if case["kind"] == "step":
            state["at"] = torch.tensor(state["parents"], device="cuda")
    return state


# ---- the plain form

def plain_select(state):
    """Totals in 64 bits: candidates of different beams may lie within a rounding of each other."""
    logits, scores, n_out = state["logits"].double(), state["scores"].double(), state["case"]["n_out"]
    top = logits.amax(-1, keepdim=True)
    lse = top + (logits - top).exp().sum(-1, keepdim=True).log()
    total = (scores[..., None] + (logits - lse)).flatten(1)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)  # (equal ones in the order of their places)
    at = at[:, :n_out]
    return {"scores": best[:, :n_out].float(), "beams": (at // logits.shape[-1]).int(), "tokens": (at % logits.shape[-1]).int()}


def plain_attend(q, shared, rows, lens):
    """Attention of q [layers][groups][sessions][heads][dim] over the prompt's rows and each session's first lens of its own."""
    layers, groups, sessions, heads, dim = q.shape
    kv = shared.shape[-2]
    q = q.view(layers, groups, sessions, kv, heads // kv, dim)
    (pk, pv), (gk, gv) = (x.float().unbind(1) for x in (shared, rows))
    # scores over the prompt: all sessions' queries of a key head at once; then over each session's own rows
    s0 = q.permute(0, 1, 3, 2, 4, 5).flatten(3, 4) @ pk.permute(0, 1, 3, 4, 2)          # [layers][groups][kv][sessions x per][rows]
    s0 = s0.unflatten(3, (sessions, -1)).permute(0, 1, 3, 2, 4, 5)
    s1 = q @ gk.permute(0, 1, 2, 4, 5, 3)                                                # [layers][groups][sessions][kv][per][rows]
    gone = torch.arange(gk.shape[3], device=q.device) >= lens[..., None]
    s1 = s1.masked_fill(gone[None, :, :, None, None, :], -math.inf)
    s = torch.cat([s0, s1], -1) / math.sqrt(dim)
    p = (s - s.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    p0, p1 = p[..., :s0.shape[-1]], p[..., s0.shape[-1]:]
    o0 = p0.permute(0, 1, 3, 2, 4, 5).flatten(3, 4) @ pv.permute(0, 1, 3, 2, 4)
    out = o0.unflatten(3, (sessions, -1)).permute(0, 1, 3, 2, 4, 5) + p1 @ gv.permute(0, 1, 2, 4, 3, 5)
    return out.reshape(layers, groups * sessions, heads, dim)


def stored(x):
    """F32 as the cache stores it: F16 cut off behind its last bit, what is below its normal range zero."""
    x = torch.where(x.abs() < 2.0 ** -14, torch.zeros_like(x), x)
    return (x.view(torch.int32) & ~0x1FFF).view(torch.float32).half()


def plain_step(state):
    rows, lens = state["rows"], state["lens"]
    rows.copy_(rows[:, :, :, state["at"]])
    at = lens[0, 0]                                                    # (beams are of one length)
    for_all = torch.stack([stored(state["k"]), stored(state["v"])], 1)[:, :, None, :, None]
    rows.index_copy_(4, at.view(1), for_all)
    return plain_attend(state["q"][:, None], state["shared"], rows, lens + 1)


# ---- the framework's

def own_run(state):
    case, ctx = state["case"], context()
    if case["kind"] == "select":
        scores, beams, tokens = state["out"]
        ctx.beam_select(state["logits"], state["scores"], scores, beams, tokens)
        return {"scores": scores, "beams": beams, "tokens": tokens}
    kvs, lens, groups, out = state["kvs"], state["lens"], state["groups"], state["out"]
    if case["kind"] == "attend":
        ctx.attn_decode_shared(kvs, 0, lens, groups, state["q"][0], out[0], case["heads"])
        return {"out": out}
    ctx.kv_reorder(kvs, state["parents"], lens)
    q, k, v = state["q"], state["k"], state["v"]
    for i in range(case["layers"]):                  # (keys and queries come rotated)
        ctx.decode_step_shared(kvs, i, lens, groups, q[i], k[i], v[i], out[i], case["heads"], rope=False)
    return {"out": out}


def run(state):
    if own:
        return own_run(state)
    case = state["case"]
    if case["kind"] == "select":
        return plain_select(state)
    if case["kind"] == "step":
        return {"out": plain_step(state)}
    return {"out": plain_attend(state["q"].unflatten(1, (case["groups"], case["sessions"])), state["shared"], state["rows"], state["lens"])}


def work(case):
    """Bytes that have to be moved and operations that have to be done."""
    if case["kind"] == "select":
        n = case["requests"] * case["beams"]
        return {"bytes": 4 * n * (case["vocab"] + 1) + 12 * case["requests"] * case["n_out"], "flops": 3 * n * case["vocab"]}
    layers, groups, sessions = case.get("layers", 1), case.get("groups", 1), case["sessions"]
    n, gen = groups * sessions, (case["gen_lo"] + case["gen_hi"]) / 2
    row = 4 * HEAD_DIM * case["kv_heads"]                              # a token's F16 keys and values
    total = groups * case["prompt"] * row + n * gen * row + 8 * n * case["heads"] * HEAD_DIM
    if case["kind"] == "step":
        # beams that go on more than once: their own rows are read, and written for every further one; the new rows
        total += 2 * (sessions - case["kept"]) * gen * row + n * 3 * row
    return {"bytes": layers * total, "flops": layers * 4 * n * case["heads"] * HEAD_DIM * (case["prompt"] + gen)}


# ---- 64 bits

def exact_select(case, seed):
    logits, scores = logit_rows(case, seed), beam_scores(case, seed)
    got = {"scores": [], "beams": [], "tokens": []}
    for g in range(case["requests"]):
        keep = []
        for b in range(case["beams"]):
            row = logits[g, b].double()
            lp = row - torch.logsumexp(row, 0) + scores[g, b].double()
            best = torch.topk(lp, min(case["n_out"], case["vocab"]))
            keep += [(-t, b, i) for t, i in zip(best.values.tolist(), best.indices.tolist())]
        keep = sorted(keep)[:case["n_out"]]
        got["scores"].append([-t for t, _, _ in keep])
        got["beams"].append([b for _, b, _ in keep])
        got["tokens"].append([i for _, _, i in keep])
    return {"scores": torch.tensor(got["scores"], dtype=torch.float64), "beams": torch.tensor(got["beams"], dtype=torch.int32),
            "tokens": torch.tensor(got["tokens"], dtype=torch.int32)}


def exact_rows(case, seed):
    shared, rows = cache_rows(case, seed)
    q, k, v = new_rows(case, seed)
    lens, per = lengths(case, seed), case["heads"] // case["kv_heads"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    for layer in range(q.shape[0]):
        for i in range(q.shape[1]):
            g, s = divmod(i, case["sessions"])
            source = parents(case, seed)[s] if case["kind"] == "step" else s
            keys, values = (torch.cat([shared[layer, w, g], rows[layer, w, g, source, :lens[g][s]]]).double() for w in (0, 1))
            if case["kind"] == "step":
                new = [x[layer, i].double().clone() for x in (k, v)]
                for x in new:                                          # to F16, towards zero
                    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -14))) - 10)
                    x.copy_(torch.where(x.abs() < 2.0 ** -14, 0.0, torch.trunc(x / step) * step))
                keys, values = torch.cat([keys, new[0][None]]), torch.cat([values, new[1][None]])
            for h in range(case["heads"]):
                p = torch.softmax(keys[:, h // per] @ q[layer, i, h].double() * HEAD_DIM ** -0.5, 0)
                out[layer, i, h] = p @ values[:, h // per]
    return {"out": out}


def exact(case, seed):
    return exact_select(case, seed) if case["kind"] == "select" else exact_rows(case, seed)
