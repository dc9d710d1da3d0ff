"""Measured cases of the batched-serving operators (loom_b200/serve.py): the
attention of a batch that shares a long prefix, low-rank adapters of many
requests, and the verification of drafted tokens.

Every case has a plain form in elementary torch operations (32 bits, rounded
once at the end) and the same call through the framework.  Row layout shared by
all three: the rows of sequence b are seq_rows[b] .. seq_rows[b + 1] - 1 -- its
last accepted token followed by its drafted tokens.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one request behind a short system prompt: the call's latency
        dict(name="attn-1seq-f32", op="attn", type="f32", seqs=1, rows=1, heads=32, kv=4, hd=128, prefix=512, own=64),
        # the benchmark's 32-sequence decode at context 2048, three quarters of it a common prompt
        dict(name="attn-32seq-f32", op="attn", type="f32", seqs=32, rows=1, heads=32, kv=4, hd=128, prefix=1536, own=512),
        # tiny llama's heads, odd lengths, up to two drafted tokens per sequence
        dict(name="attn-13seq-f16-odd", op="attn", type="f16", seqs=13, rows=3, heads=6, kv=6, hd=48, prefix=1021, own=257),
        # speculative decoding of 64 requests behind an 8192-token prompt
        dict(name="attn-64seq-bf16-drafts", op="attn", type="bf16", seqs=64, rows=5, heads=32, kv=4, hd=128, prefix=8192, own=1024),
        # the largest: a long shared document, 128 requests
        dict(name="attn-128seq-bf16-long", op="attn", type="bf16", seqs=128, rows=2, heads=32, kv=4, hd=128, prefix=32768, own=2048),
        # one request's query projection in a decode step: latency
        dict(name="lora-1row-bf16", op="lora", type="bf16", rows=1, nin=2048, nout=4096, adapters=4, rank=16, none=False),
        # 32 requests, nearly every one with its own adapter, some without
        dict(name="lora-32row-bf16", op="lora", type="bf16", rows=32, nin=2048, nout=4096, adapters=32, rank=64, none=True),
        # tiny llama's widths, small odd ranks, f32 adapters
        dict(name="lora-77row-f32-odd", op="lora", type="f32", rows=77, nin=288, nout=769, adapters=5, rank=7, none=True),
        # a prompt batch of 2048 tokens through the output projection, eight adapters
        dict(name="lora-2048row-f16", op="lora", type="f16", rows=2048, nin=4096, nout=2048, adapters=8, rank=64, none=False),
        # one request, greedy verification of four drafts: latency
        dict(name="verify-1seq-greedy", op="verify", type="f32", seqs=1, rows=5, vocab=32000, temp=0.0, probs=False),
        # 32 requests with up to four drafts drawn from a draft model's probabilities
        dict(name="verify-32seq-probs", op="verify", type="f32", seqs=32, rows=5, vocab=151936, temp=0.8, probs=True),
        # 64 requests, up to eight drafts of a deterministic drafter, 16-bit logits, odd vocabulary
        dict(name="verify-64seq-bf16-odd", op="verify", type="bf16", seqs=64, rows=9, vocab=129281, temp=1.0, probs=False),
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))
    v = min(max(v, lo), hi)
    return v - 1 if v == 3072 else v


def draw(rng):
    op = rng.choice(["attn", "lora", "verify"])
    ty = rng.choice(["f32", "f16", "bf16"])
    if op == "attn":
        heads, kv, hd = rng.choice([(32, 4, 128), (32, 4, 128), (6, 6, 48), (16, 16, 64), (24, 8, 80), (8, 1, 192)])
        rows = _log(rng, 1, 8)
        seqs = _log(rng, 1, 128 // rows)
        # f32 contexts stay within the models' caches, 16-bit ones reach the long documents
        prefix = _log(rng, 16, 8192 if ty == "f32" else 32768)
        return dict(op=op, type=ty, seqs=seqs, rows=rows, heads=heads, kv=kv, hd=hd, prefix=prefix,
                    own=max(rows, _log(rng, 1, 2048)))
    if op == "lora":
        return dict(op=op, type=ty, rows=_log(rng, 1, 2048), nin=rng.choice([288, 512, 768, 2048, 4096, _log(rng, 64, 4096)]),
                    nout=rng.choice([288, 512, 768, 2048, _log(rng, 64, 2048)]), adapters=_log(rng, 1, 32),
                    rank=_log(rng, 1, 64), none=rng.random() < 0.5)
    rows = _log(rng, 1, 9)
    return dict(op=op, type=ty, seqs=_log(rng, 1, 64), rows=rows,
                vocab=rng.choice([32000, 102400, 129280, 151936, _log(rng, 1000, 151936)]),
                temp=rng.choice([0.0, 0.6, 1.0]), probs=rng.random() < 0.5)


def _rows_of(case):
    """Rows of each sequence: between one and case["rows"]."""
    r = random.Random(case["seqs"] * 1000 + case["rows"])
    return [case["rows"] if b == 0 else r.randint(1, case["rows"]) for b in range(case["seqs"])]


def _lens_of(case):
    """Own cache rows of each sequence, its present rows included."""
    r = random.Random(case["own"] * 131 + case["seqs"])
    return [case["own"] if b == 0 else max(n, r.randint(max(1, case["own"] // 4), case["own"]))
            for b, n in enumerate(_rows_of(case))]


def _ids_of(case):
    """Adapter of each row; decode batches mix them row by row, prompts come in runs."""
    r, n = random.Random(case["rows"] * 17 + case["adapters"]), case["adapters"]
    run = 1 if case["rows"] <= 64 else max(1, case["rows"] // (2 * n))
    ids = []
    while len(ids) < case["rows"]:
        a = r.randrange(n)
        ids += [-1 if case["none"] and r.random() < 0.2 else a] * r.randint(1, 2 * run - 1)
    return ids[: case["rows"]]


def _ranks_of(case):
    r, top = random.Random(case["rank"] * 7 + case["adapters"]), case["rank"]
    return [top if a == 0 else r.choice([top, max(1, top // 2), max(1, top // 4)]) for a in range(case["adapters"])]


def _scan(v):
    s = [0]
    for x in v:
        s.append(s[-1] + x)
    return s


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    ty = TYPES[case["type"]]

    def randn(*shape, std=1.0, dtype=ty):
        out = torch.empty(shape, dtype=dtype, device="cuda")
        step = max(1, (1 << 27) // max(1, out[0].numel()))
        for i in range(0, shape[0], step):  # bounded room for the 32-bit normals
            part = out[i : i + step]
            part.copy_(torch.randn(part.shape, generator=g, device="cuda") * std)
        return out

    s = {"case": case}
    if case["op"] == "attn":
        rows, lens = _rows_of(case), _lens_of(case)
        n, h, kv, hd = sum(rows), case["heads"], case["kv"], case["hd"]
        s["q"] = randn(n, h, hd)
        s["pk"], s["pv"] = randn(case["prefix"], kv, hd, std=1.5), randn(case["prefix"], kv, hd)
        s["ok"], s["ov"] = randn(case["seqs"], case["own"], kv, hd, std=1.5), randn(case["seqs"], case["own"], kv, hd)
        s["seq_rows"], s["seq_len"] = _ints(_scan(rows)), _ints(lens)
        s["scale"] = hd ** -0.5
        s["out"] = torch.empty_like(s["q"])
    elif case["op"] == "lora":
        n, na = case["rows"], case["adapters"]
        s["x"], s["base"] = randn(n, case["nin"], dtype=torch.float32), randn(n, case["nout"], dtype=torch.float32)
        s["a"] = randn(na, case["rank"], case["nin"], std=case["nin"] ** -0.5)
        s["b"] = randn(na, case["nout"], case["rank"], std=0.5)
        s["ranks"], s["ids"] = _ints(_ranks_of(case)), _ints(_ids_of(case))
        s["scales"] = 0.5 + torch.rand(na, generator=g, device="cuda")
        s["out"] = torch.empty_like(s["base"])
    else:
        rows, v = _rows_of(case), case["vocab"]
        n, b = sum(rows), case["seqs"]
        s["logits"] = randn(n, v, std=2.5)
        s["seq_rows"] = _ints(_scan(rows))
        s["u"] = torch.rand(n, generator=g, device="cuda")
        s["temp"] = torch.full((b,), case["temp"], device="cuda")
        # drafts: what a smaller model, near the target, draws (or takes, when greedy) for the token after each row
        heads = set(_scan(rows))
        before = [r for r in range(n) if r + 1 not in heads]
        tokens = torch.randint(0, v, (n,), generator=g, device="cuda", dtype=torch.int32)
        probs = torch.zeros((n, v), device="cuda")
        t = case["temp"] if case["temp"] > 0 else 1.0
        for r in before:
            d = (s["logits"][r].float() + 0.5 * torch.randn(v, generator=g, device="cuda")) / t
            probs[r] = torch.softmax(d, 0)
        if before:
            at = _ints(before).long()
            if case["temp"] > 0:
                pick = torch.empty((len(before), v), device="cuda").exponential_(generator=g)
                tokens[at + 1] = torch.argmax(probs[at] / pick, 1).int()
            else:
                tokens[at + 1] = torch.argmax(probs[at], 1).int()
        s["tokens"] = tokens
        s["probs"] = probs if case["probs"] else None
        s["out"] = torch.empty(n, dtype=torch.int32, device="cuda")
        s["n_out"] = torch.empty(b, dtype=torch.int32, device="cuda")
        s["logprobs"] = torch.empty(n, device="cuda")
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        from loom_b200 import serve
        if op == "attn":
            return serve.attn_shared(state["q"], state["pk"], state["pv"], state["ok"], state["ov"], state["seq_rows"],
                                     state["seq_len"], state["scale"], out=state["out"])
        if op == "lora":
            return serve.lora(state["x"], state["a"], state["b"], state["ranks"], state["scales"], state["ids"],
                              base=state["base"], out=state["out"])
        return serve.verify(state["logits"], state["tokens"], state["seq_rows"], state["u"], state["temp"],
                            draft_probs=state["probs"], out=(state["out"], state["n_out"], state["logprobs"]))
    return {"attn": _attn, "lora": _lora, "verify": _verify}[op](state)


def _attn(s):
    """softmax over the prefix and the sequence's own rows, row j of n seeing len - (n - 1 - j) of them."""
    q, rows, lens, case = s["q"].float(), s["seq_rows"].long(), s["seq_len"].long(), s["case"]
    n, kv, hd = q.shape[0], case["kv"], case["hd"]
    group, most = case["heads"] // kv, case["rows"]
    q = q.view(n, kv, group, hd) * s["scale"]
    r = torch.arange(n, device="cuda")
    seq = torch.searchsorted(rows, r, right=True) - 1
    at = r - rows[seq]
    pk, pv = s["pk"].float(), s["pv"].float()
    ok, ov = s["ok"].float(), s["ov"].float()
    # rows of a sequence side by side, so that its cache is read as one batched product
    place = seq * most + at
    qs = torch.zeros((case["seqs"] * most, kv, group, hd), device="cuda")
    qs[place] = q
    qs = qs.view(case["seqs"], most, kv, group, hd).permute(0, 2, 1, 3, 4).reshape(case["seqs"], kv, most * group, hd)
    so = torch.matmul(qs, ok.permute(0, 2, 3, 1)).view(case["seqs"], kv, most, group, -1)
    so = so.permute(0, 2, 1, 3, 4).reshape(case["seqs"] * most, kv, group, -1)[place]
    seen = lens[seq] - (rows[seq + 1] - 1 - r)
    so = so.masked_fill(torch.arange(so.shape[-1], device="cuda") >= seen[:, None, None, None], float("-inf"))
    sp = torch.matmul(q.permute(1, 0, 2, 3).reshape(kv, n * group, hd), pk.permute(1, 2, 0))
    sp = sp.view(kv, n, group, -1).permute(1, 0, 2, 3)
    top = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    ep, eo = torch.exp(sp - top), torch.exp(so - top)
    del sp, so
    total = ep.sum(-1, keepdim=True) + eo.sum(-1, keepdim=True)
    out = torch.matmul(ep.permute(1, 0, 2, 3).reshape(kv, n * group, -1), pv.permute(1, 0, 2))
    out = out.view(kv, n, group, hd).permute(1, 0, 2, 3)
    es = torch.zeros((case["seqs"] * most, kv, group, eo.shape[-1]), device="cuda")
    es[place] = eo
    es = es.view(case["seqs"], most, kv, group, -1).permute(0, 2, 1, 3, 4).reshape(case["seqs"], kv, most * group, -1)
    oo = torch.matmul(es, ov.permute(0, 2, 1, 3)).view(case["seqs"], kv, most, group, hd)
    out = out + oo.permute(0, 2, 1, 3, 4).reshape(case["seqs"] * most, kv, group, hd)[place]
    return (out / total).reshape(n, case["heads"], hd).to(s["q"].dtype)


def _lora(s):
    """base + scale_a B_a (A_a x) with every adapter applied and all but the row's own masked away."""
    case = s["case"]
    n, na, rank = case["rows"], case["adapters"], case["rank"]
    t = torch.matmul(s["x"], s["a"].float().view(na * rank, -1).t()).view(n, na, rank)
    mine = s["ids"][:, None] == torch.arange(na, device="cuda")
    t = t * (mine * s["scales"])[:, :, None] * (torch.arange(rank, device="cuda") < s["ranks"][:, None])
    return s["base"] + torch.matmul(t.view(n, na * rank), s["b"].float().permute(0, 2, 1).reshape(na * rank, -1))


def _verify(s):
    """Accept drafts in order while u q < p; then one token from max(p - q, 0), or from p after the last draft.
    The sums that pick a token are 64 bits wide: at 32 their rounding, not u, would choose among near neighbours."""
    lg, rows, tok, u = s["logits"].float(), s["seq_rows"].long(), s["tokens"].long(), s["u"]
    n, v = lg.shape
    b = rows.numel() - 1
    r = torch.arange(n, device="cuda")
    seq = torch.searchsorted(rows, r, right=True) - 1
    last = rows[seq + 1] - 1 == r
    temp = s["temp"][seq]
    greedy = temp <= 0
    inv = 1.0 / torch.where(greedy, torch.ones_like(temp), temp)
    top, arg = lg.amax(1), torch.argmax(lg, 1)
    e = torch.exp((lg - top[:, None]) * inv[:, None])
    z = e.sum(1, dtype=torch.float64).float()
    nxt = torch.where(last, torch.zeros_like(tok), torch.cat([tok[1:], tok[:1]]))
    p = e.gather(1, nxt[:, None])[:, 0] / z
    qn = torch.ones_like(p) if s["probs"] is None else s["probs"].gather(1, nxt[:, None])[:, 0]
    ok = torch.where(greedy, nxt == arg, u * qn < p) & ~last
    # accepted: drafts before the first refusal of the sequence
    bad = torch.where(ok, n, r)
    stop = torch.full((b,), n, device="cuda", dtype=torch.int64).scatter_reduce(0, seq, bad, "amin")
    # the token after them, from row `stop`
    es, zs, full = e[stop], z[stop], last[stop]
    if s["probs"] is not None:
        w = torch.where(full[:, None], es, torch.clamp(es / zs[:, None] - s["probs"][stop], min=0.0))
    else:
        hit = (torch.arange(v, device="cuda") == nxt[stop][:, None]) & ~full[:, None]
        w = torch.where(hit, torch.zeros_like(es), es)
    w = torch.where(w.sum(1, keepdim=True) > 0, w, es)
    cum = w.cumsum(1, dtype=torch.float64)
    want = u[rows[1:] - 1].double() * cum[:, -1]
    drawn = torch.argmax((cum > want[:, None]).int(), 1)
    final = torch.where(greedy[stop], arg[stop], drawn)
    there = torch.where(r == stop[seq], final[seq], nxt)
    emit = r <= stop[seq]
    lp = (lg.gather(1, there[:, None])[:, 0] - top) * inv - torch.log(z)
    return (torch.where(emit, there, -1).int(), (stop - rows[:-1] + 1).int(),
            torch.where(emit, lp, torch.zeros_like(lp)))


def work(case):
    size = torch.empty((), dtype=TYPES[case["type"]]).element_size()
    if case["op"] == "attn":
        rows, lens = _rows_of(case), _lens_of(case)
        wide, cells = case["kv"] * case["hd"], 0
        for n, m in zip(rows, lens):
            cells += sum(case["prefix"] + m - (n - 1 - j) for j in range(n))
        by = size * (2 * sum(rows) * case["heads"] * case["hd"] + 2 * wide * (case["prefix"] + sum(lens)))
        return {"bytes": by + 8 * case["seqs"], "flops": 4 * case["heads"] * case["hd"] * cells}
    if case["op"] == "lora":
        ids, ranks = _ids_of(case), _ranks_of(case)
        wide = case["nin"] + case["nout"]
        by = 4 * case["rows"] * (wide + case["nout"] + 1) + size * wide * sum(ranks[a] for a in set(ids) if a >= 0)
        return {"bytes": by, "flops": 2 * wide * sum(ranks[a] for a in ids if a >= 0)}
    rows = sum(_rows_of(case))
    by = rows * case["vocab"] * size + 16 * rows
    if case["probs"] and case["temp"] > 0:  # of the drafter's rows, the one at the refusal
        by += 4 * case["vocab"] * min(case["seqs"], rows - case["seqs"])
    return {"bytes": by, "flops": 4 * rows * case["vocab"]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "lora": _exact_lora, "verify": _exact_verify}[case["op"]](case, s)


def _exact_attn(case, s):
    if 4 * case["heads"] * case["hd"] * sum(_rows_of(case)) * (case["prefix"] + case["own"]) > 1 << 40:
        return None
    group, out = case["heads"] // case["kv"], []
    at = 0
    for b, (n, m) in enumerate(zip(_rows_of(case), _lens_of(case))):
        k = torch.cat([s["pk"], s["ok"][b, :m]]).double()
        v = torch.cat([s["pv"], s["ov"][b, :m]]).double()
        q = s["q"][at : at + n].double()
        at += n
        x = torch.einsum("nhd,phd->nhp", q, k.repeat_interleave(group, 1)) * s["scale"]
        see = case["prefix"] + m - torch.arange(n - 1, -1, -1, device="cuda")
        x = x.masked_fill(torch.arange(k.shape[0], device="cuda") >= see[:, None, None], float("-inf"))
        out.append(torch.einsum("nhp,phd->nhd", torch.softmax(x, -1), v.repeat_interleave(group, 1)))
    return torch.cat(out)


def _exact_lora(case, s):
    out, ids = s["base"].double(), torch.tensor(_ids_of(case), device="cuda")
    for a, rank in enumerate(_ranks_of(case)):
        mine = torch.nonzero(ids == a)[:, 0]
        t = s["x"][mine].double() @ s["a"][a, :rank].double().t()
        out[mine] += s["scales"][a].double() * (t @ s["b"][a, :, :rank].double().t())
    return out


def _exact_verify(case, s):
    """The log-probabilities alone have a 64-bit value; the choices are whole numbers. They follow the same rule here,
    in 64 bits, to know which tokens' values to give."""
    rows, at, lps = _rows_of(case), 0, []
    for n in rows:
        x = s["logits"][at : at + n].double()
        lp = torch.log_softmax(x / case["temp"] if case["temp"] > 0 else x, 1)
        got = []
        for j in range(n):
            left = None
            if j < n - 1:
                d, u = int(s["tokens"][at + j + 1]), float(s["u"][at + j])
                q = s["probs"][at + j].double() if s["probs"] is not None else None
                if int(x[j].argmax()) == d if case["temp"] <= 0 else u * (1.0 if q is None else float(q[d])) < float(lp[j, d].exp()):
                    got.append(lp[j, d])
                    continue
                left = lp[j].exp()
                if q is None:
                    left[d] = 0
                else:
                    left = (left - q).clamp(min=0)
            w = lp[j].exp() if left is None or float(left.sum()) <= 0 else left
            c = w.cumsum(0)
            t = int(x[j].argmax()) if case["temp"] <= 0 else int(torch.searchsorted(c, c[-1] * float(s["u"][at + n - 1]), right=True))
            got.append(lp[j, min(t, case["vocab"] - 1)])
            break
        lps += got + [torch.zeros((), dtype=torch.float64, device="cuda")] * (n - len(got))
        at += n
    return (None, None, torch.stack(lps))
