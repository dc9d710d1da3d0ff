"""GPU tests of the batched-serving operators (loom_b200/serve.py) against plain
64-bit implementations.

Tolerances (relative L2 of an output), fixed before the first run:
  16-bit attention: the weights and the output are each rounded once to the
    type, unit roundoff u = 2^-11 (f16) or 2^-8 (bf16): 2 u;
  f32 attention: a score is a sum of up to 256 products of magnitude about 1,
    its error about sqrt(256) 2^-24 times a few: 2e-5;
  adapters: f32 sums over up to 4096 products, sqrt(4096) 2^-24 = 4e-6: 2e-5
    (A and B are exact in f32, whatever their type);
  log-probabilities: 2e-5 absolute plus 2e-6 of the value.
Tokens are whole numbers and must be equal, unless the 64-bit rule itself is
decided by less than the 32-bit weights resolve (1e-5 of the whole)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ATTN_TOL = {F32: 2e-5, F16: 2 * 2.0 ** -11, BF16: 2 * 2.0 ** -8}
TYPES = [F32, F16, BF16]


@pytest.fixture(scope="module")
def sv(be):
    from loom_b200 import serve
    return serve


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def ints(v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def scan(v):
    return np.concatenate([[0], np.cumsum(v)]).astype(int)


def rel(got, want):
    got, want = got.double(), want.double()
    return float((got - want).norm() / want.norm().clamp(min=1e-30))


# ---- attention ---------------------------------------------------------------

def attn_inputs(ty, rows, lens, heads, kv, hd, prefix, cap, seed=0, qstd=1.0):
    g, n, s = gen(seed), sum(rows), len(rows)
    r = lambda *sh: torch.randn(sh, generator=g, device="cuda")  # noqa: E731
    return dict(q=(r(n, heads, hd) * qstd).to(ty), pk=r(prefix, kv, hd).to(ty), pv=r(prefix, kv, hd).to(ty),
                ok=r(s, cap, kv, hd).to(ty), ov=r(s, cap, kv, hd).to(ty), seq_rows=ints(scan(rows)), seq_len=ints(lens),
                scale=1.0 / math.sqrt(hd))


def attn_ref(i, rows, lens):
    """Row by row in 64 bits, over the positions the row sees and no others."""
    out, at = torch.zeros(i["q"].shape, dtype=torch.float64, device="cuda"), 0
    group = i["q"].shape[1] // i["pk"].shape[1]
    for b, n in enumerate(rows):
        for j in range(n):
            see = max(0, min(lens[b], i["ok"].shape[1]) - (n - 1 - j))
            k = torch.cat([i["pk"], i["ok"][b, :see]]).double().repeat_interleave(group, 1)
            v = torch.cat([i["pv"], i["ov"][b, :see]]).double().repeat_interleave(group, 1)
            if k.shape[0]:
                s = torch.einsum("hd,phd->hp", i["q"][at].double(), k) * i["scale"]
                out[at] = torch.einsum("hp,phd->hd", torch.softmax(s, -1), v)
            at += 1
    return out


def attn(sv, i, **kw):
    return sv.attn_shared(i["q"], i["pk"], i["pv"], i["ok"], i["ov"], i["seq_rows"], i["seq_len"], i["scale"], **kw)


SHAPES = {
    "one row": ([1], [1], 32, 4, 128, 300, 8),
    "prefix only": ([1, 2], [0, 0], 8, 2, 64, 77, 0),
    "own only": ([1, 3, 2], [5, 70, 129], 8, 2, 64, 0, 130),
    "one position": ([1], [0], 4, 4, 32, 1, 4),
    "tile edges": ([1, 1, 1, 1], [63, 64, 65, 128], 32, 4, 128, 128, 128),
    "ragged drafts": ([5, 1, 3, 8, 2], [9, 1, 300, 8, 77], 32, 4, 128, 515, 300),
    "rows of none": ([2, 0, 1, 0], [10, 4, 3, 0], 8, 8, 48, 33, 16),
    "tiny heads": ([3] * 7, [17, 3, 40, 8, 100, 64, 65], 6, 6, 48, 101, 101),
    "odd head dim": ([2, 3], [20, 31], 6, 2, 33, 50, 40),
    "hd 1": ([2], [3], 2, 1, 1, 5, 4),
    "group of 3, hd 80": ([2, 4, 1], [90, 4, 33], 24, 8, 80, 200, 96),
    "one kv head, hd 192": ([4, 4], [64, 200], 8, 1, 192, 260, 200),
    "hd 256": ([2, 2], [64, 20], 16, 4, 256, 130, 70),
    "many rows": ([4] * 33, list(range(4, 37)), 32, 4, 128, 700, 40),
    "wide group": ([3, 3], [30, 50], 48, 1, 64, 140, 64),
    "long prefix": ([1, 2], [10, 60], 8, 1, 128, 20011, 64),
    "long own": ([2], [9001], 8, 2, 128, 3, 9001),
    "more rows than own": ([6, 20], [3, 15], 8, 2, 64, 9, 16),
}


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=[s.replace(" ", "_") for s in SHAPES])
def test_attn_matches_64_bits(sv, ty, shape):
    rows, lens, heads, kv, hd, prefix, cap = SHAPES[shape]
    i = attn_inputs(ty, rows, lens, heads, kv, hd, prefix, cap, seed=len(shape))
    out = torch.full_like(i["q"], float("nan"))
    assert attn(sv, i, out=out) is out
    assert rel(out, attn_ref(i, rows, lens)) < ATTN_TOL[ty]


# rows and prefix enough for the prefix's own kernel (16-bit types): its tiles of 128
# rows and steps of 64 positions with edges everywhere
PREFIXES = {
    "a quarter of a tile": ([1, 3], [0, 5], 32, 4, 128, 16411, 8),
    "a tile and a row, hd 80": ([40, 2, 1], [60, 2, 9], 24, 8, 80, 3301, 60),
    "group of one, hd 48": ([100, 0, 200], [120, 0, 200], 8, 8, 48, 2401, 200),
    "one kv head": ([5] * 10, [9] * 10, 16, 1, 64, 5301, 16),
    "two tiles of a CTA": ([4] * 33, list(range(33)), 32, 4, 128, 4099, 40),
    "hd 8": ([3, 5], [0, 2], 64, 1, 8, 65601, 4),
}


@pytest.mark.parametrize("ty", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", PREFIXES, ids=[s.replace(" ", "_") for s in PREFIXES])
def test_attn_prefix_of_many_rows(sv, ty, shape):
    rows, lens, heads, kv, hd, prefix, cap = PREFIXES[shape]
    for qstd in (1.0, 20.0):  # and scores of +-60
        i = attn_inputs(ty, rows, lens, heads, kv, hd, prefix, cap, seed=len(shape), qstd=qstd)
        tol = ATTN_TOL[ty] + (10 * ATTN_TOL[F32] if qstd > 1 else 0)
        want = attn_ref(i, rows, lens)
        assert rel(attn(sv, i), want) < tol
        for k in ("pk", "pv"):  # head-major
            i[k] = i[k].transpose(0, 1).contiguous().transpose(0, 1)
        assert rel(attn(sv, i), want) < tol
    i["pv"][prefix - 1, :, 0] = float("nan")  # a value that every row sees
    assert torch.isnan(attn(sv, i)[..., 0]).all()


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "f16", "bf16"])
def test_attn_peaked_scores(sv, ty):
    """Scores of +-60: one position has almost all of the weight, exp must not overflow."""
    rows, lens = [2, 1, 4], [40, 90, 4]
    i = attn_inputs(ty, rows, lens, 32, 4, 128, 600, 96, seed=5, qstd=20.0)
    # a score's error grows with it: the operands' products are exact, their sum is rounded
    assert rel(attn(sv, i), attn_ref(i, rows, lens)) < 10 * ATTN_TOL[F32] + ATTN_TOL[ty]


def test_attn_row_that_sees_nothing_is_zero(sv):
    for ty in TYPES:
        i = attn_inputs(ty, [3, 1], [1, 0], 32, 4, 128, 0, 8)
        out = attn(sv, i, out=torch.full_like(i["q"], 7.0))
        assert torch.equal(out[:2], torch.zeros_like(out[:2])) and torch.equal(out[3:], torch.zeros_like(out[3:]))
        assert rel(out[2:3], attn_ref(i, [3, 1], [1, 0])[2:3]) < ATTN_TOL[ty]


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("ty", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [128, 33])
def test_attn_does_not_touch_what_a_row_may_not_see(sv, ty, bad, hd):
    """Cache rows past a sequence's length, and drafts after a row, hold anything."""
    rows, lens = [4, 1, 3], [70, 20, 33]
    i = attn_inputs(ty, rows, lens, 8, 2, hd, 90, 80, seed=9)
    want = attn_ref(i, rows, lens)
    for b, m in enumerate(lens):
        i["ok"][b, m:] = bad
        i["ov"][b, m:] = bad
    i["ok"][0, 69] = bad  # the last draft of sequence 0: only its last row sees it
    i["ov"][0, 69] = bad
    out = attn(sv, i)
    keep = [0, 1, 2, 4, 5, 6, 7]
    assert rel(out[keep], want[keep]) < ATTN_TOL[ty]
    assert not torch.isfinite(out[3]).all() or bad == float("-inf")


def test_attn_nan_that_is_seen_is_not_hidden(sv):
    for ty in TYPES:
        i = attn_inputs(ty, [1], [40], 8, 2, 128, 60, 64)
        i["pk"][7] = float("nan")
        assert torch.isnan(attn(sv, i)).all()


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "f16", "bf16"])
def test_attn_layouts(sv, ty):
    """Head-major caches, padded rows, a base off 16-byte alignment, spaced rows of q and out."""
    rows, lens = [2, 1, 3], [40, 65, 9]
    i = attn_inputs(ty, rows, lens, 8, 2, 64, 150, 72, seed=3)
    want = attn_ref(i, rows, lens)

    def head_major(t):
        return t.transpose(-3, -2).contiguous().transpose(-3, -2)

    def shifted(t, pad, off):
        flat = torch.zeros(t.numel() // t.shape[-1] * (t.shape[-1] + pad) + off, dtype=t.dtype, device="cuda")
        view = flat[off:].view(*t.shape[:-1], t.shape[-1] + pad)[..., : t.shape[-1]]
        view.copy_(t)
        return view

    for f in (head_major, lambda t: shifted(t, 8, 0), lambda t: shifted(t, 3, 0), lambda t: shifted(t, 0, 1)):
        j = dict(i, **{k: f(i[k]) for k in ("pk", "pv", "ok", "ov")})
        assert rel(attn(sv, j), want) < ATTN_TOL[ty]
    for width, off in ((9, 0), (8, 1), (11, 3)):
        buf = torch.zeros(i["q"].shape[0] * 64 * width + off, dtype=ty, device="cuda")
        qs = buf[off:].view(-1, width * 64)[:, : 8 * 64].view(-1, 8, 64)
        qs.copy_(i["q"])
        dst = torch.zeros_like(buf)[off:].view(-1, width * 64)[:, : 8 * 64].view(-1, 8, 64)
        assert rel(attn(sv, dict(i, q=qs), out=dst), want) < ATTN_TOL[ty]


def test_attn_cache_beyond_32_bit_offsets(sv):
    """An own cache of more than 2^31 elements; the last sequence lies past them."""
    seqs, cap, kv, hd = 5, 1 << 20, 4, 128
    k = torch.empty((seqs, cap, kv, hd), dtype=F16, device="cuda")
    v = torch.empty_like(k)
    rows, lens = [1] * seqs, [0, 0, 0, 0, 300]
    i = attn_inputs(F16, rows, [0] * seqs, 8, kv, hd, 40, 1)
    g = gen(4)
    k[4, :300].copy_(torch.randn((300, kv, hd), generator=g, device="cuda"))
    v[4, :300].copy_(torch.randn((300, kv, hd), generator=g, device="cuda"))
    i.update(ok=k, ov=v, seq_len=ints(lens))
    assert rel(attn(sv, i), attn_ref(i, rows, lens)) < ATTN_TOL[F16]
    # and its end: the sequence's last 300 positions of a full cache would take 2^20 reads of the test
    i.update(ok=k[:, -300:], ov=v[:, -300:])
    i["ok"][4].copy_(torch.randn((300, kv, hd), generator=g, device="cuda"))
    i["ov"][4].copy_(torch.randn((300, kv, hd), generator=g, device="cuda"))
    assert rel(attn(sv, i), attn_ref(i, rows, lens)) < ATTN_TOL[F16]


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "f16", "bf16"])
def test_attn_repeats_bit_for_bit_on_streams_and_in_graphs(sv, ty):
    rows, lens = [3, 1, 2] * 5, [50, 300, 129] * 5
    i = attn_inputs(ty, rows, lens, 32, 4, 128, 1000, 320, seed=8)
    want = attn(sv, i).clone()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        a = attn(sv, i)
    b = attn(sv, i, stream=st.cuda_stream)
    st.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want)
    out = torch.zeros_like(i["q"])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        attn(sv, i, out=out)
    i["seq_len"].fill_(49)  # lengths are read by the kernels: a graph follows them
    g.replay()
    torch.cuda.synchronize()
    assert rel(out, attn_ref(i, rows, [49] * 15)) < ATTN_TOL[ty]


def test_attn_refusals(sv):
    from loom_b200 import LoomCudaError
    i = attn_inputs(F32, [1, 2], [3, 4], 8, 2, 64, 10, 8)

    def bad(**kw):
        with pytest.raises(LoomCudaError):
            attn(sv, dict(i, **kw))

    bad(q=i["q"].double())
    bad(q=i["q"].cpu())
    bad(q=i["q"].half())
    bad(pk=i["pk"][:, :, :32])
    bad(pv=i["pv"][1:])
    bad(ov=i["ov"][:1])
    bad(pk=i["pk"].transpose(0, 1).contiguous().transpose(0, 1))  # keys laid out unlike the values
    bad(seq_rows=i["seq_rows"].long())
    bad(seq_rows=i["seq_rows"][:2])
    bad(seq_len=i["seq_len"].cpu())
    bad(q=torch.zeros((3, 7, 64), device="cuda"))  # 7 heads over 2
    bad(scale=float("nan"))
    big = attn_inputs(F32, [1], [1], 2, 1, 257, 4, 4)
    with pytest.raises(LoomCudaError, match="head_dim"):
        attn(sv, big)
    assert attn(sv, dict(i, q=i["q"][:0], seq_rows=ints([0, 0, 0]))).shape[0] == 0


# ---- adapters ------------------------------------------------------------------

def lora_inputs(ty, n, nin, nout, ranks, ids, rank=None, seed=0):
    g, na = gen(seed), len(ranks)
    rank = max(ranks, default=0) if rank is None else rank
    r = lambda *sh: torch.randn(sh, generator=g, device="cuda")  # noqa: E731
    return dict(x=r(n, nin), a=(r(na, rank, nin) / math.sqrt(nin)).to(ty), b=r(na, nout, rank).to(ty), ranks=ints(ranks),
                scales=r(na), ids=ints(ids), base=r(n, nout))


def lora_ref(i):
    out = i["base"].double() if i["base"] is not None else 0
    rows = []
    for r, a in enumerate(i["ids"].tolist()):
        d = torch.zeros(i["b"].shape[1], dtype=torch.float64, device="cuda")
        if 0 <= a < i["a"].shape[0]:
            k = max(0, min(int(i["ranks"][a]), i["a"].shape[1]))
            d = i["scales"][a].double() * (i["b"][a, :, :k].double() @ (i["a"][a, :k].double() @ i["x"][r].double()))
        rows.append(d)
    return out + torch.stack(rows)


def lora(sv, i, **kw):
    return sv.lora(i["x"], i["a"], i["b"], i["ranks"], i["scales"], i["ids"], base=i["base"], **kw)


LORA = {
    "one row": (1, 256, 512, [16], [0]),
    "one by one": (1, 1, 1, [1], [0]),
    "no adapter at all": (5, 64, 96, [], [-1, 0, 3, -7, 2]),
    "none and out of range": (6, 288, 288, [8, 4], [-1, 0, 2, 1, 99, 0]),
    "ranks 0 to 64": (9, 512, 384, [0, 1, 7, 16, 33, 64], [0, 1, 2, 3, 4, 5, 5, 0, 3]),
    "odd widths": (17, 129, 77, [5, 3], [0, 1] * 8 + [1]),
    "one adapter": (200, 288, 768, [12], [0] * 200),
    "runs": (333, 512, 640, [64, 32, 8], [0] * 100 + [2] * 33 + [1] * 150 + [-1] * 20 + [0] * 30),
    "scattered": (150, 2048, 256, [16, 8, 4, 16], [(7 * r * r + r) % 5 for r in range(150)]),
    "wide": (40, 4096, 2048, [128, 100], [r % 2 for r in range(40)]),
    "rank 300": (20, 300, 200, [300, 257], [r % 2 for r in range(20)]),
    "many adapters": (64, 128, 128, [4] * 500, [(r * 37) % 500 for r in range(64)]),
    "prompt": (2000, 256, 264, [16, 16], [r // 1100 for r in range(2000)]),
    "many parts": (39, 4096, 200, [67, 2, 65], [0] * 20 + [2] * 10 + [1] * 9),
    "rows of two blocks, rank 66": (130, 640, 130, [66, 1], [0] * 100 + [1] * 30),
}


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", LORA, ids=[s.replace(" ", "_") for s in LORA])
def test_lora_matches_64_bits(sv, ty, shape):
    n, nin, nout, ranks, ids = LORA[shape]
    i = lora_inputs(ty, n, nin, nout, ranks, ids, seed=n)
    out = torch.full_like(i["base"], float("nan"))
    assert lora(sv, i, out=out) is out
    want = lora_ref(i)
    assert rel(out, want) < 2e-5
    keep = [r for r, a in enumerate(ids) if not 0 <= a < len(ranks)]
    assert torch.equal(out[keep], i["base"][keep])
    nobase = lora(sv, dict(i, base=None))
    assert rel(nobase, want - i["base"].double()) < 2e-5


def test_lora_in_place_unread_padding_and_layouts(sv):
    for ty in TYPES:
        i = lora_inputs(ty, 23, 200, 136, [3, 8, 5], [r % 4 - 1 for r in range(23)], rank=11, seed=2)
        want = lora_ref(i)
        for a, k in enumerate([3, 8, 5]):  # what lies past an adapter's rank is not read
            i["a"][a, k:] = float("nan")
            i["b"][a, :, k:] = float("nan")
        x = i["x"].clone()
        i["x"][0] = float("nan")  # a row without an adapter reads no x
        out = lora(sv, i)
        assert torch.equal(out[0], i["base"][0])
        i["x"] = x
        assert rel(lora(sv, i), want) < 2e-5

        def spaced(t, pad, off):
            flat = torch.zeros(t.numel() // t.shape[-1] * (t.shape[-1] + pad) + off, dtype=t.dtype, device="cuda")
            v = flat[off:].view(*t.shape[:-1], t.shape[-1] + pad)[..., : t.shape[-1]]
            v.copy_(t)
            return v

        for pad, off in ((1, 0), (0, 1), (5, 3), (8, 0)):
            j = dict(i, **{k: spaced(i[k], pad, off) for k in ("x", "a", "b", "base")})
            assert rel(lora(sv, j, out=spaced(i["base"], pad, off)), want) < 2e-5
        base = i["base"].clone()
        assert lora(sv, dict(i, base=base), out=base) is base
        assert rel(base, want) < 2e-5


def test_lora_repeats_on_streams_and_in_graphs(sv):
    i = lora_inputs(BF16, 70, 512, 512, [16, 8, 32], [r % 4 - 1 for r in range(70)], seed=6)
    want = lora(sv, i)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    got = lora(sv, i, stream=st.cuda_stream)
    st.synchronize()
    assert torch.equal(got, want)
    out, g = torch.zeros_like(want), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lora(sv, i, out=out)
    i["ids"].copy_(ints([(r // 9) % 3 for r in range(70)]))
    g.replay()
    torch.cuda.synchronize()
    assert rel(out, lora_ref(i)) < 2e-5


def test_lora_refusals(sv):
    from loom_b200 import LoomCudaError
    i = lora_inputs(F16, 4, 64, 32, [8, 8], [0, 1, 0, -1])
    for kw in (dict(x=i["x"].half()), dict(x=i["x"][:, :32]), dict(a=i["a"].double()), dict(b=i["b"].float()),
               dict(b=i["b"][:, :, :4]), dict(ranks=i["ranks"].long()), dict(ids=i["ids"][:3]), dict(ids=i["ids"].cpu()),
               dict(scales=i["scales"].half()), dict(base=i["base"][:, :16]), dict(x=i["x"].t().contiguous().t())):
        with pytest.raises(LoomCudaError):
            lora(sv, dict(i, **kw))
    with pytest.raises(LoomCudaError):
        lora(sv, i, out=torch.zeros((4, 32), device="cuda", dtype=F16))
    assert lora(sv, dict(i, x=i["x"][:0], ids=i["ids"][:0], base=i["base"][:0])).shape == (0, 32)


# ---- verification ----------------------------------------------------------------

def verify_inputs(ty, rows, vocab, temps, probs, seed=0, std=2.5, noise=0.5):
    g, n = gen(seed), sum(rows)
    logits = (torch.randn((n, vocab), generator=g, device="cuda") * std).to(ty)
    seq = np.repeat(np.arange(len(rows)), rows)
    t = torch.tensor([temps[b] if temps[b] > 0 else 1.0 for b in seq], device="cuda", dtype=torch.float32)[:, None]
    q = torch.softmax((logits.float() + noise * torch.randn((n, vocab), generator=g, device="cuda")) / t, 1)
    tokens = torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    drawn = torch.argmax(q / torch.empty_like(q).exponential_(generator=g), 1).int()
    tokens[1:] = drawn[:-1]
    return dict(logits=logits, tokens=tokens, seq_rows=ints(scan(rows)), u=torch.rand(n, generator=g, device="cuda"),
                temperature=torch.tensor(temps, device="cuda", dtype=torch.float32), draft_probs=q if probs else None)


def verify_ref(i, rows):
    """The rule in 64 bits: tokens, counts, log-probabilities, and how narrowly each sequence was decided."""
    x = np.asarray(i["logits"].double().cpu())
    q = None if i["draft_probs"] is None else np.asarray(i["draft_probs"].double().cpu())
    tok, u, temps = i["tokens"].cpu().numpy(), i["u"].double().cpu().numpy(), i["temperature"].double().cpu().numpy()
    n, v = x.shape
    out, cnt, lps, margin, at = -np.ones(n, int), [], np.zeros(n), [], 0
    for b, m in enumerate(rows):
        t, close, stop = temps[b], 1.0, at
        if not m:
            cnt.append(0)
            margin.append(1.0)
            continue

        def dist(r):
            l = np.where(np.isnan(x[r]), -np.inf, x[r])
            top = l.max()
            with np.errstate(invalid="ignore"):
                e = np.where(l == top, 1.0, np.exp((l - top) / (t if t > 0 else 1.0))) if top > -np.inf else np.zeros(v)
            arg = int(l.argmax()) if top > -np.inf else 0
            return e / max(e.sum(), 1e-300), arg
        while stop < at + m - 1:
            (p, arg), d = dist(stop), tok[stop + 1]
            if not 0 <= d < v:
                break
            if t <= 0:
                ok = d == arg
            else:
                lhs = u[stop] * (1.0 if q is None else q[stop, d])
                close = min(close, abs(lhs - p[d]) / max(p[d], 1e-30))
                ok = lhs < p[d]
            if not ok:
                break
            out[stop], lps[stop] = d, math.log(p[d])
            stop += 1
        p, arg = dist(stop)
        if t <= 0:
            pick = arg
        else:
            w = p.copy()
            if stop < at + m - 1:
                d = tok[stop + 1]
                if q is not None:
                    w = np.maximum(p - q[stop], 0)
                elif 0 <= d < v:
                    w[d] = 0
                if w.sum() <= 0:
                    w = p
            c = w.cumsum()
            want = u[at + m - 1] * c[-1]
            over = np.nonzero(c > want)[0]
            pick = int(over[0]) if len(over) else 0
            if c[-1] > 0:
                close = min(close, np.abs(c - want)[max(0, pick - 1): pick + 1].min() / c[-1])
        out[stop] = pick
        lps[stop] = math.log(p[pick]) if p[pick] > 0 else -np.inf
        cnt.append(stop - at + 1)
        margin.append(close)
        at += m
    return out, np.array(cnt), lps, np.array(margin)


def check_verify(sv, i, rows):
    n = i["logits"].shape[0]
    out = (torch.full((n,), 12345, dtype=torch.int32, device="cuda"),
           torch.full((len(rows),), 99, dtype=torch.int32, device="cuda"), torch.full((n,), float("nan"), device="cuda"))
    sv.verify(i["logits"], i["tokens"], i["seq_rows"], i["u"], i["temperature"], i["draft_probs"], out=out)
    tok, cnt, lp = (t.cpu().numpy() for t in out)
    wt, wc, wl, margin = verify_ref(i, rows)
    at, loose = 0, 0
    for b, m in enumerate(rows):
        sl = slice(at, at + m)
        at += m
        if (tok[sl] != wt[sl]).any() or cnt[b] != wc[b]:
            assert margin[b] < 1e-5, (b, tok[sl], wt[sl], margin[b])
            loose += 1
            continue
        both = np.isfinite(wl[sl])
        assert (np.isfinite(lp[sl]) == both).all()
        assert (np.abs(lp[sl] - wl[sl])[both] <= 2e-5 + 2e-6 * np.abs(wl[sl][both])).all()
    assert loose <= max(1, len(rows) // 50)
    return tok, cnt, lp


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("probs", [True, False], ids=["probs", "sure"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 1000, 1023, 32000, 151937])
def test_verify_matches_64_bits(sv, ty, probs, vocab):
    rows = [5, 1, 3, 9, 2, 4, 1, 6]
    temps = [0.8, 1.0, 0.0, 0.6, 1.5, -1.0, 0.0, 1.0]
    i = verify_inputs(ty, rows, vocab, temps, probs, seed=vocab)
    tok, cnt, _ = check_verify(sv, i, rows)
    assert (cnt >= 1).all() and (cnt <= rows).all()
    if vocab == 1000 and probs:
        assert len(set(cnt.tolist())) > 1


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [[2, 1], [3] * 12], ids=["few", "many"])
def test_verify_beyond_the_registers_of_a_cluster(sv, ty, rows):
    """A vocabulary longer than a cluster keeps, in one launch and in two passes, with and without probabilities."""
    for probs in (True, False):
        check_verify(sv, verify_inputs(ty, rows, 400001, [[0.9, 0.0, 1.0][b % 3] for b in range(len(rows))], probs, seed=3,
                                       std=3.0), rows)


def test_verify_many_sequences(sv):
    rows = [1 + (b * 7) % 4 for b in range(300)]
    i = verify_inputs(F32, rows, 513, [[1.0, 0.7, 0.0][b % 3] for b in range(300)], True, seed=1)
    _, cnt, _ = check_verify(sv, i, rows)
    assert (cnt > 1).sum() > 20 and (cnt < rows).sum() > 20


def test_verify_sequences_without_rows(sv):
    rows = [0, 2, 0, 0, 3, 0]
    check_verify(sv, verify_inputs(F32, rows, 100, [1.0] * 6, True), rows)
    i = verify_inputs(F32, [1], 10, [1.0], False)
    cnt = torch.full((3,), 5, dtype=torch.int32, device="cuda")
    e = i["u"][:0]
    sv.verify(i["logits"][:0], i["tokens"][:0], ints([0, 0, 0, 0]), e, None, out=(i["tokens"][:0], cnt, e.clone()))
    assert cnt.tolist() == [0, 0, 0]


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "f16", "bf16"])
def test_verify_masked_logits(sv, ty):
    """Vocabularies masked by -inf and by the type's lowest value, NaN, +inf, a row with nothing left."""
    rows = [3, 3, 3, 3, 2]
    i = verify_inputs(ty, rows, 700, [1.0, 0.0, 0.9, 1.0, 1.0], False, seed=3)
    i["logits"][0:3, 100:] = float("-inf")
    i["logits"][3:6, :650] = torch.finfo(ty).min
    i["logits"][6, 5] = float("nan")
    i["logits"][7, :] = float("-inf")
    i["logits"][7, 699] = -3.0
    i["logits"][9, 17] = float("inf")
    i["logits"][12] = float("-inf")
    i["tokens"][13] = 4
    tok, cnt, lp = check_verify(sv, i, rows)
    assert tok[12] == 0 and cnt[4] == 1 and lp[12] == -np.inf and tok[13] == -1


def test_verify_edges_of_the_random_numbers(sv):
    rows = [2, 2, 2, 2]
    i = verify_inputs(F32, rows, 50, [1.0] * 4, False, seed=5)
    i["u"][:] = 0.0  # accepted whenever p > 0; the first index with weight
    tok, cnt, _ = check_verify(sv, i, rows)
    assert cnt.tolist() == [2] * 4 and (tok[1::2] == 0).all()
    i["u"][:] = 1.0 - 2.0 ** -24
    i["logits"][:] = -1e4  # equal weights; the last index
    i["logits"][:, 30:] = float("-inf")
    tok, cnt, _ = check_verify(sv, i, rows)
    assert cnt.tolist() == [1] * 4 and (tok[0::2] <= 29).all()
    # a draft outside the vocabulary is refused, whatever the numbers
    i = verify_inputs(F32, rows, 50, [1.0, 0.0, 1.0, 0.0], True, seed=6)
    i["u"][:] = 0.0
    i["tokens"][1] = 50
    i["tokens"][3] = -1
    i["tokens"][5] = 2 ** 31 - 1
    i["tokens"][7] = -2 ** 31
    _, cnt, _ = check_verify(sv, i, rows)
    assert cnt.tolist() == [1] * 4


def test_verify_rest_that_is_empty_falls_back_to_the_target(sv):
    """q above p everywhere it counts: nothing is left of max(p - q, 0)."""
    i = verify_inputs(F32, [2], 40, [1.0], True, seed=7)
    i["draft_probs"][:] = 1.0
    i["u"][:] = 0.999
    _, cnt, _ = check_verify(sv, i, [2])
    assert cnt.tolist() == [1]


def test_verify_keeps_the_targets_distribution(sv):
    """20,000 sequences of one draft: the first token is distributed as the target's, drafted from another
    distribution. Each of 8 frequencies within 5 standard errors, for both kinds of drafter."""
    n, v = 20000, 8
    g = gen(11)
    l = torch.randn(v, generator=g, device="cuda") * 1.5
    q1 = torch.softmax(l + torch.randn(v, generator=g, device="cuda"), 0)
    p = torch.softmax(l / 0.9, 0).cpu().numpy()
    for probs in (True, False):
        q = q1.expand(2 * n, v)
        tokens = torch.zeros(2 * n, dtype=torch.int32, device="cuda")
        tokens[1::2] = torch.multinomial(q1, n, replacement=True, generator=g).int() if probs else 3
        out, cnt, _ = sv.verify(l.expand(2 * n, v), tokens, ints(range(0, 2 * n + 1, 2)),
                                torch.rand(2 * n, generator=g, device="cuda"), torch.full((n,), 0.9, device="cuda"),
                                draft_probs=q if probs else None)
        f = np.bincount(out[0::2].cpu().numpy(), minlength=v) / n
        assert (np.abs(f - p) < 5 * np.sqrt(p * (1 - p) / n)).all(), (f, p)
        second = out[1::2][cnt == 2].cpu().numpy()
        f2 = np.bincount(second, minlength=v) / len(second)
        assert (np.abs(f2 - p) < 5 * np.sqrt(p * (1 - p) / len(second))).all()


def test_verify_layouts_streams_graphs(sv):
    rows = [4, 1, 3] * 4
    i = verify_inputs(BF16, rows, 1001, [0.8] * 12, True, seed=9)
    want = [t.clone() for t in sv.verify(i["logits"], i["tokens"], i["seq_rows"], i["u"], i["temperature"],
                                         i["draft_probs"])]
    for pad, off in ((3, 0), (0, 1), (7, 8)):
        def spaced(t):
            flat = torch.zeros(t.shape[0] * (t.shape[1] + pad) + off, dtype=t.dtype, device="cuda")
            w = flat[off:].view(t.shape[0], -1)[:, : t.shape[1]]
            w.copy_(t)
            return w
        got = sv.verify(spaced(i["logits"]), i["tokens"], i["seq_rows"], i["u"], i["temperature"],
                        spaced(i["draft_probs"]))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = sv.verify(i["logits"], i["tokens"], i["seq_rows"], i["u"], i["temperature"], i["draft_probs"],
                    stream=st.cuda_stream)
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    out, g = [torch.zeros_like(t) for t in want], torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sv.verify(i["logits"], i["tokens"], i["seq_rows"], i["u"], i["temperature"], i["draft_probs"], out=out)
    i["temperature"].zero_()
    g.replay()
    torch.cuda.synchronize()
    wt, wc, _, _ = verify_ref(i, rows)
    assert (out[0].cpu().numpy() == wt).all() and (out[1].cpu().numpy() == wc).all()


def test_verify_refusals(sv):
    from loom_b200 import LoomCudaError
    rows = [2, 3]
    i = verify_inputs(F32, rows, 64, [1.0, 0.5], True)
    for kw in (dict(logits=i["logits"].double()), dict(logits=i["logits"].cpu()), dict(tokens=i["tokens"].long()),
               dict(tokens=i["tokens"][:4]), dict(u=i["u"].half()), dict(u=i["u"][:3]), dict(seq_rows=i["seq_rows"].cpu()),
               dict(temperature=i["temperature"][:1]), dict(draft_probs=i["draft_probs"].half()),
               dict(draft_probs=i["draft_probs"][:, :63]), dict(logits=i["logits"].t().contiguous().t())):
        j = dict(i, **kw)
        with pytest.raises(LoomCudaError):
            sv.verify(j["logits"], j["tokens"], j["seq_rows"], j["u"], j["temperature"], j["draft_probs"])


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "f16", "bf16"])
def test_what_scratch_holds_does_not_matter(sv, ty):
    """The kept buffer full of NaN gives what a fresh one gives, in every operator."""
    rows, lens = [3, 1, 0, 5] * 4, [70, 300, 9, 5] * 4
    calls = []
    for heads, kv, hd, prefix in ((32, 4, 128, 5000), (6, 2, 33, 90)):
        i = attn_inputs(ty, rows, lens, heads, kv, hd, prefix, 300, seed=2)
        calls.append(lambda i=i: (attn(sv, i),))
    for n in (5, 70):
        j = lora_inputs(ty, n, 700, 130, [67, 2, 0, 33], [r % 5 for r in range(n)], seed=n)
        calls.append(lambda j=j: (lora(sv, j),))
    for seqs, probs in ((2, True), (15, False), (15, True)):
        k = verify_inputs(ty, [3] * seqs, 5003, [1.0] * seqs, probs, seed=4)
        calls.append(lambda k=k: sv.verify(k["logits"], k["tokens"], k["seq_rows"], k["u"], k["temperature"], k["draft_probs"]))
    first = [[o.clone() for o in c()] for c in calls]
    for c, want in zip(calls, first):
        for ws in sv._kept.values():
            ws.fill_(255)
        for o, w in zip(c(), want):
            assert torch.equal(o, w)
