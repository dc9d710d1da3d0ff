"""GPU tests of the batched-serving operators' edges: streams and captures, values
and random numbers at the ends of their ranges. Inputs, plain forms and tolerances
are those of test_gpu_serve.py."""
import subprocess
import sys

import pytest
import torch

from tests.test_gpu_serve import (ATTN_TOL, BF16, F16, F32, TYPES, attn, attn_inputs, attn_ref, check_verify, lora,  # noqa: F401
                                  lora_inputs, lora_ref, rel, sv, verify_inputs)

pytestmark = pytest.mark.gpu


# ---- streams --------------------------------------------------------------------

def test_a_call_on_another_stream_takes_no_memory_that_pending_kernels_use(sv):
    """What the current stream has freed is still written by a kernel that waits there; the call on `st` does not."""
    i = attn_inputs(BF16, [3, 1, 2] * 5, [50, 300, 129] * 5, 32, 4, 128, 1000, 320, seed=8)
    j = lora_inputs(BF16, 70, 512, 512, [16, 8, 32], [r % 4 - 1 for r in range(70)], seed=6)
    k = verify_inputs(F32, [3] * 9, 3001, [1.0] * 9, True, seed=4)
    st = torch.cuda.Stream()
    for call in (lambda s: (attn(sv, i, stream=s),), lambda s: (lora(sv, j, stream=s),),
                 lambda s: sv.verify(k["logits"], k["tokens"], k["seq_rows"], k["u"], k["temperature"], k["draft_probs"],
                                     stream=s)):
        want = [t.clone() for t in call(None)]
        torch.cuda.synchronize()
        old = [torch.empty_like(t) for t in want] + [torch.empty(n << 10, dtype=torch.uint8, device="cuda")
                                                     for n in (1, 16, 256, 1024, 4096)]
        torch.cuda._sleep(50_000_000)
        for t in old:
            t.fill_(77)
        ptrs = {t.data_ptr() for t in old}
        del old, t
        got = call(st.cuda_stream)
        torch.cuda.synchronize()
        assert not ptrs & {g.data_ptr() for g in got}
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_a_captured_call_on_a_joined_stream_keeps_its_scratch(sv):
    i = attn_inputs(F16, [3, 1, 2] * 5, [50, 300, 129] * 5, 32, 4, 128, 1000, 320, seed=8)
    j = lora_inputs(F32, 70, 512, 512, [16, 8, 32], [r % 4 - 1 for r in range(70)], seed=6)
    want = attn(sv, i).clone(), lora(sv, j).clone()
    torch.cuda.synchronize()
    out, st, g = [torch.zeros_like(w) for w in want], torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cur = torch.cuda.current_stream()
        st.wait_stream(cur)
        attn(sv, i, out=out[0], stream=st.cuda_stream)
        lora(sv, j, out=out[1], stream=st.cuda_stream)
        cur.wait_stream(st)
    room = [torch.full((n << 10,), 255, dtype=torch.uint8, device="cuda") for n in (64, 1024, 4096, 16384) * 4]
    with torch.cuda.stream(st):
        more = [torch.full((n << 10,), 255, dtype=torch.uint8, device="cuda") for n in (64, 1024, 4096, 16384) * 4]
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(out, want))
    assert all(bool((t == 255).all()) for t in room + more)  # the graph writes to none of them


# ---- attention ------------------------------------------------------------------

@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-42, -0.05])
@pytest.mark.parametrize("ty", TYPES, ids=["f32", "f16", "bf16"])
def test_attn_scales_without_a_sign(sv, ty, scale):
    """A scale of zero weighs every position alike, whichever kernel takes the prefix; a negative one turns the order."""
    for rows, lens, heads, kv, hd, prefix, cap in (([4] * 33, list(range(4, 37)), 32, 4, 128, 4099, 40),
                                                   ([100, 0, 200], [120, 0, 200], 8, 8, 48, 2401, 200),
                                                   ([2, 1], [5, 70], 8, 2, 33, 77, 80)):
        i = dict(attn_inputs(ty, rows, lens, heads, kv, hd, prefix, cap, seed=prefix), scale=scale)
        assert rel(attn(sv, i), attn_ref(i, rows, lens)) < ATTN_TOL[ty]


ENDS = {
    "few rows": ([2, 1, 3], [40, 65, 9], 8, 2, 128, 150, 72),
    "many rows": ([4] * 33, list(range(4, 37)), 32, 4, 128, 4099, 40),
    "more rows of a sequence": ([20, 12], [60, 30], 8, 2, 64, 100, 60),
    "heads of 200": ([2, 1], [40, 65], 4, 2, 200, 150, 72),
    "odd heads": ([2, 1], [40, 65], 4, 2, 33, 150, 72),
}


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", ENDS, ids=[s.replace(" ", "_") for s in ENDS])
def test_attn_infinities_that_are_seen(sv, ty, shape):
    """A key whose score is -inf has no weight, one far below the others neither; an infinite value is the result's."""
    rows, lens, heads, kv, hd, prefix, cap = ENDS[shape]
    i = attn_inputs(ty, rows, lens, heads, kv, hd, prefix, cap, seed=3)
    i["q"][..., 0] = i["q"][..., 0].abs() + 0.25
    for k, at in (("pk", (7,)), ("pk", (prefix - 1,)), ("ok", (0, 3)), ("ok", (1, 0))):
        i[k][at][..., 0] = float("-inf")
    i["pk"][64, :, 0] = -torch.finfo(ty).max
    assert rel(attn(sv, i), attn_ref(i, rows, lens)) < ATTN_TOL[ty]
    i["pv"][20, 0, 5] = float("inf")
    i["ov"][0, 2, -1, 9] = float("-inf")
    out, want = attn(sv, i), attn_ref(i, rows, lens)
    assert torch.equal(torch.isinf(out), torch.isinf(want)) and torch.equal(out[torch.isinf(want)].double(), want[torch.isinf(want)])
    fin = torch.isfinite(want)
    assert bool(torch.isfinite(out[fin]).all()) and not bool(fin.all()) and rel(out[fin], want[fin]) < ATTN_TOL[ty]


# ---- verification ---------------------------------------------------------------

@pytest.mark.parametrize("ty", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("probs", [True, False], ids=["probs", "sure"])
@pytest.mark.parametrize("vocab,seqs", [(40, 2), (32000, 2), (32000, 40), (151937, 3)])
def test_verify_random_number_of_one(sv, ty, probs, vocab, seqs):
    """A uniform number rounded up to 1: no running sum exceeds the whole; the last token with weight is chosen."""
    rows, last = [2] * seqs, vocab - vocab // 5 - 1
    i = verify_inputs(ty, rows, vocab, [1.0] * seqs, probs, seed=vocab)
    i["u"][:] = 1.0
    i["logits"][:, last + 1:] = float("-inf")
    i["tokens"][1::2] = 3
    if probs:  # refuses the draft, and leaves the tokens at the end their weight
        i["draft_probs"][:, 3] = 1.0
        i["draft_probs"][:, vocab // 2:] = 0.0
        i["draft_probs"][2, 3] = 0.5  # but for the second sequence's, whose p rounds to 1: then the token after it
        i["logits"][2:4, 3] = i["logits"][2:4].float().amax(1).to(ty) + 40
    tok, cnt, _ = (t.cpu().numpy() for t in sv.verify(i["logits"], i["tokens"], i["seq_rows"], i["u"], i["temperature"],
                                                       i["draft_probs"]))
    for b in range(seqs):
        if probs and b == 1:
            assert cnt[b] == 2 and tok[2] == 3
            w = torch.exp(i["logits"][3].float() - i["logits"][3].float().amax())
            assert tok[3] == int(torch.nonzero(w > 0)[-1])
        else:
            assert cnt[b] == 1 and tok[2 * b] == last and tok[2 * b + 1] == -1


@pytest.mark.parametrize("ty", [F16, BF16], ids=["f16", "bf16"])
def test_verify_one_launch_beyond_the_registers_of_a_cluster(sv, ty):
    """The longest rows that take one launch: more than a cluster's CTAs keep in registers."""
    for vocab in (163841, 190001, 204800):
        for probs in (True, False):
            i = verify_inputs(ty, [1, 2], vocab, [0.0, 0.9], probs, seed=vocab, std=3.0)
            check_verify(sv, i, [1, 2])
            i["logits"][:, : vocab - 5] = float("-inf")
            check_verify(sv, i, [1, 2])


def test_verify_one_launch_of_very_many_rows(sv):
    """More rows than the two passes' grid holds, of more logits than registers do: all the same row, each with its
    own random number."""
    n, vocab = 65537, 120001
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    l = torch.randn(vocab, generator=g, device="cuda") * 3
    u = torch.rand(n, generator=g, device="cuda")
    temp = torch.full((n,), 0.9, device="cuda")
    temp[::3] = 0.0
    rows = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    tok, cnt, lp = sv.verify(l.expand(n, vocab), torch.zeros(n, dtype=torch.int32, device="cuda"), rows, u, temp)
    assert bool((cnt == 1).all()) and bool((tok[::3] == l.argmax()).all())
    x = torch.log_softmax(l.double() / 0.9, 0)
    c = x.exp().cumsum(0)
    t, want = tok.long(), u.double() * c[-1]
    over = c[t] - want, want - (c[t] - x[t].exp())  # what the choice is above and below the threshold
    drawn = torch.arange(n, device="cuda") % 3 != 0
    assert bool((torch.minimum(*over)[drawn] > -1e-5).all())
    want_lp = torch.where(drawn, x[t], torch.log_softmax(l.double(), 0)[t])
    assert bool(((lp.double() - want_lp).abs() <= 2e-5 + 2e-6 * want_lp.abs()).all())


# ---- adapters -------------------------------------------------------------------

@pytest.mark.parametrize("ty", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 20, 40, 150])
def test_lora_infinite_operands(sv, ty, n):
    """Infinities and values at the end of the range go where plain arithmetic takes them, and no further."""
    ranks, ids = [1, 16, 70], [r % 3 for r in range(n)]
    for k, at, v in (("x", (0, 5), float("inf")), ("x", (n // 2, 600), float("-inf")), ("x", (0, 7), torch.finfo(F32).max),
                     ("a", (0, 0, 3), float("inf")), ("a", (1 % n, 2, 300), float("-inf")), ("b", (0, 9, 0), float("inf")),
                     ("b", (1, 100, 15), float("-inf")), ("b", (2, 33, 69), float("inf")), ("b", (2, 40, 68), torch.finfo(ty).max)):
        i = lora_inputs(ty, n, 700, 130, ranks, ids, seed=n)
        i["a"] = i["a"] * 2.0 ** -8  # the largest x stays in range
        i[k][at] = v
        out, want = lora(sv, i), lora_ref(i)
        fin = torch.isfinite(want)
        assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(torch.isinf(out), torch.isinf(want))
        big = torch.isinf(want)
        assert torch.equal(out[big].double(), want[big])
        # by rows: those with huge results have a norm of their own
        for r in range(n):
            f = fin[r]
            if f.any():
                assert float((out[r][f].double() - want[r][f]).abs().max()) <= 2e-5 * float(want[r][f].abs().max())


# ---- the backend's life ---------------------------------------------------------

def test_calls_after_a_shutdown_bring_the_backend_up_again():
    code = """
import torch
from loom_b200 import _lib, serve
x, a, b = torch.ones(2, 8, device="cuda"), torch.ones(1, 2, 8, device="cuda"), torch.ones(1, 4, 2, device="cuda")
ranks, ids, scales = (torch.tensor(v, dtype=t, device="cuda") for v, t in (([2], torch.int32), ([0, -1], torch.int32), ([0.5], torch.float32)))
for _ in range(2):
    y = serve.lora(x, a, b, ranks, scales, ids)
    assert y.tolist() == [[8.0] * 4, [0.0] * 4], y
    torch.cuda.synchronize()
    _lib.lib().loom_cuda_shutdown()
print("up again")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "up again" in r.stdout, r.stderr[-2000:]


def alone(code):
    """In a process of its own: the word of waits that gave up stays set."""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.endswith("done\n"), r.stdout + r.stderr[-2000:]


def test_attn_waits_that_give_up():
    """No result, the error word, and the next call is right."""
    alone("""
import torch
from loom_b200 import _lib, backend
from tests.test_gpu_serve import ATTN_TOL, TYPES, attn, attn_inputs, attn_ref, rel
import loom_b200.serve as sv
backend.init(0)
L = _lib.lib()
assert L.loom_cuda_device_error() == 0
shapes = (([3, 1, 2] * 5, [50, 300, 129] * 5, 32, 4, 128, 1000, 320), ([4] * 33, list(range(4, 37)), 32, 4, 128, 4099, 40),
          ([100, 0, 200], [120, 0, 200], 8, 8, 48, 2401, 200), ([2, 2], [64, 20], 16, 4, 256, 130, 70))
for ty in TYPES:
    for rows, lens, *rest in shapes:
        i = attn_inputs(ty, rows, lens, *rest, seed=8)
        assert rel(attn(sv, i), attn_ref(i, rows, lens)) < ATTN_TOL[ty]
        assert L.loom_cuda_attn_fail_waits(1) == 0
        for _ in range(3):
            out = attn(sv, i)
        torch.cuda.synchronize()
        assert L.loom_cuda_device_error() == 128
        if ty is not torch.float32:  # f32 takes rows that came out NaN again
            assert bool(torch.isnan(out).all())
        assert L.loom_cuda_attn_fail_waits(0) == 1
        assert rel(attn(sv, i), attn_ref(i, rows, lens)) < ATTN_TOL[ty]
print("done")
""")
