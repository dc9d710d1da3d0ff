"""GPU tests of the drafted step of sequences that share a prompt
(loom_cuda_model_shared_step: shared-prefix attention, adapters and draft
verification through every layer of a model), against the same model's
single-sequence decode.

Logits are held to 2e-2 relative L2, the tolerance of the model's other fast
forms: the attention sums in another order, which can move an int8 activation of
the next matvec."""
import dataclasses
import subprocess
import sys

import numpy as np
import pytest
import torch

from loom_b200 import LoomCudaError, _lib
from loom_b200.model import Adapters, DeviceModel, qwen3_moe, tiny_llama
from tests.conftest import rel_l2

pytestmark = pytest.mark.gpu
TOL = 2e-2


def small_llama(ctx=96):
    s = tiny_llama(ctx_len=ctx)
    s.n_layers = 2
    return s


def alone(dev, prompt, tokens):
    """The sequence decoded by itself behind the prompt: logits after each of its tokens."""
    return np.stack([dev.decode(int(t), len(prompt) + i, logits=True)[1].copy() for i, t in enumerate(tokens)])


@pytest.mark.parametrize("spec", [small_llama(), qwen3_moe(n_layers=2, ctx_len=640, n_expert=16, vocab=4096)],
                         ids=["tiny_llama", "qwen3"])
def test_logits_match_each_sequence_alone_over_two_steps(be, spec):
    dev = DeviceModel(spec)
    rng = np.random.default_rng(5)
    try:
        prompt = rng.integers(1, spec.vocab, size=33)
        dev.prefill(prompt)
        seqs = [rng.integers(1, spec.vocab, size=n).tolist() for n in (5, 2, 7, 3)]
        cuts = [2, 1, 4, 1]  # rows of the first step; the rest are the second's
        first = dev.shared_step(len(prompt), [s[:c] for s, c in zip(seqs, cuts)], cuts, logits=True)
        second = dev.shared_step(len(prompt), [s[c:] for s, c in zip(seqs, cuts)], [len(s) for s in seqs], logits=True)
        at = [0, 0]
        for s, c in zip(seqs, cuts):
            want = alone(dev, prompt, s)
            got = np.concatenate([first[2][at[0]: at[0] + c], second[2][at[1]: at[1] + len(s) - c]])
            at = [at[0] + c, at[1] + len(s) - c]
            for g, w in zip(got, want):
                assert rel_l2(g, w) < TOL
    finally:
        dev.free()


def test_greedy_drafts_give_the_greedy_sequence(be):
    """Whatever is drafted, the emitted tokens are those of greedy decoding; right drafts are accepted."""
    spec = small_llama()
    dev = DeviceModel(spec)
    rng = np.random.default_rng(9)
    try:
        prompt = rng.integers(1, spec.vocab, size=20)
        nxt, _ = dev.prefill(prompt)
        starts = [int(nxt), 17, 4242]
        want, gaps = [], []
        for s in starts:  # greedy continuation of each start, and how clear each choice was
            toks, clear, t = [], [], s
            for i in range(10):
                n, lg = dev.decode(t, len(prompt) + i, logits=True)
                top = np.sort(lg)[-2:]
                clear.append(float(top[1] - top[0]) > 1e-3)
                toks.append(int(n))
                t = int(n)
            want.append(toks)
            gaps.append(clear)
        assert all(all(g) for g in gaps)
        done, length, last = [[] for _ in starts], [0] * 3, list(starts)
        steps = 0
        while min(len(d) for d in done) < 8:
            rows = []
            for b, d in enumerate(done):
                right = (want[b] + [1, 1])[len(d): len(d) + 2] or [1, 1]  # sequence 0 drafts right, 1 one right and one wrong, 2 wrong
                draft = right if b == 0 else [right[0], (right[1] + 1) % spec.vocab] if b == 1 and len(right) == 2 else [7, 7]
                rows.append([last[b]] + draft[: max(0, 9 - len(d))])
            got, lps, _ = dev.shared_step(len(prompt), rows, [n + len(r) for n, r in zip(length, rows)])
            for b, toks in enumerate(got):
                assert len(toks) <= len(rows[b]) and all(p <= 0 for p in lps[b])
                done[b] += toks
                length[b] += len(toks)
                last[b] = toks[-1]
            steps += 1
            for b in range(3):
                assert done[b][: len(want[b])] == want[b][: len(done[b])], (b, done[b], want[b])
            if steps == 1:
                assert [len(t) for t in got] == [3, 2, 1]
    finally:
        dev.free()


def test_each_sequence_has_its_adapter(be):
    """Several adapters in one step: every sequence as when it is alone with its own, those without as the plain model."""
    spec = small_llama()
    rng = np.random.default_rng(3)
    d, q, v, n, rank = spec.dim, spec.n_heads * spec.head_dim, spec.n_kv_heads * spec.head_dim, 3, 5
    rand = lambda *s: torch.tensor(rng.standard_normal(s).astype(np.float32), device="cuda")  # noqa: E731
    layers = {k: [(rand(n, rank, d) / d ** 0.5, rand(n, rows, rank)) for _ in range(spec.n_layers)] for k, rows in (("q", q), ("v", v))}
    ad = Adapters(layers["q"], layers["v"], [5, 2, 4], [0.5, -1.25, 2.0])
    prompt, seqs, ids = rng.integers(1, spec.vocab, size=12), [rng.integers(1, spec.vocab, size=3).tolist() for _ in range(4)], [2, -1, 0, 1]
    dev = DeviceModel(spec)
    try:
        dev.prefill(prompt)
        _, _, got = dev.shared_step(len(prompt), seqs, [3] * 4, adapters=ad, adapter_ids=ids, logits=True)
        _, _, none = dev.shared_step(len(prompt), seqs, [3] * 4, adapters=ad, adapter_ids=[-1] * 4, logits=True)
        _, _, without = dev.shared_step(len(prompt), seqs, [3] * 4, logits=True)
        assert np.array_equal(none, without)
        for b, i in enumerate(ids):
            _, _, solo = dev.shared_step(len(prompt), [seqs[b]], [3], adapters=ad, adapter_ids=[i], logits=True)
            assert rel_l2(got[3 * b: 3 * b + 3], solo) < TOL
            assert (rel_l2(got[3 * b: 3 * b + 3], without[3 * b: 3 * b + 3]) > 0.1) == (i >= 0)
    finally:
        dev.free()


def test_adapters_equal_merged_weights(be):
    """A query adapter beside f32 weights W against a model whose weights are W + scale B A: in one layer the
    prompt's keys and values are the same in both."""
    spec = small_llama()
    spec = dataclasses.replace(spec, types=dict(spec.types, attn_q=0, attn_v=0))
    spec.n_layers = 1  # the prompt's keys and values then come from the embeddings alone
    rng = np.random.default_rng(4)
    d, q, v = spec.dim, spec.n_heads * spec.head_dim, spec.n_kv_heads * spec.head_dim
    host = {"blk.0.attn_q": (rng.standard_normal((q, d)) / np.sqrt(d)).astype(np.float32),
            "blk.0.attn_v": (rng.standard_normal((v, d)) / np.sqrt(d)).astype(np.float32)}
    a = (rng.standard_normal((1, 4, d)) / np.sqrt(d)).astype(np.float32)
    b = (rng.standard_normal((1, q, 4)) * 0.3).astype(np.float32)
    ad = Adapters([(torch.tensor(a, device="cuda"), torch.tensor(b, device="cuda"))], [None], [4], [1.5])
    merged = dict(host, **{"blk.0.attn_q": (host["blk.0.attn_q"] + 1.5 * b[0].astype(np.float64) @ a[0]).astype(np.float32)})
    prompt, toks = rng.integers(1, spec.vocab, size=9), rng.integers(1, spec.vocab, size=4).tolist()
    one, two = DeviceModel(spec, host=host), DeviceModel(spec, host=merged)
    try:
        one.prefill(prompt)
        two.prefill(prompt)  # its queries differ, its keys and values do not
        got = one.shared_step(len(prompt), [toks], [4], adapters=ad, adapter_ids=[0], logits=True)[2]
        want = alone(two, prompt, toks)
        plain = alone(one, prompt, toks)
        for g, w, p in zip(got, want, plain):
            assert rel_l2(g, w) < TOL and rel_l2(p, w) > rel_l2(g, w)
    finally:
        one.free()
        two.free()


def test_sampling_uses_the_random_numbers(be):
    spec = small_llama()
    dev = DeviceModel(spec)
    rng = np.random.default_rng(2)
    try:
        prompt = rng.integers(1, spec.vocab, size=10)
        dev.prefill(prompt)
        rows = [[5, 6], [7]]
        seen = set()
        for u in (0.0, 0.3, 0.6, 0.99):
            got, lps, lg = dev.shared_step(len(prompt), rows, [2, 1], u=[0.999, u, u], temperature=[1.0, 0.5], logits=True)
            x = lg[2].astype(np.float64) / 0.5
            p = np.exp(x - x.max())
            p /= p.sum()
            c = p.cumsum()
            t = got[1][0]
            assert c[t] > u * c[-1] - 1e-6 and (c[t - 1] if t else 0.0) <= u * c[-1] + 1e-6
            assert abs(lps[1][0] - np.log(p[t])) < 1e-4 * max(1, abs(np.log(p[t])))
            seen.add(t)
        assert len(seen) > 1
        q = torch.full((3, spec.vocab), 1.0 / spec.vocab, device="cuda")
        got, _, _ = dev.shared_step(len(prompt), rows, [2, 1], u=[0.0, 0.5, 0.5], temperature=[1.0, 1.0], draft_probs=q)
        assert got[0][0] == 6 and len(got[0]) == 2  # p > 0 is enough at u = 0
    finally:
        dev.free()


def test_refusals_leave_the_model_working(be):
    spec = small_llama()
    dev = DeviceModel(spec)
    try:
        dev.prefill([1, 2, 3])
        good = dict(prefix_len=3, rows=[[4, 5], [6]], seq_len=[2, 1])
        for bad in (dict(prefix_len=96), dict(rows=[[4, 32000], [6]]), dict(rows=[[4, 5], []]), dict(seq_len=[1, 1]),
                    dict(seq_len=[2, 94]), dict(seq_len=[2]), dict(u=[0.5]), dict(temperature=[1.0]),
                    dict(draft_probs=torch.zeros((3, 10), device="cuda"))):
            with pytest.raises(LoomCudaError):
                dev.shared_step(**dict(good, **bad))
        with pytest.raises(LoomCudaError):
            z = torch.zeros((1, 2, 300), device="cuda")
            ad = Adapters([(z, z.transpose(1, 2).contiguous())] * 2, None, [2], [1.0])
            dev.shared_step(**good, adapters=ad, adapter_ids=[0, 0])
        with pytest.raises(LoomCudaError):
            Adapters(None, None, [], [])
        got, _, _ = dev.shared_step(**good)
        assert [len(g) for g in got] in ([1, 1], [2, 1])
        with pytest.raises(LoomCudaError):  # the first call fixed the number of sequences
            dev.shared_step(3, [[1]] * 3, [1] * 3)
    finally:
        dev.free()


def test_batched_decode_and_prefill_keep_their_results(be):
    """decode_batch before and after a shared step of the same model: bit for bit the same."""
    spec = small_llama()
    dev = DeviceModel(spec)
    other = DeviceModel(spec)
    rng = np.random.default_rng(8)
    try:
        for m in (dev, other):
            m.prefill([3, 1, 4, 1, 5])
        dev.shared_step(5, [[9, 2], [6]], [2, 1])
        toks = rng.integers(1, spec.vocab, size=(4, 2))
        for p in range(4):
            a, la = dev.decode_batch(toks[p], [p, p], logits=True)
            b, lb = other.decode_batch(toks[p], [p, p], logits=True)
            assert np.array_equal(a, b) and np.array_equal(la, lb)
        assert dev.decode(7, 5, logits=True)[0] == other.decode(7, 5, logits=True)[0]
    finally:
        dev.free()
        other.free()


def test_growing_steps_hold_what_the_largest_needs(be):
    """Steps of 1 to 60 rows: the device memory they hold follows the largest, not all of them together."""
    spec = small_llama()
    dev = DeviceModel(spec)
    other = DeviceModel(spec)
    rng = np.random.default_rng(7)
    try:
        for m in (dev, other):
            m.prefill([3, 1, 4, 1, 5])
        toks = rng.integers(1, spec.vocab, size=60).tolist()
        dev.shared_step(5, [[9]], [1])
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0]
        for n in range(1, 61):
            _, _, got = dev.shared_step(5, [toks[:n]], [n], logits=True)
        held = before - torch.cuda.mem_get_info()[0]
        # logits of 60 rows: 7.7 MB; the layers' rows and the scratch less. Twice that, and whole pages of 2 MB each
        assert held < 64 << 20, held
        _, _, want = other.shared_step(5, [toks], [60], logits=True)
        assert np.array_equal(got, want)
    finally:
        dev.free()
        other.free()


def test_the_scratch_follows_the_prompt(be):
    """Another cut of the prompt, another number of sequences within the first call's: results as in a fresh model."""
    spec = small_llama(ctx=640)
    dev, fresh = DeviceModel(spec), None
    rng = np.random.default_rng(17)
    try:
        prompt = rng.integers(1, spec.vocab, size=500).tolist()
        dev.prefill(prompt)
        for pre, cuts in ((3, [1, 1, 1]), (500, [3, 1, 2]), (40, [9, 9])):
            rows = [rng.integers(1, spec.vocab, size=c).tolist() for c in cuts]
            _, _, got = dev.shared_step(pre, rows, cuts, logits=True)
            fresh = DeviceModel(spec)
            fresh.prefill(prompt)
            _, _, want = fresh.shared_step(pre, rows, cuts, logits=True)
            assert np.array_equal(got, want)
            fresh.free()
            fresh = None
    finally:
        dev.free()
        if fresh is not None:
            fresh.free()


def test_a_missing_matrix_is_refused_before_anything_runs(be):
    """A layer with the first matrix of an adapter and not the second."""
    spec = small_llama()
    dev = DeviceModel(spec)
    try:
        dev.prefill([1, 2, 3])
        d, q = spec.dim, spec.n_heads * spec.head_dim
        pair = (torch.zeros((1, 2, d), device="cuda"), torch.zeros((1, q, 2), device="cuda"))
        ad = Adapters([pair] * spec.n_layers, [pair] * spec.n_layers, [2], [1.0])  # q and v are as wide here
        step = dict(adapters=ad, adapter_ids=[0, -1])
        dev.shared_step(3, [[4, 5], [6]], [2, 1], **step)
        for k in (1, 3):  # B of q, of v
            was, ad._tables[k][1] = ad._tables[k][1], None
            launched = be.kernelLaunches()
            with pytest.raises(LoomCudaError, match="matrices"):
                dev.shared_step(3, [[4, 5], [6]], [2, 1], **step)
            assert be.kernelLaunches() == launched
            ad._tables[k][1] = was
        dev.shared_step(3, [[4, 5], [6]], [2, 1], **step)
    finally:
        dev.free()


def test_a_step_whose_attention_gave_up_is_an_error():
    """Waits of the attention that give up end the step with an error, not with tokens; the next step is right. (In a
    process of its own: the word of waits that gave up stays set.)"""
    code = """
import numpy as np
from loom_b200 import LoomCudaError, _lib, backend
from loom_b200.model import DeviceModel
from tests.test_gpu_shared_step import small_llama
backend.init(0)
dev = DeviceModel(small_llama())
dev.prefill([3, 1, 4, 1, 5])
step = dict(prefix_len=5, rows=[[9, 2], [6]], seq_len=[2, 1], logits=True)
want = dev.shared_step(**step)
_lib.lib().loom_cuda_attn_fail_waits(1)
for _ in range(2):
    try:
        dev.shared_step(**step)
        raise SystemExit("no error")
    except LoomCudaError as e:
        assert "gave up" in str(e), e
_lib.lib().loom_cuda_attn_fail_waits(0)
got = dev.shared_step(**step)
assert got[0] == want[0] and got[1] == want[1] and np.array_equal(got[2], want[2])
assert _lib.lib().loom_cuda_device_error() == 128
print("done")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.endswith("done\n"), r.stdout + r.stderr[-2000:]


def test_a_step_after_memory_was_refused(be):
    """An allocation that failed is reported by the call that asked for it, not by the next one."""
    spec = small_llama()
    dev = DeviceModel(spec)
    try:
        dev.prefill([3, 1, 4, 1, 5])
        step = dict(prefix_len=5, rows=[[9, 2], [6]], seq_len=[2, 1], logits=True)
        want = dev.shared_step(**step)
        plain = dev.decode(7, 5, logits=True)[1].copy()
        for call, same in ((lambda: dev.shared_step(**step)[2], want[2]), (lambda: dev.decode(7, 5, logits=True)[1], plain),
                           (lambda: dev.shared_step(**step)[2], want[2])):
            assert _lib.lib().loom_cuda_reserve(1 << 30, 1 << 16, 1 << 10, 1, 1) == _lib.ERROR  # 2^46 bytes
            assert "out of memory" in _lib.last_error()
            assert np.array_equal(call(), same)
    finally:
        dev.free()
