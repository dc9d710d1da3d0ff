"""Operators of one batched serving step (include/loom_cuda.h, "batched
serving"): attention of sequences that share a prompt, low-rank adapters of many
requests, verification of drafted tokens.

All three share one row layout: the rows of sequence b are seq_rows[b] ..
seq_rows[b + 1] - 1 (cuda int32 [n_seqs + 1]): its last accepted token, then its
drafts. Buffers are torch cuda tensors; arguments of a wrong type, shape or
layout raise LoomCudaError before anything runs. A call runs on `stream` (a
cudaStream_t), or torch's current stream, and only launches. What it allocates,
scratch and outputs, is allocated on the stream it runs on; as with any second
stream, the caller orders `stream` after what made the tensors given, keeps them
until the call is done, and orders what reads the outputs after it. Under
torch.cuda.graph a call can be captured, on the current stream or on one that has
joined the capture; a `stream` that is captured by other means is refused, since
nothing would keep its scratch for the graph.
"""
from __future__ import annotations

import ctypes as C
import threading
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import LoomCudaError

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


_device = -1  # the device a call here brought the backend up on


def _need(ok: bool, why: str) -> None:
    if not ok:
        raise LoomCudaError(why)


def _up(op: str, dev: int) -> None:
    """Bring-up, unless it is up, or the refusal of a second device."""
    _lib.must(_lib.lib().loom_cuda_init(dev), op)


def _on(op: str, t) -> int:
    """The cuda device of t, on which the backend is up."""
    global _device
    dev = t.get_device() if isinstance(t, torch.Tensor) else -1
    _need(dev >= 0, f"{op}: tensors must be on a cuda device")
    if dev != _device:
        _up(op, dev)
        _device = dev
    return dev


def _refuse(op: str, dev: int, want: Sequence[tuple]) -> None:
    """Name the first tensor that is not as wanted: (name, tensor, dtype, shape, strides it must have or None)."""
    for name, t, dtype, shape, strides in want:
        if t is None or (t.dtype is dtype and t.shape == shape and t.get_device() == dev and
                         (strides is None or _laid(t, strides))):
            continue
        raise LoomCudaError(f"{op}: {name} must be {dtype} {tuple(shape)} on cuda:{dev}"
                            f"{'' if strides is None else f' with strides {strides}'}, got {t.dtype} "
                            f"{tuple(t.shape)} with strides {t.stride()} on {t.device}")
    raise LoomCudaError(f"{op}: arguments do not fit together")


def _laid(t, strides) -> bool:
    """The strides of t are these (None: any), where a dimension of more than one element has a say."""
    return t.numel() == 0 or all(w is None or s == w or n == 1 for s, w, n in zip(t.stride(), strides, t.shape))


_stream = torch._C._cuda_getCurrentRawStream  # what torch.cuda.current_stream(dev).cuda_stream gives, 1.2 us sooner
_capturing = torch.cuda.is_current_stream_capturing
_alone = threading.Lock()
_kept = {}          # (device, stream) -> scratch of calls on that stream, in their order
_KEEP = 32 << 20    # bytes of it; calls that need more take theirs from torch's allocator


def _at(dev: int, st: int):
    """Stream `st` as torch's current one."""
    return torch.cuda.stream(torch.cuda.ExternalStream(st, device=dev) if st else torch.cuda.default_stream(dev))


def _new(op: str, shape, dtype, dev: int, stream: Optional[int], read: bool = True):
    """An uninitialised tensor for a call on `stream`. Its memory comes from that stream's pool: what the current
    stream has freed may still be in use by kernels that wait there, which `stream` does not wait for. `read`: on the
    current stream, later."""
    cur = _stream(dev)
    if stream is None or stream == cur:
        return torch.empty(shape, dtype=dtype, device=dev)
    joined = _capturing()  # torch's graph is taking the current stream, and `stream` with it if that is captured too
    with _at(dev, stream):
        _need(joined or not _capturing(), f"{op}: a stream that is captured must be torch's current one, or have joined its capture")
        t = torch.empty(shape, dtype=dtype, device=dev)
    if read and t.numel() and not joined:
        t.record_stream(torch.cuda.current_stream(dev))
    return t


def _run(op: str, entry, size, desc, args, dev: int, stream: Optional[int]) -> None:
    """One call: its stream (the current one unless given) and scratch, the refusal as LoomCudaError. Small calls on one
    stream share a buffer, as they run one after the other; one that is being captured gets its own, which the graph
    keeps."""
    cur = _stream(dev)
    st = cur if stream is None else stream
    if st == cur and not _capturing():
        with _alone:  # launches of two threads on one stream may not mix while they share the buffer
            ws = _kept.get((dev, cur))
            if ws is None:
                ws = _kept[dev, cur] = torch.empty(_KEEP, dtype=torch.uint8, device=dev)
            if entry(desc, *args, ws.data_ptr(), _KEEP, cur) == _lib.OK:
                return
    # larger, captured, on a stream of the caller's, or refused: then for the reason it names, unless the backend was shut
    # down since a call here brought it up
    _up(op, dev)
    need = size(desc)
    ws = _new(op, need, torch.uint8, dev, st, read=False)
    _lib.must(entry(desc, *args, ws.data_ptr(), need, st), op)


def attn_shared(q, prefix_k, prefix_v, own_k, own_v, seq_rows, seq_len, scale: float, out=None,
                stream: Optional[int] = None):
    """Attention over a shared prefix cache and each sequence's own cache.

    q [rows, heads, hd]; prefix_k/v [prefix, kv_heads, hd]; own_k/v [seqs, cap, kv_heads, hd], all of one type
    (float32, float16, bfloat16), any strides but a last dimension of 1 (q, out: heads side by side; keys and values
    laid out alike). seq_len (cuda int32 [seqs]) counts each sequence's own positions, this step's rows included: row j
    of n sees seq_len - (n - 1 - j) of them. Returns out [rows, heads, hd]."""
    dev = _on("attn_shared", q)
    _need(q.dim() == 3 and own_k.dim() == 4 and prefix_k.dim() == 3 and q.shape[1] > 0 and q.shape[2] > 0,
          "attn_shared: q [rows, heads, hd], prefix_k/v [prefix, kv, hd], own_k/v [seqs, cap, kv, hd]")
    ty, qs = q.dtype, q.shape
    n, h, hd = qs
    seqs, cap, kv, _ = own_k.shape
    pre = prefix_k.shape[0]
    _need(ty in TYPES, f"attn_shared: type must be float32, float16 or bfloat16, got {ty}")
    if out is None:
        out = _new("attn_shared", qs, ty, dev, stream)
    pshape, oshape, i32 = (pre, kv, hd), (seqs, cap, kv, hd), torch.int32
    pst, ost, qst, dst = prefix_k.stride(), own_k.stride(), q.stride(), out.stride()
    if not (prefix_k.dtype is ty and prefix_v.dtype is ty and own_k.dtype is ty and own_v.dtype is ty and
            out.dtype is ty and seq_rows.dtype is i32 and seq_len.dtype is i32 and prefix_k.shape == pshape and
            prefix_v.shape == pshape and own_k.shape == oshape and own_v.shape == oshape and out.shape == qs and
            seq_rows.shape == (seqs + 1,) and seq_len.shape == (seqs,) and
            dev == prefix_k.get_device() == prefix_v.get_device() == own_k.get_device() == own_v.get_device() ==
            out.get_device() == seq_rows.get_device() == seq_len.get_device() and
            pst[2] == ost[3] == qst[2] == dst[2] == 1 and qst[1] == dst[1] == hd and prefix_v.stride() == pst and
            own_v.stride() == ost and seq_rows.is_contiguous() and seq_len.is_contiguous()):
        heads, one = (None, hd, 1), (1,)
        like = lambda t, u: _laid(u, t.stride()) and _laid(t, u.stride())  # noqa: E731
        if not (_laid(q, heads) and _laid(out, heads) and _laid(prefix_k, (None, None, 1)) and
                _laid(own_k, (None, None, None, 1)) and like(prefix_k, prefix_v) and like(own_k, own_v) and
                all(t.dtype is d and t.shape == s and t.get_device() == dev for t, d, s in (
                    (prefix_k, ty, pshape), (prefix_v, ty, pshape), (own_k, ty, oshape), (own_v, ty, oshape),
                    (out, ty, qs), (seq_rows, i32, (seqs + 1,)), (seq_len, i32, (seqs,)))) and
                _laid(seq_rows, one) and _laid(seq_len, one)):
            _refuse("attn_shared", dev, (
                ("q", q, ty, qs, heads), ("out", out, ty, qs, heads), ("prefix_k", prefix_k, ty, pshape, (None, None, 1)),
                ("prefix_v", prefix_v, ty, pshape, pst), ("own_k", own_k, ty, oshape, (None, None, None, 1)),
                ("own_v", own_v, ty, oshape, ost), ("seq_rows", seq_rows, i32, (seqs + 1,), one),
                ("seq_len", seq_len, i32, (seqs,), one)))
    ref = C.byref(_lib.AttnSharedDesc(TYPES[ty], scale, seqs, n, h, kv, hd, qst[0], dst[0], pre, pst[0], pst[1], cap,
                                      ost[1], ost[2], ost[0]))
    L = _lib.lib()
    _run("attn_shared", L.loom_cuda_attn_shared, L.loom_cuda_attn_shared_workspace, ref,
         (q.data_ptr(), prefix_k.data_ptr(), prefix_v.data_ptr(), own_k.data_ptr(), own_v.data_ptr(),
          seq_rows.data_ptr(), seq_len.data_ptr(), out.data_ptr()), dev, stream)
    return out


def lora(x, a, b, ranks, scales, ids, base=None, out=None, stream: Optional[int] = None):
    """out = base + scales[id] * B[id] (A[id] x) row by row; rows whose id names no adapter keep their base.

    x [rows, n_in] float32; a [adapters, max_rank, n_in], b [adapters, n_out, max_rank] of one type (float32, float16,
    bfloat16); ranks (int32) and scales (float32) [adapters]; ids int32 [rows]; base, out [rows, n_out] float32 (base
    None: zeros; out may be base). Last dimensions contiguous. Returns out."""
    dev = _on("lora", a)
    _need(a.dim() == 3 and b.dim() == 3 and x.dim() == 2, "lora: x [rows, n_in], a [n, rank, n_in], b [n, n_out, rank]")
    ty, f32, i32 = a.dtype, torch.float32, torch.int32
    na, rank, nin = a.shape
    n, nout = x.shape[0], b.shape[1]
    _need(ty in TYPES, f"lora: type must be float32, float16 or bfloat16, got {ty}")
    if out is None:
        out = _new("lora", (n, nout), f32, dev, stream)
    xst, ast, bst, dst = x.stride(), a.stride(), b.stride(), out.stride()
    cst = dst if base is None else base.stride()
    bshape, oshape = (na, nout, rank), (n, nout)
    if not (x.dtype is f32 and b.dtype is ty and ranks.dtype is i32 and scales.dtype is f32 and ids.dtype is i32 and
            out.dtype is f32 and x.shape == (n, nin) and b.shape == bshape and ranks.shape == (na,) and
            scales.shape == (na,) and ids.shape == (n,) and out.shape == oshape and
            dev == x.get_device() == b.get_device() == ranks.get_device() == scales.get_device() == ids.get_device() ==
            out.get_device() and
            (base is None or (base.dtype is f32 and base.shape == oshape and base.get_device() == dev)) and
            xst[1] == ast[2] == bst[2] == dst[1] == cst[1] == 1 and ranks.is_contiguous() and scales.is_contiguous() and
            ids.is_contiguous()):
        want = (("x", x, f32, (n, nin), (None, 1)), ("a", a, ty, (na, rank, nin), (None, None, 1)),
                ("b", b, ty, bshape, (None, None, 1)), ("ranks", ranks, i32, (na,), (1,)),
                ("scales", scales, f32, (na,), (1,)), ("ids", ids, i32, (n,), (1,)),
                ("base", base, f32, oshape, (None, 1)), ("out", out, f32, oshape, (None, 1)))
        if not all(t is None or (t.dtype is d and t.shape == s and t.get_device() == dev and _laid(t, w))
                   for _, t, d, s, w in want):
            _refuse("lora", dev, want)
    ref = C.byref(_lib.LoraDesc(TYPES[ty], n, nin, nout, na, rank, xst[0], cst[0], dst[0], ast[1], ast[0], bst[1],
                                bst[0]))
    L = _lib.lib()
    _run("lora", L.loom_cuda_lora, L.loom_cuda_lora_workspace, ref,
         (x.data_ptr(), a.data_ptr(), b.data_ptr(), ranks.data_ptr(), scales.data_ptr(), ids.data_ptr(),
          None if base is None else base.data_ptr(), out.data_ptr()), dev, stream)
    return out


def verify(logits, tokens, seq_rows, u, temperature=None, draft_probs=None, out=None, stream: Optional[int] = None):
    """Accept drafted tokens against the target's probabilities and choose the token after them.

    logits [rows, vocab] (float32, float16, bfloat16), row r for the token after row r; tokens int32 [rows] (row r's own
    token: the drafts are the rows after each sequence's first); u float32 [rows] in [0, 1): row r's for the draft after
    it, a sequence's last row's for the chosen token; temperature float32 [seqs] (None: 1; <= 0: greedy); draft_probs
    float32 [rows, vocab], row r what the token after row r was drawn from (None: drafts without chance).
    Returns (token after each row or -1 [rows] int32, tokens per sequence [seqs] int32, log-probabilities [rows]);
    `out` gives those three buffers."""
    dev = _on("verify", logits)
    _need(logits.dim() == 2 and seq_rows.numel() > 0, "verify: logits [rows, vocab], seq_rows [seqs + 1]")
    ty, f32, i32 = logits.dtype, torch.float32, torch.int32
    n, v = logits.shape
    seqs = seq_rows.numel() - 1
    _need(ty in TYPES, f"verify: type must be float32, float16 or bfloat16, got {ty}")
    if out is None:
        out = tuple(_new("verify", *w, dev, stream) for w in ((n, i32), (seqs, i32), (n, f32)))
    tok, cnt, lp = out
    lst = logits.stride()
    pst = (0, 1) if draft_probs is None else draft_probs.stride()
    rows, per = (n,), (seqs,)
    if not (tokens.dtype is i32 and seq_rows.dtype is i32 and u.dtype is f32 and tok.dtype is i32 and cnt.dtype is i32 and
            lp.dtype is f32 and tokens.shape == rows and seq_rows.dim() == 1 and u.shape == rows and tok.shape == rows and
            cnt.shape == per and lp.shape == rows and
            dev == tokens.get_device() == seq_rows.get_device() == u.get_device() == tok.get_device() ==
            cnt.get_device() == lp.get_device() and
            (temperature is None or (temperature.dtype is f32 and temperature.shape == per and
                                     temperature.get_device() == dev and temperature.is_contiguous())) and
            (draft_probs is None or (draft_probs.dtype is f32 and draft_probs.shape == (n, v) and
                                     draft_probs.get_device() == dev)) and
            lst[1] == pst[1] == 1 and tokens.is_contiguous() and seq_rows.is_contiguous() and u.is_contiguous() and
            tok.is_contiguous() and cnt.is_contiguous() and lp.is_contiguous()):
        want = (("logits", logits, ty, (n, v), (None, 1)), ("tokens", tokens, i32, rows, (1,)),
                ("seq_rows", seq_rows, i32, (seqs + 1,), (1,)), ("u", u, f32, rows, (1,)),
                ("temperature", temperature, f32, per, (1,)), ("draft_probs", draft_probs, f32, (n, v), (None, 1)),
                ("out tokens", tok, i32, rows, (1,)), ("out counts", cnt, i32, per, (1,)),
                ("out logprobs", lp, f32, rows, (1,)))
        if not all(t is None or (t.dtype is d and t.shape == s and t.get_device() == dev and _laid(t, w))
                   for _, t, d, s, w in want):
            _refuse("verify", dev, want)
    ref = C.byref(_lib.VerifyDesc(TYPES[ty], seqs, n, v, lst[0], pst[0]))
    L = _lib.lib()
    _run("verify", L.loom_cuda_verify, L.loom_cuda_verify_workspace, ref,
         (logits.data_ptr(), None if draft_probs is None else draft_probs.data_ptr(), tokens.data_ptr(),
          seq_rows.data_ptr(), u.data_ptr(), None if temperature is None else temperature.data_ptr(), tok.data_ptr(),
          cnt.data_ptr(), lp.data_ptr()), dev, stream)
    return out
