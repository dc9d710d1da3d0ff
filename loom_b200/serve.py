"""Operators of one batched serving step (include/loom_cuda.h, "batched
serving"): attention of sequences that share a prompt, low-rank adapters of many
requests, verification of drafted tokens.

All three share one row layout: the rows of sequence b are seq_rows[b] ..
seq_rows[b + 1] - 1 (cuda int32 [n_seqs + 1]): its last accepted token, then its
drafts. Buffers are torch cuda tensors; arguments of a wrong type, shape or
layout raise LoomCudaError before anything runs. A call runs on `stream` (a
cudaStream_t), or torch's current stream, and only launches: it can be captured
in a CUDA graph.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from ._lib import LoomCudaError

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


def _need(ok: bool, why: str) -> None:
    if not ok:
        raise LoomCudaError(why)


def _typed(op: str, name: str, t, dtype, shape, like, dense: bool = True) -> None:
    """t is a tensor of this dtype and shape on like's device (dense: contiguous)."""
    if t.dtype is not dtype or t.shape != shape or t.device != like.device or (dense and not t.is_contiguous()):
        raise LoomCudaError(f"{op}: {name} must be {'a contiguous ' if dense else ''}{dtype} {tuple(shape)} on "
                            f"{like.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


_device = None  # the device the backend was brought up on by a call here


def _on(op: str, t) -> None:
    global _device
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{op}: tensors must be on a cuda device")
    if t.device != _device:  # bring-up, or the refusal of a second device
        _lib.must(_lib.lib().loom_cuda_init(t.device.index), op)
        _device = t.device
    _need(t.dtype in TYPES, f"{op}: type must be float32, float16 or bfloat16, got {t.dtype}")


def _stream(stream, like):
    cur = torch.cuda.current_stream(like.device).cuda_stream
    return cur if stream is None else stream, cur


def _workspace(n: int, like, stream: int, cur: int):
    """Scratch from torch's allocator, kept from reuse until the call's stream is done with it."""
    ws = torch.empty(n, dtype=torch.uint8, device=like.device)
    if stream != cur and n:
        ws.record_stream(torch.cuda.ExternalStream(stream, device=like.device))
    return ws


def attn_shared(q, prefix_k, prefix_v, own_k, own_v, seq_rows, seq_len, scale: float, out=None,
                stream: Optional[int] = None):
    """Attention over a shared prefix cache and each sequence's own cache.

    q [rows, heads, hd]; prefix_k/v [prefix, kv_heads, hd]; own_k/v [seqs, cap, kv_heads, hd], all of one type
    (float32, float16, bfloat16), any strides but a last dimension of 1 (q, out: heads side by side). seq_len (cuda
    int32 [seqs]) counts each sequence's own positions, this step's rows included: row j of n sees seq_len - (n - 1 - j)
    of them. Returns out [rows, heads, hd]."""
    _on("attn_shared", q)
    n, h, hd = q.shape if q.dim() == 3 else (0, 0, 0)
    _need(h > 0 and hd > 0 and own_k.dim() == 4 and prefix_k.dim() == 3,
          "attn_shared: q [rows, heads, hd], prefix_k/v [prefix, kv, hd], own_k/v [seqs, cap, kv, hd]")
    seqs, cap, kv, _ = own_k.shape
    pre = prefix_k.shape[0]
    ty, pst, ost = q.dtype, prefix_k.stride(), own_k.stride()
    _typed("attn_shared", "prefix_k", prefix_k, ty, (pre, kv, hd), q, False)
    _typed("attn_shared", "prefix_v", prefix_v, ty, (pre, kv, hd), q, False)
    _typed("attn_shared", "own_k", own_k, ty, (seqs, cap, kv, hd), q, False)
    _typed("attn_shared", "own_v", own_v, ty, (seqs, cap, kv, hd), q, False)
    _typed("attn_shared", "seq_rows", seq_rows, torch.int32, (seqs + 1,), q)
    _typed("attn_shared", "seq_len", seq_len, torch.int32, (seqs,), q)
    if out is None:
        out = torch.empty((n, h, hd), dtype=ty, device=q.device)
    _typed("attn_shared", "out", out, ty, (n, h, hd), q, False)
    qst, dst = q.stride(), out.stride()
    _need(prefix_v.stride() == pst and own_v.stride() == ost, "attn_shared: keys and values must be laid out alike")
    _need((pst[2] == 1 or hd == 1) and (ost[3] == 1 or hd == 1) and (qst[2] == 1 or hd == 1) and (dst[2] == 1 or hd == 1)
          and (qst[1] == hd or h == 1) and (dst[1] == hd or h == 1),
          "attn_shared: the last dimension must be contiguous, and the heads of q and out side by side")
    d = _lib.AttnSharedDesc(TYPES[ty], scale, seqs, n, h, kv, hd, qst[0], dst[0], pre, pst[0], pst[1], cap, ost[1],
                            ost[2], ost[0])
    L, (st, cur) = _lib.lib(), _stream(stream, q)
    ref = C.byref(d)
    ws = _workspace(L.loom_cuda_attn_shared_workspace(ref), q, st, cur)
    _lib.must(L.loom_cuda_attn_shared(ref, q.data_ptr(), prefix_k.data_ptr(), prefix_v.data_ptr(), own_k.data_ptr(),
                                      own_v.data_ptr(), seq_rows.data_ptr(), seq_len.data_ptr(), out.data_ptr(),
                                      ws.data_ptr(), ws.numel(), st), "attn_shared")
    return out


def lora(x, a, b, ranks, scales, ids, base=None, out=None, stream: Optional[int] = None):
    """out = base + scales[id] * B[id] (A[id] x) row by row; rows whose id names no adapter keep their base.

    x [rows, n_in] float32; a [adapters, max_rank, n_in], b [adapters, n_out, max_rank] of one type (float32, float16,
    bfloat16); ranks (int32) and scales (float32) [adapters]; ids int32 [rows]; base, out [rows, n_out] float32 (base
    None: zeros; out may be base). Last dimensions contiguous. Returns out."""
    _on("lora", a)
    _need(a.dim() == 3 and b.dim() == 3 and x.dim() == 2, "lora: x [rows, n_in], a [n, rank, n_in], b [n, n_out, rank]")
    na, rank, nin = a.shape
    n, nout = x.shape[0], b.shape[1]
    f32 = torch.float32
    _typed("lora", "x", x, f32, (n, nin), a, False)
    _typed("lora", "b", b, a.dtype, (na, nout, rank), a, False)
    _typed("lora", "ranks", ranks, torch.int32, (na,), a)
    _typed("lora", "scales", scales, f32, (na,), a)
    _typed("lora", "ids", ids, torch.int32, (n,), a)
    if base is not None:
        _typed("lora", "base", base, f32, (n, nout), a, False)
    if out is None:
        out = torch.empty((n, nout), dtype=f32, device=a.device)
    _typed("lora", "out", out, f32, (n, nout), a, False)
    xst, ast, bst, dst = x.stride(), a.stride(), b.stride(), out.stride()
    cst = dst if base is None else base.stride()
    _need((xst[1] == 1 or nin == 1) and (ast[2] == 1 or nin == 1) and (bst[2] == 1 or rank == 1) and
          ((dst[1] == 1 and cst[1] == 1) or nout == 1), "lora: the last dimension must be contiguous")
    d = _lib.LoraDesc(TYPES[a.dtype], n, nin, nout, na, rank, xst[0], cst[0], dst[0], ast[1], ast[0], bst[1], bst[0])
    L, (st, cur) = _lib.lib(), _stream(stream, a)
    ref = C.byref(d)
    ws = _workspace(L.loom_cuda_lora_workspace(ref), a, st, cur)
    _lib.must(L.loom_cuda_lora(ref, x.data_ptr(), a.data_ptr(), b.data_ptr(), ranks.data_ptr(), scales.data_ptr(),
                               ids.data_ptr(), None if base is None else base.data_ptr(), out.data_ptr(),
                               ws.data_ptr(), ws.numel(), st), "lora")
    return out


def verify(logits, tokens, seq_rows, u, temperature=None, draft_probs=None, out=None, stream: Optional[int] = None):
    """Accept drafted tokens against the target's probabilities and choose the token after them.

    logits [rows, vocab] (float32, float16, bfloat16), row r for the token after row r; tokens int32 [rows] (row r's own
    token: the drafts are the rows after each sequence's first); u float32 [rows] in [0, 1): row r's for the draft after
    it, a sequence's last row's for the chosen token; temperature float32 [seqs] (None: 1; <= 0: greedy); draft_probs
    float32 [rows, vocab], row r what the token after row r was drawn from (None: drafts without chance).
    Returns (token after each row or -1 [rows] int32, tokens per sequence [seqs] int32, log-probabilities [rows]);
    `out` gives those three buffers."""
    _on("verify", logits)
    _need(logits.dim() == 2, "verify: logits must be [rows, vocab]")
    n, v = logits.shape
    seqs = seq_rows.numel() - 1
    _need(seqs >= 0, "verify: seq_rows must be [seqs + 1]")
    f32, i32 = torch.float32, torch.int32
    _typed("verify", "tokens", tokens, i32, (n,), logits)
    _typed("verify", "seq_rows", seq_rows, i32, (seqs + 1,), logits)
    _typed("verify", "u", u, f32, (n,), logits)
    if temperature is not None:
        _typed("verify", "temperature", temperature, f32, (seqs,), logits)
    if draft_probs is not None:
        _typed("verify", "draft_probs", draft_probs, f32, (n, v), logits, False)
        _need(draft_probs.stride(1) == 1 or v == 1, "verify: the last dimension must be contiguous")
    _need(logits.stride(1) == 1 or v == 1, "verify: the last dimension must be contiguous")
    if out is None:
        dev = logits.device
        out = (torch.empty(n, dtype=i32, device=dev), torch.empty(seqs, dtype=i32, device=dev),
               torch.empty(n, dtype=f32, device=dev))
    tok, cnt, lp = out
    _typed("verify", "out tokens", tok, i32, (n,), logits)
    _typed("verify", "out counts", cnt, i32, (seqs,), logits)
    _typed("verify", "out logprobs", lp, f32, (n,), logits)
    d = _lib.VerifyDesc(TYPES[logits.dtype], seqs, n, v, logits.stride(0),
                        0 if draft_probs is None else draft_probs.stride(0))
    L, (st, cur) = _lib.lib(), _stream(stream, logits)
    ref = C.byref(d)
    ws = _workspace(L.loom_cuda_verify_workspace(ref), logits, st, cur)
    _lib.must(L.loom_cuda_verify(ref, logits.data_ptr(), None if draft_probs is None else draft_probs.data_ptr(),
                                 tokens.data_ptr(), seq_rows.data_ptr(), u.data_ptr(),
                                 None if temperature is None else temperature.data_ptr(), tok.data_ptr(),
                                 cnt.data_ptr(), lp.data_ptr(), ws.data_ptr(), ws.numel(), st), "verify")
    return out
