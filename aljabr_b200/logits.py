"""The logits step of a decode loop (aljabr_blackwell_logits_process_dev):
penalties for repeated tokens, biases, a grammar mask and the greedy token."""
from __future__ import annotations

import torch

from . import native
from .kv4 import bad, current_stream, dtype_id, select_device


def process_logits(logits: torch.Tensor, history=None, history_len=None, penalties=None, bias_tokens=None,
                   bias_values=None, bias_len=None, allow=None, out=None, token=None, stream=None):
    """Returns (processed logits fp32 [rows, vocab], greedy token int32 [rows]).

    logits: [rows, vocab] float32 or bfloat16 (rows may be strided); `out` may be `logits` itself.
    history: int32 [rows, n] with history_len [rows] live entries; penalties: fp32 [rows, 3] = repetition,
    frequency, presence (needed with a history).  bias_tokens int32 / bias_values fp32 [rows, n] with
    bias_len [rows].  allow: int32 [rows, >= ceil(vocab / 32)] words, bit t % 32 of word t / 32 allows token t.
    The formulas are in include/aljabr_blackwell.h."""
    shape, st, dev = logits.shape, logits.stride(), logits.get_device()
    if len(shape) != 2 or st[1] != 1 or dev < 0:
        raise bad("logits must be a [rows, vocab] CUDA tensor with contiguous rows")
    rows, vocab = shape
    select_device(dev)

    def ptr(t, dtype, shape, what):
        if t is None:
            return None
        if t.dtype is not dtype or t.get_device() != dev or t.shape != shape or not t.is_contiguous():
            raise bad(f"{what} must be contiguous {dtype} {shape} on {logits.device}")
        return t.data_ptr()

    if out is None:
        out = torch.empty(rows, vocab, dtype=torch.float32, device=logits.device)
    elif out.dtype is not torch.float32 or out.shape != shape or out.stride(1) != 1 or out.get_device() != dev:
        raise bad(f"out must be float32 [{rows}, {vocab}] on {logits.device} with contiguous rows")
    if token is None:
        token = torch.empty(rows, dtype=torch.int32, device=logits.device)
    nh = 0 if history is None else history.shape[-1]
    nb = 0 if bias_tokens is None else bias_tokens.shape[-1]
    na = 0 if allow is None else allow.shape[-1]
    i32, f32 = torch.int32, torch.float32
    rc = native.lib().aljabr_blackwell_logits_process_dev(
        out.data_ptr(), out.stride(0) if rows > 1 else vocab, logits.data_ptr(), dtype_id(logits, "logits"),
        st[0] if rows > 1 else vocab, rows, vocab, ptr(history, i32, (rows, nh), "history"),
        ptr(history_len, i32, (rows,), "history_len"), nh, ptr(penalties, f32, (rows, 3), "penalties"),
        ptr(bias_tokens, i32, (rows, nb), "bias_tokens"), ptr(bias_values, f32, (rows, nb), "bias_values"),
        ptr(bias_len, i32, (rows,), "bias_len"), nb, ptr(allow, i32, (rows, na), "allow"), na,
        ptr(token, i32, (rows,), "token"), stream or current_stream(dev))
    if rc:
        native.check(rc)
    return out, token
