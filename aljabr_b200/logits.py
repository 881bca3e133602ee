"""The logits step of a decode loop (aljabr_blackwell_logits_process_dev):
penalties for repeated tokens, biases, a grammar mask and the greedy token."""
from __future__ import annotations

import torch

from . import native
from .kv4 import bad, current_stream, dtype_id


def process_logits(logits: torch.Tensor, history=None, history_len=None, penalties=None, bias_tokens=None,
                   bias_values=None, bias_len=None, allow=None, out=None, token=None, stream=None):
    """Returns (processed logits fp32 [rows, vocab], greedy token int32 [rows]).

    logits: [rows, vocab] float32 or bfloat16 (rows may be strided); `out` may be `logits` itself.
    history: int32 [rows, n] with history_len [rows] live entries; penalties: fp32 [rows, 3] = repetition,
    frequency, presence (needed with a history).  bias_tokens int32 / bias_values fp32 [rows, n] with
    bias_len [rows].  allow: int32 [rows, >= ceil(vocab / 32)] words, bit t % 32 of word t / 32 allows token t.
    The formulas are in include/aljabr_blackwell.h."""
    if logits.dim() != 2 or logits.stride(1) != 1 or logits.device.type != "cuda":
        raise bad("logits must be a [rows, vocab] CUDA tensor with contiguous rows")
    rows, vocab = logits.shape
    dev = logits.device

    def ptr(t, dtype, shape, what):
        if t is None:
            return None
        if t.dtype != dtype or t.device != dev or not t.is_contiguous() or tuple(t.shape) != shape:
            raise bad(f"{what} must be contiguous {dtype} {shape} on {dev}")
        return t.data_ptr()

    def width(t):
        return 0 if t is None else t.shape[-1]

    if out is None:
        out = torch.empty(rows, vocab, dtype=torch.float32, device=dev)
    elif out.dtype != torch.float32 or out.shape != logits.shape or out.stride(1) != 1 or out.device != dev:
        raise bad(f"out must be float32 [{rows}, {vocab}] on {dev} with contiguous rows")
    if token is None:
        token = torch.empty(rows, dtype=torch.int32, device=dev)
    nh, nb, na = width(history), width(bias_tokens), width(allow)
    i32, f32 = torch.int32, torch.float32
    native.call("aljabr_blackwell_logits_process_dev", out.data_ptr(), out.stride(0) if rows > 1 else vocab,
                logits.data_ptr(), dtype_id(logits, "logits"), logits.stride(0) if rows > 1 else vocab, rows, vocab,
                ptr(history, i32, (rows, nh), "history"), ptr(history_len, i32, (rows,), "history_len"), nh,
                ptr(penalties, f32, (rows, 3), "penalties"), ptr(bias_tokens, i32, (rows, nb), "bias_tokens"),
                ptr(bias_values, f32, (rows, nb), "bias_values"), ptr(bias_len, i32, (rows,), "bias_len"), nb,
                ptr(allow, i32, (rows, na), "allow"), na, ptr(token, i32, (rows,), "token"),
                stream or current_stream(dev))
    return out, token
