"""The logits step of a decode loop (aljabr_blackwell_logits_process_dev):
penalties for repeated tokens, biases, a grammar mask and the greedy token."""
from __future__ import annotations

import torch

from . import native
from .kv4 import bad, current_stream, dtype_id, new_output, selecting


_process = native.lib().aljabr_blackwell_logits_process_dev
_I32, _F32 = torch.int32, torch.float32


def _ptr(t, dtype, count, dev, what):
    if t.dtype is not dtype or t.numel() != count or t.get_device() != dev or not t.is_contiguous():
        raise bad(f"{what} must be {count} contiguous {dtype} on device {dev}, not {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


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
    stream = stream or current_stream(dev)
    if out is None:
        out = new_output((rows, vocab), torch.float32, logits.device, dev, stream)
    elif out.dtype is not torch.float32 or out.shape != shape or out.stride(1) != 1 or out.get_device() != dev:
        raise bad(f"out must be float32 [{rows}, {vocab}] on {logits.device} with contiguous rows")
    if token is None:
        token = new_output((rows,), torch.int32, logits.device, dev, stream)
    h = hl = pen = bt = bv = bl = al = None
    nh = nb = na = 0
    if history is not None:
        if history_len is None or penalties is None or penalties.shape[-1] != 3:
            raise bad("a history needs history_len [rows] and penalties [rows, 3]")
        nh = history.shape[-1]
        h, hl = _ptr(history, _I32, rows * nh, dev, "history"), _ptr(history_len, _I32, rows, dev, "history_len")
        pen = _ptr(penalties, _F32, rows * 3, dev, "penalties")
    if bias_tokens is not None:
        if bias_values is None or bias_len is None:
            raise bad("bias_tokens needs bias_values and bias_len")
        nb = bias_tokens.shape[-1]
        bt, bv = _ptr(bias_tokens, _I32, rows * nb, dev, "bias_tokens"), _ptr(bias_values, _F32, rows * nb, dev, "bias_values")
        bl = _ptr(bias_len, _I32, rows, dev, "bias_len")
    if allow is not None:
        na = allow.shape[-1]
        al = _ptr(allow, _I32, rows * na, dev, "allow")
    rc = _process(out.data_ptr(), out.stride(0) if rows > 1 else vocab, logits.data_ptr(), dtype_id(logits, "logits"),
                  st[0] if rows > 1 else vocab, rows, vocab, h, hl, nh, pen, bt, bv, bl, nb, al, na,
                  _ptr(token, _I32, rows, dev, "token"), stream)
    if rc:
        native.check(rc)
    return out, token


process_logits = selecting(process_logits, lambda logits, *_, **__: logits.get_device())
