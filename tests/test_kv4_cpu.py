"""Refusals of the 4-bit cache's and the logits step's entry points: every
argument is checked before the GPU is touched, so they run without one."""
import numpy as np
import pytest

from aljabr_b200 import native
from tests import kv4_ref as ref

P = 1 << 20      # a well-aligned address that is never followed


def rc(name, *args):
    return getattr(native.lib(), name)(*args)


def append(pages=4, ps=16, hkv=2, D=128, k=P, v=P, dt=native.KV_F32, ks=256, vs=256, slots=P, n=3, kb=None, vb=None, cache=P):
    return rc("aljabr_blackwell_kv4_append_dev", cache, pages, ps, hkv, D, k, v, dt, ks, vs, slots, n, kb, vb, None)


def read(k=P, v=P, dt=native.KV_F32, cache=P, pages=4, ps=16, hkv=2, D=128, slots=P, n=3):
    return rc("aljabr_blackwell_kv4_read_dev", k, v, dt, cache, pages, ps, hkv, D, slots, n, None)


def attend(out=P, q=P, dt=native.KV_F32, qs=1024, cache=P, pages=4, ps=16, hkv=2, D=128, table=P, width=4, lens=P, batch=2,
           T=1, hq=8, window=0, scale=0.1, cap=0.0, work=P, size=1 << 40):
    return rc("aljabr_blackwell_kv4_attention_dev", out, q, dt, qs, cache, pages, ps, hkv, D, table, width, lens, batch, T, hq,
              window, scale, cap, work, size, None)


def logits(out=P, os=100, x=P, dt=native.KV_F32, xs=100, rows=2, vocab=100, h=P, hl=P, hs=4, pen=P, bt=P, bv=P, bl=P, bs=4,
           allow=P, als=4, token=P):
    return rc("aljabr_blackwell_logits_process_dev", out, os, x, dt, xs, rows, vocab, h, hl, hs, pen, bt, bv, bl, bs, allow, als,
              token, None)


DIMS, UNSUP, ARG = native.ALJ_ERR_BAD_DIMS, native.ALJ_ERR_UNSUPPORTED, native.ALJ_ERR_BAD_ARG


@pytest.mark.parametrize("kw,code", [
    (dict(pages=0), DIMS), (dict(ps=0), DIMS), (dict(hkv=0), DIMS), (dict(D=-64), DIMS), (dict(pages=1 << 28), DIMS),
    (dict(D=96), UNSUP), (dict(D=512), UNSUP), (dict(ps=24), UNSUP), (dict(dt=2), UNSUP), (dict(n=-1), DIMS),
    (dict(cache=None), ARG), (dict(cache=P + 8), ARG), (dict(slots=None), ARG)])
def test_rows_refuse(kw, code):
    assert append(**kw) == code and native.last_error()
    assert read(**kw) == code


def test_append_and_read_refuse():
    assert append(k=None) == ARG and append(v=None) == ARG
    assert append(kb=P) == ARG and append(vb=P) == ARG and append(kb=P + 2, vb=P) == ARG
    assert append(ks=255) == DIMS and append(vs=0) == DIMS
    assert append(k=P + 2) == ARG and append(v=P + 1, dt=native.KV_BF16) == ARG
    assert read(k=None, v=None) == ARG
    assert append(n=0, k=None, slots=None) == native.ALJ_OK and read(n=0, k=None) == native.ALJ_OK


@pytest.mark.parametrize("kw,code", [
    (dict(D=80), UNSUP), (dict(ps=8), UNSUP), (dict(pages=0), DIMS), (dict(T=0), DIMS), (dict(hq=7), DIMS), (dict(hq=0), DIMS),
    (dict(T=257), UNSUP), (dict(dt=5), UNSUP), (dict(batch=-1), DIMS), (dict(batch=2049), DIMS), (dict(window=-1), ARG),
    (dict(cap=-1.0), ARG), (dict(cap=float("nan")), ARG), (dict(out=None), ARG), (dict(q=None), ARG), (dict(cache=None), ARG),
    (dict(lens=None), ARG), (dict(work=None), ARG), (dict(width=0), DIMS), (dict(table=None, batch=5), DIMS),
    (dict(qs=1023), DIMS), (dict(out=P + 8), ARG), (dict(q=P + 1, dt=native.KV_BF16), ARG), (dict(cache=P + 4), ARG)])
def test_attention_refuses(kw, code):
    assert attend(**kw) == code and native.last_error()


def test_attention_of_an_empty_batch_is_nothing():
    assert attend(batch=0, out=None, lens=None) == native.ALJ_OK


def test_sizes():
    size = native.lib().aljabr_blackwell_kv4_cache_size
    assert size(3, 48, 5, 128) == 3 * 48 * 5 * 144
    assert size(30000, 64, 8, 256) == 30000 * 64 * 8 * 288
    assert size(1, 16, 1, 100) == UNSUP
    work = native.lib().aljabr_blackwell_kv4_attention_workspace_size
    assert work(1, 32, 8, 128) > 0 and work(4, 32, 8, 128) > work(1, 32, 8, 128) and work(1, 9, 8, 128) == DIMS


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), DIMS), (dict(rows=65536), DIMS), (dict(vocab=0), DIMS), (dict(dt=3), UNSUP), (dict(os=99), DIMS),
    (dict(xs=99), DIMS), (dict(out=None), ARG), (dict(x=None), ARG), (dict(dt=native.KV_BF16), ARG),
    (dict(os=101), ARG), (dict(hl=None), ARG), (dict(pen=None), ARG), (dict(hs=0), ARG), (dict(bv=None), ARG),
    (dict(bl=None), ARG), (dict(bs=0), ARG), (dict(als=3), DIMS)])
def test_logits_refuse(kw, code):
    assert logits(**kw) == code and native.last_error()


def test_logits_of_no_rows_is_nothing():
    assert logits(rows=0, out=None) == native.ALJ_OK


def test_reference_layout_round_trip():
    """The plain layout the GPU tests compare bytes with: every nibble has one place."""
    c = ref.RefCache(1, 16, 1, 64)
    x = np.linspace(-8, 7, 64).astype(np.float32)
    c.write(3, 0, x, -x)
    used = np.flatnonzero(c.data)
    assert used.min() >= 3 * 32 and used.max() < c.block
    codes, d = ref.quantise(x)
    assert np.abs(ref.values(codes, d) - x).max() <= np.abs(d.astype(np.float64)).max()
