"""Decode models with a 4-bit KV cache (kv_dtype KV_Q4), and the logits step
between their tokens."""
import numpy as np
import pytest

from tests import kv4_ref as ref
from tests import synth
from tests.test_gpu_decode import SHAPES, _build, _model

pytestmark = pytest.mark.gpu


def _pair(which, *kinds):
    from aljabr_b200 import native
    from aljabr_b200.decode import LlamaShape
    native.call("aljabr_blackwell_init", 0)
    shapes = [LlamaShape(**SHAPES[which], kv_dtype=k) for k in kinds]
    weights = _model(41, shapes[0])
    return shapes[0], [_build(s, *weights) for s in shapes]


@pytest.mark.parametrize("which", ["small", "wide"])
def test_cache_holds_the_quantised_rows(which):
    """Layer 0's K and V depend on token and position alone, so the 4-bit model's must be the fp32 model's,
    quantised; the models' logits differ by the cache's error only (d / 2 of each group: some percent)."""
    shape, (a, b) = _pair(which, 2, 0)
    try:
        n = 12
        for pos in range(n):
            _, la = a.step(7 * pos + 3, pos, want_logits=True)
            _, lb = b.step(7 * pos + 3, pos, want_logits=True)
            assert synth.normwise_rel_err(la, lb) < 0.2, pos
        _, ka, va = a.read_state()
        _, kb, vb = b.read_state()
        for got, full in ((ka, kb), (va, vb)):
            rows = full[0, :n].reshape(n, shape.kv_heads, shape.head_dim)
            want = ref.values(*ref.quantise(rows)).reshape(n, -1)
            assert np.array_equal(got[0, :n], want.astype(np.float32))
            assert (got[:, n:] == 0).all()
    finally:
        a.close()
        b.close()


def test_restored_cache_continues_alike():
    """Quantising values that come from the cache changes nothing, so a session read out and synced into another
    model decodes the same tokens."""
    shape, (a, b) = _pair("small", 2, 2)
    try:
        n = 9
        for pos in range(n):
            a.step(5 * pos + 1, pos)
        _, k, v = a.read_state()
        for l in range(shape.layers):
            b.sync_kv_cache(l, n, np.ascontiguousarray(k[l, :n]), np.ascontiguousarray(v[l, :n]))
        _, kb, vb = b.read_state()
        assert np.array_equal(kb, k) and np.array_equal(vb, v)
        _, la = a.step(77, n, want_logits=True)
        _, lb = b.step(77, n, want_logits=True)
        assert np.array_equal(la, lb)
        assert np.array_equal(a.run(5, n + 1, 8), b.run(5, n + 1, 8))
    finally:
        a.close()
        b.close()


def test_context_that_is_no_multiple_of_a_tile():
    """max_ctx 21: the cache is padded to 32 positions, the model still ends at 21."""
    from aljabr_b200 import native
    from aljabr_b200.decode import LlamaShape
    native.call("aljabr_blackwell_init", 0)
    shape = LlamaShape(**{**SHAPES["small"], "max_ctx": 21}, kv_dtype=2)
    weights = _model(43, shape)
    a, b = _build(shape, *weights), _build(shape, *weights)
    try:
        run = a.run(9, 0, 21)
        token = 9
        for pos in range(21):
            token, _ = b.step(token, pos)
            assert token == run[pos]
        _, ka, va = a.read_state()
        _, kb, vb = b.read_state()
        assert ka.shape[1] == 21 and np.array_equal(ka, kb) and np.array_equal(va, vb) and np.abs(ka[:, 20]).max() > 0
        with pytest.raises(native.ProviderError):
            a.step(1, 21)
    finally:
        a.close()
        b.close()


def test_generate_applies_the_rules():
    from tests.test_gpu_logits import reference
    shape, (a, b) = _pair("small", 2, 2)
    try:
        V = shape.vocab
        allowed = np.random.default_rng(0).random(V) < 0.5
        words = np.packbits(allowed.astype(np.uint8), bitorder="little").view(np.uint32)
        rules = dict(penalties=(1.3, 0.2, 0.1), bias={5: 1.5, 9: -2.0})
        got = a.generate(11, 0, 10, history=[3, 3, 8], allow=lambda emitted: words, **rules)
        token, seen, want = 11, [3, 3, 8, 11], []
        for pos in range(10):
            _, logits = b.step(token, pos, want_logits=True)
            _, token = reference(logits, seen, np.float32([1.3, 0.2, 0.1]), [(5, np.float32(1.5)), (9, np.float32(-2))],
                                 allowed, np.float32)
            seen.append(token)
            want.append(token)
        assert got.tolist() == want and all(allowed[t] for t in want)
        assert a.generate(11, 0, 5, allow=lambda e: words if len(e) < 2 else words * 0).tolist()[2:] == []
        plain = b.generate(11, 0, 6)
        assert np.array_equal(plain, a.run(11, 0, 6))
    finally:
        a.close()
        b.close()


def test_refusals():
    import ctypes
    from aljabr_b200 import native
    from aljabr_b200.decode import LlamaNf4Decoder, LlamaShape
    native.call("aljabr_blackwell_init", 0)
    with pytest.raises(native.UnsupportedOperation):
        LlamaNf4Decoder(LlamaShape(**SHAPES["small"], kv_dtype=3))
    with pytest.raises(native.UnsupportedOperation):
        LlamaNf4Decoder(LlamaShape(**SHAPES["small"], kv_dtype=2), tp_world=2, nccl_id=b"\0" * 128)
    dec = LlamaNf4Decoder(LlamaShape(**SHAPES["small"], kv_dtype=2))
    try:
        with pytest.raises(native.ProviderError):     # no step has run
            native.call("aljabr_blackwell_decode_logits", ctypes.c_ulonglong(dec.handle), ctypes.byref(ctypes.c_void_p()))
    finally:
        dec.close()
