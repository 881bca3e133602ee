"""What the decode wrapper takes and refuses before the library sees an
address: the library's calls are stubs, no GPU."""
import ctypes

import numpy as np
import pytest

from aljabr_b200 import decode, native


def decoder(monkeypatch, kv_dtype):
    """A one-layer model of 2 kv heads x 64, and the calls it makes."""
    d = object.__new__(decode.LlamaNf4Decoder)
    d.shape = decode.LlamaShape(1, 256, 4, 2, 64, 512, 1000, 32, kv_dtype=kv_dtype)
    d.tp_world, d.tp_rank, d.handle = 1, 0, 1
    calls = []
    monkeypatch.setattr(native, "call", lambda name, *a: calls.append((name, a)))
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(torch.cuda, "set_device", lambda index: None)
    return d, calls


@pytest.mark.parametrize("kv_dtype,good,wrong", [
    (native.KV_Q4, [np.float32], [np.uint16, np.float16, np.float64]),
    (native.KV_F32, [np.float32], [np.uint16, np.float64]),
    (native.KV_BF16, [np.uint16, np.int16], [np.float32, np.float16])])
def test_cache_rows_of_another_type_are_refused(monkeypatch, kv_dtype, good, wrong):
    """The library reads 4 (or 2) bytes an element from the address it is given."""
    d, calls = decoder(monkeypatch, kv_dtype)
    for t in good:
        rows = np.zeros((7, 128), t)
        d.sync_kv_cache(0, 7, rows, rows)
        d.sync_kv_cache(0, 5, rows, rows)                     # the first rows of a longer buffer
    d.sync_kv_cache(0, 7, 1 << 20, 1 << 20)                   # an address is the caller's own word
    assert len(calls) == 2 * len(good) + 1
    ok = np.zeros((7, 128), good[0])
    for t in wrong:
        bad = np.zeros((7, 128), t)
        for k, v in ((bad, bad), (ok, bad), (bad, ok)):
            with pytest.raises(native.ProviderError):
                d.sync_kv_cache(0, 7, k, v)
    with pytest.raises(native.ProviderError):
        d.sync_kv_cache(0, 8, ok, ok)                         # fewer rows than it says
    assert len(calls) == 2 * len(good) + 1


def test_cache_rows_as_tensors(monkeypatch):
    torch = pytest.importorskip("torch")
    for kv_dtype, good, wrong in ((native.KV_Q4, torch.float32, torch.bfloat16), (native.KV_BF16, torch.bfloat16, torch.float32),
                                  (native.KV_BF16, torch.int16, torch.half)):
        d, calls = decoder(monkeypatch, kv_dtype)
        rows = torch.zeros(3, 128, dtype=good)
        d.sync_kv_cache(0, 3, rows, rows)
        for bad in (rows.to(wrong), torch.zeros(128, 3, dtype=good).t(), rows[:2]):
            with pytest.raises(native.ProviderError):
                d.sync_kv_cache(0, 3, bad, bad)
        assert len(calls) == 1 and calls[0][1][3].value == rows.data_ptr()


def test_strided_arrays_are_copied_and_outlive_the_call(monkeypatch):
    d, _ = decoder(monkeypatch, native.KV_Q4)
    k = np.arange(2 * 7 * 128, dtype=np.float32).reshape(7, 256)[:, 128:]
    v = np.arange(2 * 7 * 128, dtype=np.float32).reshape(7, 2, 128)[:, 0] + 0.5
    seen = []

    def call(name, handle, layer, n, kp, vp):
        other = [np.full(7 * 128, -1.0, np.float32) for _ in range(64)]     # what would take a freed copy's place
        for p in (kp, vp):
            seen.append(np.ctypeslib.as_array(ctypes.cast(p, ctypes.POINTER(ctypes.c_float)), (7, 128)).copy())
        assert len(other) == 64
    monkeypatch.setattr(native, "call", call)
    d.sync_kv_cache(0, 7, k, v)
    assert np.array_equal(seen[0], k) and np.array_equal(seen[1], v)


@pytest.mark.parametrize("penalties", [(1.1,), (1.1, 0.0), (1.0, 0.0, 0.0, 0.0), [(1.0, 0.0, 0.0)]])
def test_generate_takes_three_penalties(monkeypatch, penalties):
    """The library reads three numbers from the address it is given."""
    torch = pytest.importorskip("torch")
    d, calls = decoder(monkeypatch, native.KV_Q4)
    real = torch.device
    monkeypatch.setattr(torch, "device", lambda *a: real("cpu"))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    d.step = lambda token, pos: calls.append(("step", (token, pos)))
    with pytest.raises(native.ProviderError):
        d.generate(3, 0, 2, penalties=penalties)
    assert calls == []


def test_a_grammar_may_allow_everything_for_a_token(monkeypatch):
    """`allow` gives words, or None where the grammar says nothing about the next token."""
    torch = pytest.importorskip("torch")
    d, _ = decoder(monkeypatch, native.KV_Q4)
    real, masks = torch.device, []
    monkeypatch.setattr(torch, "device", lambda *a: real("cpu"))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    from aljabr_b200 import kv4
    monkeypatch.setattr(kv4, "current_stream", lambda index: 1)
    monkeypatch.setattr(native, "call", lambda name, *a: masks.append((a[15], a[16])) if "logits_process" in name else None)
    d.step = lambda token, pos: None
    words = np.full((1000 + 31) // 32, 0xFFFFFFFF, np.uint32)
    monkeypatch.setattr(torch.Tensor, "__int__", lambda t: 5)
    got = d.generate(3, 0, 3, allow=lambda emitted: words if len(emitted) == 1 else None)
    assert got.tolist() == [5, 5, 5] and [m[1] for m in masks] == [0, 32, 0] and masks[0][0] is None and masks[2][0] is None


def test_generate_runs_on_the_model_s_device(monkeypatch):
    """Two models on two GPUs: the thread's device is the last one's.  The logits step of the other must be launched, and
    its tensors made, where that model is; afterwards the thread's choice is as before."""
    torch = pytest.importorskip("torch")
    d, _ = decoder(monkeypatch, native.KV_Q4)
    real, state, seen = torch.device, {"cuda": 1, "library": 1}, []

    def call(name, *a):
        if name == "aljabr_blackwell_decode_device":
            a[1]._obj.value = 0
        elif name == "aljabr_blackwell_device_swap":
            a[1]._obj.value, state["library"] = state["library"], a[0]
            if a[0] >= 0:
                state["cuda"] = a[0]
        elif "logits_process" in name:
            seen.append(dict(state))

    def step(token, pos):
        state["cuda"] = 0                     # as the library leaves it
    made = []
    monkeypatch.setattr(native, "call", call)
    monkeypatch.setattr(torch, "device", lambda kind, index: made.append(index) or real("cpu"))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["cuda"])
    monkeypatch.setattr(torch.cuda, "set_device", lambda i: state.update(cuda=i))
    from aljabr_b200 import kv4
    monkeypatch.setattr(kv4, "current_stream", lambda index: 1)
    monkeypatch.setattr(torch.Tensor, "__int__", lambda t: 5)
    d.step = step
    d.generate(3, 0, 2)
    assert made == [0] and seen == [{"cuda": 0, "library": 0}] * 2 and state == {"cuda": 1, "library": 1}
