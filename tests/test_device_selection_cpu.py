"""With several GPUs a wrapper's call selects its tensors' device; afterwards the caller's own choice, torch's and the
library's, is as before.  The library and torch's device are stubs."""
import importlib

import pytest

torch = pytest.importorskip("torch")

from aljabr_b200 import kv4, logits, native


@pytest.fixture
def devices(monkeypatch):
    """{'cuda': device of the thread, 'library': device selected in the library or -1, 'at': devices of the calls}"""
    d = {"cuda": 0, "library": -1, "at": []}

    def call(name, *a):
        if name == "aljabr_blackwell_init":
            d["cuda"] = d["library"] = a[0]
        elif name == "aljabr_blackwell_device_swap":
            a[1]._obj.value, d["library"] = d["library"], a[0]
            if a[0] >= 0:
                d["cuda"] = a[0]
        return 0
    monkeypatch.setattr(native, "call", call)
    monkeypatch.setattr(torch.cuda, "device_count", lambda: 2)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: d["cuda"])
    monkeypatch.setattr(torch.cuda, "set_device", lambda i: d.update(cuda=i))
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 1)
    importlib.reload(kv4), importlib.reload(logits)
    monkeypatch.setattr(kv4, "current_stream", lambda index: 1)
    monkeypatch.setattr(logits, "current_stream", lambda index: 1)
    yield d
    monkeypatch.undo()
    importlib.reload(kv4), importlib.reload(logits)


def cache_on_1(d):
    c = object.__new__(kv4.Kv4Cache)
    c.kv_heads, c.head_dim, c.device, c._index, c._row = 2, 64, torch.device("cpu"), 1, 128
    c._shape, c._buffers, c._work = (0, 4, 16, 2, 64), {}, {}
    c._work_size = lambda *a: 1024

    def entry(*a):
        d["at"].append((d["cuda"], d["library"]))
        return 0
    c._append = c._read = c._attend = entry
    return c, entry


@pytest.mark.parametrize("cuda,library", [(0, -1), (0, 0), (0, 1), (1, 0)])
def test_calls_leave_the_device_as_it_was(devices, monkeypatch, cuda, library):
    c, entry = cache_on_1(devices)
    monkeypatch.setattr(logits, "_process", entry)
    k, slots = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32)
    q, one, table = torch.zeros(1, 1, 2, 64), torch.ones(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    x = torch.zeros(2, 33)
    for call in (lambda: c.append(k, k, slots), lambda: c.read(slots, k_out=k), lambda: c.attend(q, one, table, out=q),
                 lambda: logits.process_logits(logits=x, out=x, token=one.expand(2).contiguous())):
        devices.update(cuda=cuda, library=library, at=[])
        call()
        assert devices == {"cuda": cuda, "library": library, "at": [(1, 1)]}
    for call in (lambda: c.append(k, k[:2], slots), lambda: logits.process_logits(x, out=k)):     # refusals too
        devices.update(cuda=cuda, library=library, at=[])
        with pytest.raises(native.ProviderError):
            call()
        assert devices == {"cuda": cuda, "library": library, "at": []}


def test_making_a_cache_leaves_the_device_as_it_was(devices, monkeypatch):
    class Data:
        dtype, device = torch.uint8, torch.device("cuda", 1)
        is_contiguous, numel, data_ptr, get_device = (lambda s: True), (lambda s: 1 << 30), (lambda s: 4096), (lambda s: 1)
    kv4.Kv4Cache(4, 16, 2, 64, data=Data())
    assert devices["cuda"] == 0 and devices["library"] == -1
