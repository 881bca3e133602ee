"""Host-side state of the tensor wrappers, without a GPU: the library's calls
and torch's streams are stubs, the tensors live on the CPU."""
import gc
import weakref
from contextlib import contextmanager

import pytest

torch = pytest.importorskip("torch")

from aljabr_b200 import kv4


@pytest.fixture
def cache(monkeypatch):
    """A Kv4Cache of 2 x 64 whose workspace needs 1024 bytes up to 8 rows a kv head, 2048 above."""
    c = object.__new__(kv4.Kv4Cache)
    c.pages, c.page_size, c.kv_heads, c.head_dim = 4, 16, 2, 64
    c.device, c._index, c._row = torch.device("cpu"), -1, 128
    c.data = torch.zeros(4 * 16 * 2 * 72, dtype=torch.uint8)
    c._shape = (c.data.data_ptr(), 4, 16, 2, 64)
    c._buffers, c._work = {}, {}
    c._work_size = lambda q_len, q_heads, kv_heads, head_dim: 1024 if q_len * q_heads // kv_heads <= 8 else 2048
    c._append = c._read = c._attend = lambda *a: 0
    monkeypatch.setattr(kv4, "current_stream", lambda index: 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda s, device=None: s)

    @contextmanager
    def switch(s):
        c.at.append(s)
        yield
        c.at.pop()
    c.at = [7]           # torch's current stream, as its context managers set it
    monkeypatch.setattr(torch.cuda, "stream", switch)
    return c


def test_a_workspace_is_never_given_up(cache):
    """A graph captured with one query token keeps its workspace's address: a later call with more rows must leave it."""
    first, size = cache._workspace(1, 8, 7)
    alive = weakref.ref(cache._buffers[7])
    assert size >= 1024
    second, size = cache._workspace(5, 8, 7)
    gc.collect()
    assert size >= 2048 and alive() is not None and alive().data_ptr() == first
    assert cache._workspace(1, 8, 7)[0] == first


@pytest.mark.parametrize("D", [64, 128, 256])
def test_no_accepted_call_needs_more_than_the_most_rows(D):
    from aljabr_b200 import native
    size = native.lib().aljabr_blackwell_kv4_attention_workspace_size
    most = size(native.KV4_MAX_ROWS, 2, 2, D)
    assert all(size(rows, 2, 2, D) <= most for rows in range(1, native.KV4_MAX_ROWS))
    assert size(native.KV4_MAX_ROWS + 1, 2, 2, D) == native.ALJ_ERR_UNSUPPORTED


def attend(cache, stream=None, rows=1):
    """The workspace address that a call of the wrapper hands to the library."""
    got = []
    cache._attend = lambda *a: got.append(a[-3]) or 0
    q = torch.zeros(1, rows, 2, 64)
    cache.attend(q, torch.ones(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32), out=q, stream=stream)
    return got[0]


def test_each_capture_has_a_workspace_of_its_own(cache, monkeypatch):
    """Two graphs captured one after the other on one stream, and calls before, between and after them: a buffer whose
    zeroing is a node of one graph must serve nothing else, and no graph the buffer of plain calls."""
    capture = 0
    monkeypatch.setattr(kv4, "capture_id", lambda stream: capture, raising=False)
    capture = 11
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capture != 0)
    first = attend(cache)
    assert attend(cache) == first                       # calls of one stream in one graph follow one another
    other_branch = attend(cache, stream=8)
    capture = 0
    plain = attend(cache)
    kept = dict(cache._buffers)
    capture = 12
    second = attend(cache)
    assert attend(cache) == second and second != plain
    capture = 0
    assert attend(cache) == plain and cache._buffers == kept
    assert plain not in (first, other_branch) and first != other_branch
    assert len(cache._buffers) == 1


def test_outputs_belong_to_the_stream_that_writes_them(cache, monkeypatch):
    """With `stream` given, an output from the allocator's pool of torch's current stream could be a block whose last
    reader there has not run yet; and its own readers there must keep it from being handed out again."""
    at, made, readers = [7], [], []
    real = torch.empty

    @contextmanager
    def switch(s):
        at.append(s)
        yield
        at.pop()

    def empty(*a, **kw):
        made.append(at[-1])
        return real(*a, **kw)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda s, device=None: s)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: at[-1])
    monkeypatch.setattr(torch.cuda, "stream", switch)
    monkeypatch.setattr(torch, "empty", empty)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: readers.append(s))
    monkeypatch.setattr(kv4, "capture_id", lambda stream: 0)
    q, lens, slots = torch.zeros(1, 1, 2, 64), torch.ones(1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    table = torch.zeros(1, 1, dtype=torch.int32)
    cache.attend(q, lens, table)
    cache.read(slots)
    assert made == [7, 7, 7] and readers == []
    made.clear()
    cache.attend(q, lens, table, stream=9)
    cache.read(slots, stream=9)
    assert made == [9, 9, 9] and readers == [7, 7, 7]
    from aljabr_b200 import logits
    monkeypatch.setattr(logits, "_process", lambda *a: 0)
    monkeypatch.setattr(logits, "current_stream", lambda index: 7)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    made.clear(), readers.clear()
    logits.process_logits(torch.zeros(2, 33))
    assert made == [7, 7] and readers == []
    logits.process_logits(torch.zeros(2, 33), stream=9)
    assert made == [7, 7, 9, 9] and readers == [7, 7]


@pytest.mark.parametrize("window,passed", [(0, 0), (7, 7), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1),
                                           (2 ** 32 + 5, 2 ** 31 - 1), (2 ** 63 - 1, 2 ** 31 - 1), (-1, -1), (-2 ** 32, None)])
def test_a_window_that_an_int_does_not_hold(cache, monkeypatch, window, passed):
    """ctypes would cut it to its low 32 bits: 2^32 + 5 to a window of 5.  Longer than any sequence is no window."""
    from aljabr_b200 import native
    got = []
    cache._attend = lambda *a: got.append(a[-6]) or 0
    q = torch.zeros(1, 1, 2, 64)
    args = q, torch.ones(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    monkeypatch.setattr(kv4, "capture_id", lambda stream: 0)
    import ctypes
    cache.attend(*args, window=window, out=q)
    sent = ctypes.c_int(got[0]).value
    assert sent == passed if passed is not None else sent < 0


def test_the_legacy_stream_s_outputs_come_from_the_default_stream_s_pool(cache, monkeypatch):
    """Handle 1 names the legacy stream; torch takes an odd number for one of its own streams, not for a handle."""
    asked = []

    class Nothing:
        __enter__ = __exit__ = lambda *a: None
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda s, device=None: asked.append(s))
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: asked.append("default"))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: None)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: Nothing())
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: None)
    cache.read(torch.zeros(3, dtype=torch.int32), stream=1)
    cache.read(torch.zeros(3, dtype=torch.int32), stream=0x7f00)
    assert asked == ["default"] * 2 + [0x7f00] * 2


@pytest.mark.parametrize("capture", [0, 31])
def test_a_workspace_is_zeroed_on_the_stream_that_uses_it(cache, monkeypatch, capture):
    """In a capture, zeroing on another stream is a node of no graph or of an unordered branch; outside, a wait for the
    whole device would be needed."""
    zeroed, waits, real = [], [], torch.zeros
    monkeypatch.setattr(kv4, "capture_id", lambda stream: capture)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capture != 0)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: waits.append(1))
    monkeypatch.setattr(torch, "zeros", lambda *a, **kw: (zeroed.append(cache.at[-1]) if kw.get("dtype") is torch.uint8 else None,
                                                          real(*a, **kw))[1])
    kv4._captured.clear()
    attend(cache)
    attend(cache, stream=8)
    assert zeroed == [7, 8] and waits == []


def test_a_capture_named_by_its_stream_keeps_its_workspace(cache, monkeypatch):
    """A stream given by handle may be captured by other means than torch's, whose graphs keep their memory."""
    capture = 41
    monkeypatch.setattr(kv4, "capture_id", lambda stream: capture)
    kv4._captured.clear()
    first = attend(cache, stream=8)
    held = [weakref.ref(t) for t in kv4._captured[-1, 8][1]]
    capture = 42
    assert attend(cache, stream=8) != first
    gc.collect()
    assert held and all(t() is not None for t in held)
