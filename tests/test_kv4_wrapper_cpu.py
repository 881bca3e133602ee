"""Host-side state of the tensor wrappers, without a GPU: the library's calls
and torch's streams are stubs, the tensors live on the CPU."""
import gc
import weakref

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
