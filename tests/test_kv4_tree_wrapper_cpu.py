"""Host-side state of the tree wrappers, without a GPU (the stubs of
test_kv4_wrapper_cpu.py)."""
import gc
import threading
import time
import weakref

import pytest

torch = pytest.importorskip("torch")

from aljabr_b200 import kv4, native
from tests.test_kv4_wrapper_cpu import cache  # noqa: F401


@pytest.mark.parametrize("tree", [True, False])
def test_threads_that_meet_at_a_stream_s_first_call_use_one_workspace(cache, monkeypatch, tree):  # noqa: F811
    """Making one lets other threads run; each goes on with an address, which has to be that of a tensor that stays."""
    made = []

    def zeros(self, size, stream):
        t = torch.zeros(64, dtype=torch.uint8)
        made.append(weakref.ref(t))
        time.sleep(0.05)
        return t
    monkeypatch.setattr(kv4.Kv4Cache, "_zeros", zeros)
    monkeypatch.setattr(kv4, "_tree_work", {})
    got, gate = [], threading.Barrier(4)

    def first():
        gate.wait()
        got.append(cache._tree_workspace(7)[0] if tree else cache._workspace(1, 8, 7)[0])
    threads = [threading.Thread(target=first) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    gc.collect()
    alive = [t().data_ptr() for t in made if t() is not None]
    assert len(set(got)) == 1 and got[0] in alive


@pytest.mark.parametrize("nodes,q_heads,tree", [(257, 2, True), (300, 2, True), (256, 10, True), (3, 5, True), (0, 2, True),
                                                (1025, 2, False)])
@pytest.mark.parametrize("size", [0, 1 << 26])
def test_a_capture_refuses_what_a_call_refuses(cache, monkeypatch, nodes, q_heads, tree, size):  # noqa: F811
    """With the library's error, also where the capture has a workspace already."""
    monkeypatch.setattr(kv4, "_captured", {(-1, 7): (5, [torch.zeros(size, dtype=torch.uint8)] if size else [])})
    cache._work_size = native.lib().aljabr_blackwell_kv4_attention_workspace_size
    with pytest.raises(native.ProviderError):
        cache._captured_workspace(5, nodes, q_heads, 7, tree)


@pytest.mark.parametrize("tree", [True, False])
def test_the_per_thread_stream_is_another_in_each_thread(cache, monkeypatch, tree):  # noqa: F811
    """Handle 2 names a stream of the calling thread: two threads' calls on it run side by side, and want two workspaces."""
    monkeypatch.setattr(kv4.Kv4Cache, "_zeros", lambda self, size, stream: torch.zeros(64, dtype=torch.uint8))
    monkeypatch.setattr(kv4, "_tree_work", {})
    monkeypatch.setattr(kv4, "capture_id", lambda stream: 0)
    got = []
    cache._attend = lambda *a: got.append(a[-3]) or 0
    q, lens, table = torch.zeros(1, 1, 2, 64), torch.ones(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)

    def call():
        if tree:
            got.append(cache._tree_workspace(2)[0])
        else:
            cache.attend(q, lens, table, out=q, stream=2)
    call()
    call()
    gate = threading.Barrier(2)
    threads = [threading.Thread(target=lambda: (gate.wait(), call(), call(), gate.wait())) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert got[0] == got[1] and len(set(got)) == 3 and all(got.count(g) == 2 for g in got)
