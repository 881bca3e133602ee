"""Host-side state of the tree wrappers, without a GPU (the stubs of
test_kv4_wrapper_cpu.py)."""
import gc
import threading
import time
import weakref

import pytest

torch = pytest.importorskip("torch")

from aljabr_b200 import kv4
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
