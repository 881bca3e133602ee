"""Calls of two threads over the 4-bit KV cache, on one stream and with one workspace."""
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from aljabr_b200 import native
from tests import tree_ref as tree
from tests.test_gpu_kv4 import fault_bits
from tests.test_gpu_kv4_tree import tree_case

pytestmark = pytest.mark.gpu


def together(*work):
    """Runs the functions in threads that start at once; what one raises is raised here."""
    gate, wrong = threading.Barrier(len(work)), []

    def run(f):
        try:
            gate.wait()
            f()
        except BaseException as e:      # noqa: BLE001
            wrong.append(e)
    threads = [threading.Thread(target=run, args=(f,)) for f in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if wrong:
        raise wrong[0]


def test_a_chain_and_a_tree_share_a_workspace():
    """Through the C-ABI: a tree's attention is two launches, and the other thread's chain, whose partial sums lie where the tree
    keeps its list of cuts, comes before or after both."""
    p = tree.grow(np.random.default_rng(70), 20)
    cache, q, sl, parents, table, _, _ = tree_case(71, 128, 2, 4, 64, [3000, 500], [p] * 2, torch.bfloat16, wide=True)
    lib, rows = native.lib(), q.shape[1] * 4
    want = cache.attend_tree(q, sl, parents, table), cache.attend(q, sl, table)
    size = max(lib.aljabr_blackwell_kv4_tree_attention_workspace_size(q.shape[1], 8, 2, 128),
               lib.aljabr_blackwell_kv4_attention_workspace_size(q.shape[1], 8, 2, 128))
    assert rows > 32
    work = torch.zeros(size, dtype=torch.uint8, device="cuda")
    outs = [[torch.empty_like(w) for _ in range(300)] for w in want]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    common = q.data_ptr(), native.KV_BF16, 8 * 128, cache.data.data_ptr(), cache.pages, 64, 2, 128, table.data_ptr(), table.shape[1], \
        sl.data_ptr(), 2
    tail = 20, 8, 0, 128 ** -0.5, 0.0, work.data_ptr(), size, stream.cuda_stream

    def trees():
        for o in outs[0]:
            native.check(lib.aljabr_blackwell_kv4_tree_attention_dev(o.data_ptr(), *common, parents.data_ptr(), 20, *tail))

    def chains():
        for o in outs[1]:
            native.check(lib.aljabr_blackwell_kv4_attention_dev(o.data_ptr(), *common, *tail))
    together(trees, chains, trees)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for os, w in zip(outs, want) for o in os)
    assert fault_bits() == 0


def test_first_calls_of_two_threads_that_allocate():
    """A stream's first calls come from two threads, each with caches of its own, whose outputs are made in between."""
    p = tree.grow(np.random.default_rng(72), 20)
    cases = [tree_case(73 + i, 128, 2, 4, 64, [1000, 500], [p] * 2, torch.bfloat16, wide=i > 1) for i in range(4)]
    want = [c[0].attend_tree(*c[1:5]) for c in cases]
    for _ in range(5):
        stream, got = torch.cuda.Stream(), [[] for _ in cases]
        torch.cuda.synchronize()

        def work(i):
            with torch.cuda.stream(stream):
                for _ in range(8):
                    got[i].append(cases[i][0].attend_tree(*cases[i][1:5]))
                    got[i].append(torch.full_like(want[i], float("nan")))
        together(*(lambda i=i: work(i) for i in range(4)))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(o, w) for o in g[::2]) and all(torch.isnan(o).all() for o in g[1::2])
    assert fault_bits() == 0
