"""Captured calls of the 4-bit cache's attention: what a graph holds stays its own."""
import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_kv4 import attend_case

pytestmark = pytest.mark.gpu


def capture(stream, call):
    """`call` captured on `stream`, not yet run."""
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    return graph


def test_a_graph_survives_a_later_call_with_more_rows():
    """One token of 4 query heads captured, then 5 tokens (20 rows, twice the workspace) on the same stream."""
    cache, q, sl, table, want, _, _ = attend_case(30, 128, 2, 4, 1, 16, [4000, 100, 9000])
    out, many = torch.zeros_like(q), q.expand(-1, 5, -1, -1).contiguous()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.attend(q, sl, table)
    graph = capture(side, lambda: cache.attend(q, sl, table, out=out))
    with torch.cuda.stream(side):
        cache.attend(many, sl, table)
    side.synchronize()
    others = [torch.full((1 << 20,), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(64)]
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert all(bool((t == 0x5A).all()) for t in others)
