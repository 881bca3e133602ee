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


def test_graphs_of_a_stream_that_was_not_warmed_up():
    """Two batch sizes captured on one stream with nothing run on it before, replayed in reverse, with plain calls on the
    stream between and both at once on two streams."""
    cache, q, sl, table, want, _, _ = attend_case(31, 128, 2, 4, 1, 16, [4000, 100, 9000, 2500])
    side = torch.cuda.Stream()
    graphs = []
    for n in (4, 2):
        out = torch.zeros_like(q[:n])
        graphs.append((capture(side, lambda: cache.attend(q[:n], sl[:n], table[:n], out=out)), out, n))
    few = cache.attend(q[:2], sl[:2], table[:2])
    for graph, out, n in reversed(graphs):
        graph.replay()
        with torch.cuda.stream(side):
            plain = cache.attend(q, sl, table)
        torch.cuda.synchronize()
        assert torch.equal(out, want if n == 4 else few) and torch.equal(plain, want)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _, out, _ in graphs:
        out.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, (graph, _, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], few)


def test_one_graph_of_several_caches_and_row_counts():
    a, q, sl, table, want, _, _ = attend_case(32, 128, 2, 4, 1, 16, [3000, 5000])
    b, qb, slb, tb, want_b, _, _ = attend_case(33, 64, 1, 2, 7, 32, [700, 6000])
    outs = torch.zeros_like(q), torch.zeros_like(qb)

    def both():
        a.attend(q, sl, table, out=outs[0])
        b.attend(qb, slb, tb, out=outs[1])

    graph = capture(torch.cuda.Stream(), both)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want_b)


def test_calls_on_a_stream_of_their_own():
    """`stream=`: the results, and outputs that do not take memory from work still pending on the current stream."""
    from aljabr_b200.logits import process_logits
    cache, q, sl, table, want, _, _ = attend_case(34, 128, 2, 4, 1, 16, [4000, 100])
    slots = torch.arange(64, dtype=torch.int32, device="cuda")
    rows = cache.read(slots)
    logits = torch.randn(3, 5000, device="cuda")
    plain = process_logits(logits)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(20):
        # a block of the output's size, freed while the current stream has yet to read it
        block = torch.zeros(want.numel(), device="cuda")
        torch.cuda._sleep(2_000_000)
        copy = block.clone()
        del block
        out = cache.attend(q, sl, table, stream=side.cuda_stream)
        k, v = cache.read(slots, stream=side.cuda_stream)
        got, token = process_logits(logits, stream=side.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(k, rows[0]) and torch.equal(v, rows[1])
        assert torch.equal(got, plain[0]) and torch.equal(token, plain[1]) and not copy.any()


def test_the_legacy_stream_named_from_another_one():
    cache, q, sl, table, want, _, _ = attend_case(35, 128, 2, 4, 1, 16, [4000, 100])
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        out = cache.attend(q, sl, table, stream=1)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_a_captured_branch_on_a_stream_given_by_handle():
    """Two branches of one graph, the second joined from a stream that the call names; cold, so that both make their
    workspaces in the capture."""
    cache, q, sl, table, want, _, _ = attend_case(36, 128, 2, 4, 1, 16, [4000, 9000])
    outs, side, branch = (torch.zeros_like(q), torch.zeros_like(q)), torch.cuda.Stream(), torch.cuda.Stream()

    def both():
        branch.wait_stream(side)
        cache.attend(q, sl, table, out=outs[0])
        cache.attend(q, sl, table, out=outs[1], stream=branch.cuda_stream)
        side.wait_stream(branch)

    graph = capture(side, both)
    for _ in range(5):
        for out in outs:
            out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
