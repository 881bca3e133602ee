"""Trees of drafted tokens over the 4-bit KV cache on the GPU, against the
plain forms of tests/tree_ref.py and tests/kv4_ref.py."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from aljabr_b200 import native
from tests import kv4_ref as ref
from tests import tree_ref as tree
from tests.test_gpu_kv4 import fault_bits, make

pytestmark = pytest.mark.gpu


def cuda(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dtype is None else t.to(dtype)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def table_of(positions, n, theta=10000.0):
    a = np.arange(positions)[:, None] * theta ** (-np.arange(n) / n)
    return np.stack((np.cos(a), np.sin(a)), -1).astype(np.float32)


# ---------------------------------------------------------------- rows with their rotation
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,hq,hkv,D,rot,inter,ps", [
    (1, 4, 1, 64, 64, False, 16), (1, 32, 8, 128, 128, False, 64), (5, 9, 3, 128, 128, True, 48), (7, 2, 2, 64, 32, True, 16),
    (33, 6, 2, 256, 48, False, 16), (3, 1, 1, 256, 256, False, 16), (130, 8, 8, 128, 16, False, 64), (61, 7, 1, 64, 48, True, 16),
    (700, 5, 1, 64, 64, False, 32), (601, 3, 1, 256, 128, True, 16)])
def test_rotated_append_writes_what_the_plain_form_does(n, hq, hkv, D, rot, inter, ps, dtype):
    rng = np.random.default_rng(n + D + rot)
    pages, far = -(-n // ps) + 1, 50
    table = table_of(far, rot // 2)
    cache, want = make(pages, ps, hkv, D, fill=0xA5), ref.RefCache(pages, ps, hkv, D, fill=0xA5)
    q, k, v = (cuda(rng.normal(size=(n, h, D)).astype(np.float32), dtype) for h in (hq, hkv, hkv))
    qn, kn, vn = (t.float().cpu().numpy() for t in (q, k, v))
    slots, pos = rng.permutation(pages * ps)[:n].astype(np.int32), rng.integers(0, far, n).astype(np.int32)
    if n > 4:
        slots[1], pos[2], slots[3], pos[3] = -1, -1, -1, -7
    back = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    out = cache.append_rotated(q, k, v, cuda(slots), cuda(pos), cuda(table), interleaved=inter, k_back=back[0], v_back=back[1])
    assert torch.equal(out.cpu(), torch.from_numpy(tree.rotate(qn, table, pos, inter)).to(dtype))
    kr = tree.rotate(kn, table, pos, inter)
    keep = (slots >= 0) & (pos >= 0)
    for i in np.flatnonzero(keep):
        for h in range(hkv):
            want.write(int(slots[i]), h, kr[i, h], vn[i, h])
    assert np.array_equal(cache.data.cpu().numpy(), want.data)
    for x, b in zip((kr, vn), back):
        exact = ref.values(*ref.quantise(x))
        exact[~keep] = 0.0
        assert torch.equal(b.cpu(), torch.from_numpy(exact.astype(np.float32)).to(dtype))
    assert fault_bits() == 0


def test_a_rotation_by_nothing_is_append():
    rng = np.random.default_rng(4)
    a, b = make(3, 16, 2, 128), make(3, 16, 2, 128)
    k, v, q = (cuda(rng.normal(size=(40, h, 128)).astype(np.float32)) for h in (2, 2, 6))
    slots = torch.arange(40, dtype=torch.int32, device="cuda")
    out = a.append_rotated(q, k, v, slots, torch.zeros_like(slots), cuda(table_of(1, 64)))
    b.append(k, v, slots)
    assert torch.equal(out, q) and torch.equal(a.data, b.data)


@pytest.mark.parametrize("dtype,cut", [(torch.float32, 0), (torch.float32, 1), (torch.float32, 4), (torch.bfloat16, 0),
                                       (torch.bfloat16, 3), (torch.bfloat16, 8)])
def test_rotated_append_of_columns_of_one_buffer_and_in_place(dtype, cut):
    rng = np.random.default_rng(5)
    wide = cuda(rng.normal(size=(37, 6 * 64 + 8)).astype(np.float32), dtype)
    q, k, v = (wide[:, cut + a:cut + b].unflatten(1, (-1, 64)) for a, b in ((0, 256), (256, 320), (320, 384)))
    table, slots, pos = cuda(table_of(99, 32)), torch.arange(37, dtype=torch.int32, device="cuda"), cuda(rng.integers(0, 99, 37).astype(np.int32))
    a, b = make(3, 16, 1, 64), make(3, 16, 1, 64)
    want = a.append_rotated(q.contiguous(), k.contiguous(), v.contiguous(), slots, pos, table)
    kept = wide[:, cut + 256:].clone()
    got = b.append_rotated(q, k, v, slots, pos, table, q_out=q)
    assert got is q and torch.equal(q, want) and torch.equal(a.data, b.data) and torch.equal(wide[:, cut + 256:], kept)


def test_positions_and_slots_outside_their_ranges_are_absent():
    cache = make(1, 16, 1, 64)
    x = torch.ones(4, 1, 64, device="cuda")
    out = cache.append_rotated(x, x, x, ints([0, 16, 2, 3]), ints([9, 0, 10, 2 ** 31 - 1]), cuda(table_of(10, 32)))
    assert fault_bits() & 2
    k, v = cache.read(ints([0, 1, 2, 3]))
    assert (v[0] == 1).all() and not v[1:].any() and not k[1:].any()
    assert out[0].any() and torch.equal(out[1], x[1]) and not out[2:].any()
    assert fault_bits() == 0


# ---------------------------------------------------------------- attention
def widen(t, ps):
    """More columns of absent pages: room for 131072 positions a sequence."""
    return np.pad(t, ((0, 0), (0, 131072 // ps - t.shape[1])), constant_values=-1)


def tree_case(seed, D, hkv, G, ps, lens, trees, dtype=torch.float32, paged=True, fill=0xFF, v_size=1.0, wide=False):
    """A cache whose unused bytes, absent nodes' rows among them, are `fill` (0xFF: scales that are NaN).  wide: a block
    table of many more columns, for which more than 32 rows of bf16 run on the tensor cores' kernel."""
    rng = np.random.default_rng(seed)
    B, T = len(lens), len(trees[0])
    per = max(1, -(-max(lens) // ps))
    cache = make(B * per + 1, ps, hkv, D, fill=fill)
    order = rng.permutation(B * per).reshape(B, per) if paged else np.arange(B).reshape(B, 1)
    k64, v64 = [], []
    for b, n in enumerate(lens):
        k = rng.normal(size=(n, hkv, D)).astype(np.float32) * (0.3 + 2 * rng.random((1, hkv, D)) ** 4).astype(np.float32)
        v = rng.normal(size=(n, hkv, D)).astype(np.float32) * np.float32(v_size)
        pos = np.arange(n)
        slots = order[b, pos // ps] * ps + pos % ps
        for t, path in enumerate(tree.chains(trees[b])):
            if not path and n >= T:
                slots[n - T + t] = -1
        if n:
            cache.append(cuda(k), cuda(v), cuda(slots.astype(np.int32)))
        k64.append(ref.values(*ref.quantise(k)) if n else k.astype(np.float64))
        v64.append(ref.values(*ref.quantise(v)) if n else v.astype(np.float64))
    q = cuda((rng.normal(size=(B, T, hkv * G, D)) * 1.5).astype(np.float32), dtype)
    table = None
    if paged:
        t = order.astype(np.int32)
        for b, n in enumerate(lens):
            t[b, -(-n // ps):] = -1
        table = cuda(widen(t, ps) if wide else t)
    return cache, q, ints(lens), ints(trees), table, k64, v64


def check(out, q, k64, v64, lens, trees, window=0, soft_cap=0.0):
    """fp32: the bound of check() in tests/test_gpu_kv4.py.  bf16: K in fp16 (half a step, 2^-11 of each value: at most
    2^-11 of delta a score, the output 2 of those of sum P |v|), P and V in fp16 (2^-11 each), with values far below
    their tile's largest to 2^-24 of it; the output to 8 bits.  And the error's norm, over a case: errors of 2^-11 and
    below a value that do not add up, within the output's own rounding of 2^-8."""
    qn, on = q.float().cpu().numpy(), out.double().cpu().numpy()
    bf16 = q.dtype == torch.bfloat16
    off = size = 0.0
    for b, n in enumerate(lens):
        want, weight, delta = tree.attention(qn[b], k64[b], v64[b], trees[b], n, window=window, soft_cap=soft_cap)
        floor = n * 2.0 ** (-24 if bf16 else -28) * (np.abs(v64[b]).max() if n else 0.0)
        tol = weight * (2 * delta[..., None] * 2.0 ** (-11 if bf16 else -20) + 2.0 ** (-10 if bf16 else -18)) + floor
        if bf16:
            tol = tol + np.abs(want) * 2.0 ** -8
        err = np.abs(on[b] - want)
        assert np.all(err <= tol), (b, n, float(err.max()), float((err / np.maximum(tol, 1e-300)).max()))
        off, size = off + (err ** 2).sum(), size + (want ** 2).sum()
        gone = [t for t, p in enumerate(tree.chains(trees[b])) if not p or n < len(trees[b])]
        assert not out[b, gone].any()
    assert off <= size * (2.0 ** -8 if bf16 else 2.0 ** -18) ** 2, (off / size) ** 0.5


# type, absent nodes behind the tree: fp32; bf16 on the kernel of few columns; bf16 on the tensor cores' kernel
KERNELS = [(torch.float32, 0), (torch.bfloat16, 0), (torch.bfloat16, 60)]
CASES = [
    # D, hkv, G, page size, nodes, roots, absent, lens, window, cap
    (128, 2, 4, 16, 1, 1, 0, [1, 40, 0], 0, 0.0),
    (128, 8, 4, 64, 5, 1, 0, [257], 0, 0.0),
    (128, 2, 4, 16, 7, 2, 2, [7, 6, 0, 300, 129], 0, 0.0),
    (128, 1, 8, 48, 33, 1, 4, [1000, 33, 140], 0, 0.0),
    (128, 1, 1, 4096, 61, 3, 0, [3000], 0, 0.0),
    (128, 3, 3, 64, 64, 1, 10, [200, 700], 100, 0.0),
    (64, 4, 2, 16, 21, 1, 3, [21, 513, 90], 33, 30.0),
    (64, 1, 16, 32, 64, 1, 0, [64, 65, 400], 0, 0.0),
    (64, 2, 7, 16, 40, 4, 5, [777], 3, 0.0),
    (256, 2, 4, 16, 16, 1, 2, [16, 640], 0, 0.0),
    (256, 1, 5, 80, 30, 2, 0, [400, 31], 20, 50.0),
    (128, 1, 4, 64, 256, 1, 9, [256, 900], 0, 0.0),
]


@pytest.mark.parametrize("dtype,wide", [(torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("D,hkv,G,ps,nodes,roots,absent,lens,window,cap", CASES)
def test_tree_attention_matches_64_bits(D, hkv, G, ps, nodes, roots, absent, lens, window, cap, dtype, wide):
    rng = np.random.default_rng(nodes)
    trees = [tree.grow(rng, nodes, roots, absent) for _ in lens]
    cache, q, sl, parents, table, k64, v64 = tree_case(D + G + nodes, D, hkv, G, ps, lens, trees, dtype, wide=wide)
    out = cache.attend_tree(q, sl, parents, table, window=window, soft_cap=cap)
    check(out, q, k64, v64, lens, trees, window, cap)
    assert fault_bits() == 0


@pytest.mark.parametrize("D,hkv,G,nodes,lens", [(256, 1, 4, 10, [20000, 3]), (256, 2, 2, 64, [5000, 9000]), (128, 1, 8, 17, [30000, 700]),
                                                (64, 2, 4, 30, [25000, 40]), (128, 1, 4, 40, [2000] * 40)])
def test_long_contexts_and_many_pieces(D, hkv, G, nodes, lens):
    """Every stage of the pipeline goes round many times, and items are cut over CTAs: against fp32 queries, whose kernel
    is another.  The same queries, so what differs is bf16's rounding of the output and the fp16 operands: 2^-8 in norm."""
    p = tree.grow(np.random.default_rng(50), nodes, 1, nodes // 9)
    rng = np.random.default_rng(51)
    per = -(-max(lens) // 64)
    cache = make(len(lens) * per, 64, hkv, D)
    order = rng.permutation(len(lens) * per).reshape(len(lens), per)
    n = len(lens) * per * 64
    k, v = (torch.randn(n, hkv, D, device="cuda", generator=torch.Generator("cuda").manual_seed(s)) for s in (1, 2))
    cache.append(k, v, torch.arange(n, dtype=torch.int32, device="cuda"))
    q = cuda(rng.normal(size=(len(lens), nodes, hkv * G, D)).astype(np.float32), torch.bfloat16)
    args = ints(lens), ints(p), cuda(widen(order.astype(np.int32), 64))
    want, got = cache.attend_tree(q.float(), *args).double(), cache.attend_tree(q, *args)
    assert float((got.double() - want).norm()) <= 2.0 ** -8 * float(want.norm())
    gone = [t for t, path in enumerate(tree.chains(p)) if not path]
    assert not got[:, gone].any() and torch.equal(got, cache.attend_tree(q, *args))
    assert fault_bits() == 0


def test_more_sequences_than_threads():
    """1400 sequences, some of no length; against fp32, as in the test before."""
    rng = np.random.default_rng(52)
    lens = rng.integers(0, 130, 1400)
    p = tree.grow(rng, 12, 2, 1)
    cache, q, sl, parents, table, _, _ = tree_case(53, 128, 1, 4, 64, lens.tolist(), [p] * 1400, torch.bfloat16)
    want, got = cache.attend_tree(q.float(), sl, parents, table).double(), cache.attend_tree(q, sl, parents, table)
    assert float((got.double() - want).norm()) <= 2.0 ** -8 * float(want.norm())
    assert torch.equal(got == 0, want == 0) and fault_bits() == 0


@pytest.mark.parametrize("dtype,pad", KERNELS)
def test_queries_of_a_wider_buffer_and_any_scale(dtype, pad):
    """Rows at offsets that are no multiple of 16 bytes; scales of 0 and below; the same results as contiguous rows."""
    p = tree.grow(np.random.default_rng(54), 20) + [-2] * pad
    T = len(p)
    cache, q, sl, parents, table, k64, v64 = tree_case(54, 64, 2, 2, 16, [90 + pad, 300 + pad], [p] * 2, dtype, wide=True)
    for scale in (None, 0.0, -0.07):
        want = cache.attend_tree(q, sl, parents, table, scale=scale)
        for cut in (0, 1, 4, 8):
            wide = torch.full((2 * T, 256 + 11), float("nan"), device="cuda", dtype=dtype)
            view = wide[:, cut:cut + 256]
            view.copy_(q.view(2 * T, 256))
            assert torch.equal(cache.attend_tree(view.view(2, T, 4, 64), sl, parents, table, scale=scale), want)
    check(cache.attend_tree(q, sl, parents, table, scale=-0.125), -q, k64, v64, [90 + pad, 300 + pad], [p] * 2)
    assert fault_bits() == 0


@pytest.mark.parametrize("nodes,lens", [(10, [4000]), (40, [4000, 900, 3000])])
def test_two_graphs_and_calls_at_once(nodes, lens):
    """Two captured graphs and eager calls on three streams, all in flight together: none uses another's workspace."""
    p = tree.grow(np.random.default_rng(55), nodes)
    cases = [tree_case(56 + i, 128, 2, 4, 64, lens, [p] * len(lens), torch.bfloat16, wide=True) for i in range(3)]
    want = [c[0].attend_tree(*c[1:5]) for c in cases]
    out = [torch.empty_like(w) for w in want]
    torch.cuda.synchronize()
    streams, graphs = [torch.cuda.Stream() for _ in cases], []
    for c, o in zip(cases[:2], out):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=streams[0]):
            for _ in range(3):
                c[0].attend_tree(*c[1:5], out=o)
    for _ in range(20):
        for o in out:
            o.fill_(7)
        torch.cuda.synchronize()
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
        with torch.cuda.stream(streams[2]):
            for _ in range(3):
                cases[2][0].attend_tree(*cases[2][1:5], out=out[2])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out))
    assert fault_bits() == 0


def test_calls_of_two_threads():
    """On one stream, whose workspace they share, and on two."""
    import threading
    p = tree.grow(np.random.default_rng(57), 20)
    cases = [tree_case(58 + i, 128, 2, 4, 64, [3000, 500], [p] * 2, torch.bfloat16, wide=True) for i in range(2)]
    want = [c[0].attend_tree(*c[1:5]) for c in cases]
    torch.cuda.synchronize()
    for streams in ([torch.cuda.Stream()] * 2, [torch.cuda.Stream(), torch.cuda.Stream()]):
        outs = [[torch.empty_like(w) for _ in range(30)] for w in want]

        def work(i):
            for o in outs[i]:
                cases[i][0].attend_tree(*cases[i][1:5], out=o, stream=streams[i].cuda_stream)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for os, w in zip(outs, want) for o in os)
    assert fault_bits() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_window_far_shorter_than_the_context(dtype):
    for window in (1, 5, 200, 4000):
        rng = np.random.default_rng(window)
        trees = [tree.grow(rng, 40, 1, 4) for _ in range(2)]
        lens = [5000, 130]
        cache, q, sl, parents, table, k64, v64 = tree_case(59, 128, 1, 4, 64, lens, trees, dtype, wide=True)
        check(cache.attend_tree(q, sl, parents, table, window=window), q, k64, v64, lens, trees, window)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_tree_for_all_and_no_table(dtype):
    p = tree.grow(np.random.default_rng(1), 12)
    lens = [int(n) for n in np.random.default_rng(2).integers(0, 200, 70)]
    cache, q, sl, _, _, k64, v64 = tree_case(3, 64, 2, 2, 208, lens, [p] * 70, dtype, paged=False)
    out = cache.attend_tree(q, sl, ints(p))
    check(out, q, k64, v64, lens, [p] * 70)
    assert torch.equal(out, cache.attend_tree(q, sl, ints([p] * 70)))


def test_a_chain_is_attend():
    """fp32, where both take the same steps: a tree without branches."""
    for T, lens in ((1, [30, 1]), (5, [5, 700, 64])):
        chain = [list(range(-1, T - 1))] * len(lens)
        cache, q, sl, parents, table, k64, v64 = tree_case(T, 128, 2, 4, 16, lens, chain)
        out = cache.attend_tree(q, sl, parents, table)
        check(out, q, k64, v64, lens, chain)
        near = cache.attend(q, sl, table)
        assert float((out - near).norm() / near.norm()) < 2.0 ** -18


@pytest.mark.parametrize("dtype,pad", KERNELS)
def test_nan_rows_of_other_branches_do_not_leak(dtype, pad):
    """A node's row of NaN reaches the node and what descends from it; one before the window reaches nothing."""
    p = [-1, 0, 0, 1, 2, 2, 3] + [-2] * pad
    lens = [200 + pad]
    cache, q, sl, parents, table, k64, v64 = tree_case(7, 128, 2, 4, 16, lens, [p], dtype, wide=True)
    clean = cache.attend_tree(q, sl, parents, table, window=50)
    bad = torch.full((2, 2, 128), float("nan"), device="cuda")
    cache.append(bad, bad, ints([int(table[0, w // 16]) * 16 + w % 16 for w in (100, 193 + 1)]))
    out = cache.attend_tree(q, sl, parents, table, window=50)
    assert torch.isnan(out[0, [1, 3, 6]]).all()
    assert torch.equal(out[0, [0, 2, 4, 5]], clean[0, [0, 2, 4, 5]])


@pytest.mark.parametrize("dtype,pad", KERNELS)
def test_a_nan_group_of_v_stays_in_its_dims_and_branch(dtype, pad):
    p = [-1, 0, 0, 1] + [-2] * pad
    cache, q, sl, parents, table, k64, v64 = tree_case(8, 128, 1, 2, 16, [40 + pad], [p], dtype, wide=True)
    clean = cache.attend_tree(q, sl, parents, table)
    for at, rows in ((37, [1, 3]), (20, [0, 1, 2, 3])):
        slot = ints([int(table[0, at // 16]) * 16 + at % 16])
        k, v = cache.read(slot)
        v[0, 0, 33] = float("inf")
        cache.append(k, v, slot)
        out = cache.attend_tree(q, sl, parents, table)
        assert torch.isnan(out[0, rows, :, 32:64]).all()
        rest = [t for t in range(4) if t not in rows]
        assert torch.isfinite(out[0][rest]).all() and torch.isfinite(out[..., :32]).all() and torch.isfinite(out[..., 64:]).all()
        tol = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -18
        keep = [d for d in range(128) if not 32 <= d < 64]
        # the requantised row is the same row: its other groups are d * integers, d their extreme / -8
        assert float((out - clean)[..., keep].double().norm()) <= 2 * tol * float(clean.double().norm())


@pytest.mark.parametrize("dtype,pad", KERNELS)
@pytest.mark.parametrize("factor", [0.0, 1e-30, 1e-6, 1e6])
def test_queries_of_any_size(factor, dtype, pad):
    p = tree.grow(np.random.default_rng(9), 20) + [-2] * pad
    cache, q, sl, parents, table, k64, v64 = tree_case(9, 128, 2, 2, 16, [150 + pad], [p], dtype, wide=True)
    q = (q.float() * factor).to(dtype)
    out = cache.attend_tree(q, sl, parents, table)
    if factor < 1e5:
        check(out, q, k64, v64, [150 + pad], [p])
    else:                                          # one position takes all: the largest score's V, where it leads by far
        qn = q.double().cpu().numpy()[0]
        for t, rows in enumerate(tree.visible(p, 150 + pad)[:20]):
            for h in range(4):
                s = k64[0][rows, h // 2] @ qn[t, h]
                if np.sort(s)[-1] - (np.sort(s)[-2] if len(s) > 1 else -np.inf) > 2.0 ** -8 * np.abs(s).max():
                    want = v64[0][rows[int(s.argmax())], h // 2]
                    assert np.abs(out[0, t, h].double().cpu().numpy() - want).max() <= 2.0 ** -8 * np.abs(want).max()


@pytest.mark.parametrize("dtype,pad", KERNELS)
@pytest.mark.parametrize("size", [1e-6, 1e-3, 3e4])
def test_values_of_any_size(size, dtype, pad):
    p = tree.grow(np.random.default_rng(10), 40) + [-2] * pad
    cache, q, sl, parents, table, k64, v64 = tree_case(10, 128, 1, 4, 16, [300 + pad], [p], dtype, v_size=size, wide=pad > 0)
    check(cache.attend_tree(q, sl, parents, table), q, k64, v64, [300 + pad], [p])


@pytest.mark.parametrize("dtype,pad", KERNELS)
def test_non_finite_queries_stay_in_their_rows(dtype, pad):
    p = tree.grow(np.random.default_rng(11), 9) + [-2] * pad
    cache, q, sl, parents, table, _, _ = tree_case(11, 128, 2, 4, 16, [70 + pad], [p], dtype, wide=True)
    out = cache.attend_tree(q, sl, parents, table)
    bad = q.clone()
    bad[0, 3, 1, 5], bad[0, 4, 6, 0] = float("nan"), float("inf")
    got = cache.attend_tree(bad, sl, parents, table)
    hit = torch.zeros(9 + pad, 8, dtype=torch.bool)
    hit[3, 1] = hit[4, 6] = True
    assert torch.isnan(got[0][hit]).all() and torch.equal(got[0][~hit], out[0][~hit])


def test_what_is_no_tree_is_absent_and_reported():
    cache, q, sl, parents, table, k64, v64 = tree_case(12, 64, 1, 2, 16, [50], [[-1, 0, 1, 0, 2]])
    out = cache.attend_tree(q, sl, ints([[-1, 0, 2, 0, 2]]), table)       # node 2 its own parent, node 4 a child of it
    assert fault_bits() & 2
    check(out, q, k64, v64, [50], [[-1, 0, -2, 0, 2]])
    assert fault_bits() == 0
    for t in (-3, -2 ** 31, 2 ** 31 - 1):
        out = cache.attend_tree(q, sl, ints([[-1, 0, t, 0, 2]]), table)
        assert fault_bits() & 2
        check(out, q, k64, v64, [50], [[-1, 0, -2, 0, 2]])
    for lens in ([-1], [10 ** 6]):
        cache.attend_tree(q, ints(lens), parents, table)
        assert fault_bits() & 2
    assert not cache.attend_tree(q, ints([-5]), parents, table).any() and fault_bits() & 2


def test_pages_lengths_and_parents_outside_their_ranges_on_both_kernels():
    """A page that is not there reads as zeros, a length beyond the table as the table's, a wrong parent as an absent node:
    bf16 on either kernel as fp32, within the output's rounding (2^-8 in norm)."""
    p = tree.grow(np.random.default_rng(15), 30)
    wrong = list(p)
    wrong[7], wrong[20] = 7, 4000
    cache, q, sl, parents, table, _, _ = tree_case(15, 128, 2, 4, 16, [300, 90], [p] * 2, torch.bfloat16, fill=0)
    wide = cuda(widen(table.cpu().numpy(), 16))

    def all_agree(lens, parents, edit=None):
        outs = []
        for x, t in ((q.float(), table), (q, table), (q, wide)):
            t = t.clone()
            if edit is not None:
                t[0, 3], t[0, 10], t[1, 1] = edit
            assert fault_bits() == 0
            outs.append(cache.attend_tree(x, lens, parents, t).double())
            assert fault_bits() & 2
        for o in outs[1:]:
            assert float((o - outs[0]).norm()) <= 2.0 ** -8 * float(outs[0].norm())

    for bad in (-1, cache.pages, 2 ** 31 - 1):
        all_agree(sl, parents, (bad, bad, bad))
    all_agree(sl, ints([wrong, p]))
    cut = table.shape[1] * 16
    assert not cache.attend_tree(q, ints([-1, -2 ** 31]), parents, wide).any() and fault_bits() & 2
    outs = [cache.attend_tree(x, ints([cut + 1, 90]), parents, table) for x in (q.float(), q)]
    assert fault_bits() & 2 and float((outs[1].double() - outs[0].double()).norm()) <= 2.0 ** -8 * float(outs[0].double().norm())


# ---------------------------------------------------------------- acceptance
def read_all(cache):
    return cache.data.cpu().numpy().copy()


@pytest.mark.parametrize("D,hkv,ps,layers,batch,nodes", [
    (64, 1, 16, 1, 1, 1), (128, 2, 16, 3, 5, 9), (256, 1, 48, 2, 3, 40), (128, 8, 64, 4, 2, 64), (64, 3, 16, 2, 4, 256)])
def test_acceptance_moves_the_path_of_every_layer(D, hkv, ps, layers, batch, nodes):
    rng = np.random.default_rng(D + nodes)
    trees = [tree.grow(rng, nodes, 1, nodes // 8) for _ in range(batch)]
    lens = [nodes + int(rng.integers(0, 50)) for _ in range(batch)]
    if batch > 2:
        lens[1] = nodes - 1                        # no tree
        trees[2][0] = -2                           # no node 0
    per = -(-max(lens) // ps)
    order = rng.permutation(batch * per).reshape(batch, per)
    caches = [make(batch * per, ps, hkv, D) for _ in range(layers)]
    for c in caches:
        c.data.copy_(cuda(rng.integers(0, 256, c.data.numel(), dtype=np.uint8)))
    before = [read_all(c) for c in caches]
    # three tokens: many accepted nodes, siblings with the same token
    drafted, picked = rng.integers(0, 3, (batch, nodes)), rng.integers(0, 3, (batch, nodes))
    from aljabr_b200.kv4 import accept_tree
    path, count, token, new = (t.cpu().numpy() for t in accept_tree(
        caches, ints(lens), ints(trees), ints(drafted), ints(picked), cuda(order.astype(np.int32))))
    image = [ref.RefCache(batch * per, ps, hkv, D) for _ in caches]
    for i, b4 in zip(image, before):
        i.data[:] = b4
    longest = 0
    for b in range(batch):
        want = tree.walk(trees[b], drafted[b], picked[b]) if lens[b] >= nodes else []
        longest = max(longest, len(want))
        assert path[b].tolist() == want + [-1] * (nodes - len(want)) and count[b] == len(want)
        assert token[b] == (picked[b][want[-1]] if want else -1)
        assert new[b] == (lens[b] - nodes + len(want) if lens[b] >= nodes else lens[b])
        slot = lambda p: int(order[b, p // ps] * ps + p % ps)  # noqa: E731
        for img, b4 in zip(image, before):
            for i, t in enumerate(want):
                src, dst = slot(lens[b] - nodes + t), slot(lens[b] - nodes + i)
                for h in range(hkv):
                    for (a, z), w in zip(zip(img._places(src, h), img._places(dst, h)), (D // 2, D // 2, D // 16, D // 16)):
                        img.data[z:z + w] = b4[a:a + w]
    assert nodes < 9 or longest > 2
    for c, img in zip(caches, image):
        assert np.array_equal(read_all(c), img.data)
    assert fault_bits() == 0


def test_acceptance_of_a_whole_chain_moves_nothing():
    from aljabr_b200.kv4 import accept_tree
    T = 30
    cache = make(4, 16, 2, 128)
    cache.data.random_(0, 256)
    before = cache.data.clone()
    d = torch.arange(T, dtype=torch.int32, device="cuda")[None]
    out = accept_tree(cache, ints([T + 3]), ints(list(range(-1, T - 1))), d.contiguous(), d + 1, ints([[3, 0, 2]]))
    assert out[0][0].tolist() == list(range(T)) and [int(t) for t in out[1:]] == [T, T, T + 3]
    assert torch.equal(cache.data, before)
    again = accept_tree(cache, ints([T + 3]), ints(list(range(-1, T - 1))), d.contiguous(), d + 1, ints([[3, 0, 2]]), out=out)
    assert again is out and fault_bits() == 0


def test_acceptance_on_a_page_that_is_not_there():
    from aljabr_b200.kv4 import accept_tree
    cache = make(2, 16, 1, 64)
    cache.data.random_(0, 256)
    before = cache.data.clone()
    p, d = ints([-1, 0, 0, 1]), ints([[0, 5, 6, 7]])
    got = accept_tree(cache, ints([20]), p, d, ints([[6, 0, 0, 0]]), ints([[1, 2]]))
    assert fault_bits() & 2 and got[0].tolist() == [[0, 2, -1, -1]] and torch.equal(cache.data, before)
    accept_tree(cache, ints([33]), p, d, ints([[6, 0, 0, 0]]), ints([[1, 0]]))
    assert fault_bits() & 2 and torch.equal(cache.data, before)


# ---------------------------------------------------------------- a step
def test_wrapper_refusals():
    from aljabr_b200.kv4 import accept_tree
    cache = make(2, 16, 1, 64)
    x, n, table = torch.ones(3, 1, 64, device="cuda"), ints([0, 1, 2]), cuda(table_of(5, 32))
    q, lens, parents = torch.ones(1, 3, 2, 64, device="cuda"), ints([10]), ints([-1, 0, 1])
    for kw in (dict(q=x.half()), dict(q=x.bfloat16()), dict(q=x[:2]), dict(q=x.flatten(1)), dict(positions=n[:2]), dict(positions=n.long()),
               dict(rope=table.double()), dict(rope=table[:, :, 0]), dict(rope=table[:, :12]), dict(q_out=x.bfloat16()),
               dict(q_out=torch.empty(3, 2, 64, device="cuda")), dict(q=x.cpu()), dict(rope=table.cpu())):
        args = dict(dict(q=x, k=x, v=x, slots=n, positions=n, rope=table), **kw)
        with pytest.raises(native.ProviderError):
            cache.append_rotated(**args)
    for kw in (dict(parents=parents.long()), dict(parents=parents[:2]), dict(parents=ints([[-1, 0, 1]] * 2)), dict(parents=parents.cpu()),
               dict(q=q[0]), dict(q=q.half()), dict(seq_lens=ints([10, 10])), dict(out=q.bfloat16()),
               dict(block_table=torch.zeros(1, 0, dtype=torch.int32, device="cuda"))):
        with pytest.raises(native.ProviderError):
            cache.attend_tree(**dict(dict(q=q, seq_lens=lens, parents=parents), **kw))
    d = ints([[1, 2, 3]])
    for kw in (dict(caches=[]), dict(caches=[cache, make(2, 16, 2, 64)]), dict(caches=[cache, cache]), dict(drafted=d[0]),
               dict(picked=d[:, :2]), dict(picked=d.long()), dict(seq_lens=ints([10, 1])), dict(parents=ints([-1])),
               dict(block_table=torch.zeros(1, 0, dtype=torch.int32, device="cuda")), dict(out=(d, lens, lens, lens))):
        with pytest.raises(native.ProviderError):
            accept_tree(**dict(dict(caches=cache, seq_lens=lens, parents=parents, drafted=d, picked=d), **kw))
    assert fault_bits() == 0


def step_case(dtype, seed=40, layers=3, D=128, hkv=2, G=4, ps=16, lens=(70, 300, 12)):
    """The state of a serving step: caches filled up to each base, and the drafted rows."""
    rng = np.random.default_rng(seed)
    T, B = 12, len(lens)
    trees = [tree.grow(rng, T, 1, b % 3) for b in range(B)]
    per = -(-max(lens) // ps) + 1
    order = rng.permutation(B * per).reshape(B, per)
    caches = [make(B * per, ps, hkv, D, fill=0xFF) for _ in range(layers)]
    old = []
    for c in caches:
        rows = []
        for b, n in enumerate(lens):
            k, v = (rng.normal(size=(n - T, hkv, D)).astype(np.float32) for _ in range(2))
            pos = np.arange(n - T)
            if n > T:
                c.append(cuda(k), cuda(v), cuda((order[b, pos // ps] * ps + pos % ps).astype(np.int32)))
            rows.append((k, v))
        old.append(rows)
    slots, positions = [], []
    for b, n in enumerate(lens):
        for t, path in enumerate(tree.chains(trees[b])):
            p = n - T + t
            slots.append(int(order[b, p // ps] * ps + p % ps) if path else -1)
            positions.append(n - T + len(path) - 1 if path else -1)
    q, k, v = (cuda(rng.normal(size=(layers, B * T, h, D)).astype(np.float32), dtype) for h in (hkv * G, hkv, hkv))
    drafted, picked = rng.integers(0, 2, (B, T)), rng.integers(0, 2, (B, T))
    table = table_of(400, D // 2)
    return dict(caches=caches, lens=ints(list(lens)), trees=trees, parents=ints(trees), table=cuda(order.astype(np.int32)),
                slots=ints(slots), positions=ints(positions), rope=cuda(table), q=q, k=k, v=v, drafted=ints(drafted),
                picked=ints(picked), old=old, rope_np=table, order=order)


def run_step(s):
    from aljabr_b200.kv4 import accept_tree
    B, T = s["drafted"].shape
    outs = []
    for i, c in enumerate(s["caches"]):
        q = c.append_rotated(s["q"][i], s["k"][i], s["v"][i], s["slots"], s["positions"], s["rope"])
        outs.append(c.attend_tree(q.view(B, T, *q.shape[1:]), s["lens"], s["parents"], s["table"]))
    return outs, accept_tree(s["caches"], s["lens"], s["parents"], s["drafted"], s["picked"], s["table"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_step_and_the_next_token(dtype):
    """Rows in, attention, acceptance; then the next token's attention sees the accepted path and nothing of the rest."""
    s = step_case(dtype)
    outs, (path, count, token, new) = run_step(s)
    B, T = s["drafted"].shape
    lens = s["lens"].tolist()
    rng = np.random.default_rng(41)
    pos = s["positions"].cpu().numpy()
    for i, cache in enumerate(s["caches"]):
        kn, vn = (s[x][i].float().cpu().numpy() for x in "kv")
        qr, kr = (tree.rotate(x, s["rope_np"], pos, False) for x in (s["q"][i].float().cpu().numpy(), kn))
        qr = torch.from_numpy(qr).to(dtype).view(B, T, *qr.shape[1:])
        k64 = [ref.values(*ref.quantise(np.concatenate((s["old"][i][b][0], kr[b * T:(b + 1) * T])))) for b in range(B)]
        v64 = [ref.values(*ref.quantise(np.concatenate((s["old"][i][b][1], vn[b * T:(b + 1) * T])))) for b in range(B)]
        check(outs[i], qr, k64, v64, lens, s["trees"])
        # the next token, fp32
        q = cuda(rng.normal(size=(B, 1, qr.shape[2], qr.shape[3])).astype(np.float32))
        k, v = (cuda(rng.normal(size=(B, *kn.shape[1:])).astype(np.float32)) for _ in range(2))
        at = new.cpu().numpy()
        slots = [int(s["order"][b, at[b] // 16] * 16 + at[b] % 16) for b in range(B)]
        cache.append(k, v, ints(slots))
        out = cache.attend(q, new + 1, s["table"])
        for b in range(B):
            p = tree.walk(s["trees"][b], s["drafted"][b].tolist(), s["picked"][b].tolist())
            assert path[b, :len(p)].tolist() == p and at[b] == lens[b] - T + len(p)
            keep = list(range(lens[b] - T)) + [lens[b] - T + t for t in p]
            kk, vv = (np.concatenate((x[b][keep], ref.values(*ref.quantise(y[b:b + 1].cpu().numpy())))) for x, y in ((k64, k), (v64, v)))
            want, weight, delta = ref.attention(q[b].cpu().numpy(), kk, vv, len(kk))
            tol = weight * (2 * delta[..., None] * 2.0 ** -20 + 2.0 ** -18) + len(kk) * 2.0 ** -28 * np.abs(vv).max()
            assert np.all(np.abs(out[b].double().cpu().numpy() - want) <= tol)
    assert fault_bits() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_step_replays_in_a_graph(dtype):
    """Captured cold on a stream of its own; replays give what calls give, also after other calls on that stream."""
    want = run_step(step_case(dtype))
    s = step_case(dtype)
    images = [c.data.clone() for c in s["caches"]]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = run_step(s)
    assert all(torch.equal(c.data, i) for c, i in zip(s["caches"], images))
    for _ in range(3):
        for c, i in zip(s["caches"], images):
            c.data.copy_(i)
        with torch.cuda.stream(side):
            s["caches"][0].attend_tree(s["q"][0][:1].view(1, 1, *s["q"].shape[2:]), s["lens"][:1], ints([-1]), s["table"][:1])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want[0], got[0])) and all(torch.equal(a, b) for a, b in zip(want[1], got[1]))
    assert fault_bits() == 0


def test_calls_on_a_stream_of_their_own():
    want = run_step(step_case(torch.bfloat16))
    s = step_case(torch.bfloat16)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    from aljabr_b200.kv4 import accept_tree
    h = side.cuda_stream
    q = s["caches"][0].append_rotated(s["q"][0], s["k"][0], s["v"][0], s["slots"], s["positions"], s["rope"], stream=h)
    B, T = s["drafted"].shape
    out = s["caches"][0].attend_tree(q.view(B, T, *q.shape[1:]), s["lens"], s["parents"], s["table"], stream=h)
    got = accept_tree(s["caches"], s["lens"], s["parents"], s["drafted"], s["picked"], s["table"], stream=h)
    torch.cuda.synchronize()
    assert torch.equal(out, want[0][0]) and all(torch.equal(a, b) for a, b in zip(got, want[1]))


def test_results_repeat():
    for dtype in (torch.float32, torch.bfloat16):
        p = tree.grow(np.random.default_rng(13), 30)
        cache, q, sl, parents, table, _, _ = tree_case(13, 128, 2, 4, 16, [5000, 40, 2000], [p] * 3, dtype)
        out = cache.attend_tree(q, sl, parents, table)
        assert all(torch.equal(cache.attend_tree(q, sl, parents, table), out) for _ in range(5))


def test_a_cache_of_more_than_4_gib():
    """Rows and moves on pages beyond 2^32 bytes: 5 GB, the last pages in use."""
    from aljabr_b200.kv4 import accept_tree
    ps, D, hkv, pages = 64, 128, 8, 70000
    cache = make(pages, ps, hkv, D)
    assert cache.bytes > 5e9
    rng = np.random.default_rng(14)
    p = [-1, 0, 0, 2, 3]
    n, table = 130, ints([[pages - 1, pages - 3, pages - 2]])
    k, v = (rng.normal(size=(n, hkv, D)).astype(np.float32) for _ in range(2))
    slots = table[0].cpu().numpy()[np.arange(n) // ps] * ps + np.arange(n) % ps
    zero = torch.zeros(n, dtype=torch.int32, device="cuda")
    q = cuda(rng.normal(size=(n, 16, D)).astype(np.float32))
    rot = cache.append_rotated(q, cuda(k), cuda(v), cuda(slots.astype(np.int32)), zero, cuda(table_of(1, 64)))
    k64, v64 = ref.values(*ref.quantise(k)), ref.values(*ref.quantise(v))
    for dtype in (torch.float32, torch.bfloat16):
        qt = rot[-5:][None].to(dtype).contiguous()
        check(cache.attend_tree(qt, ints([n]), ints(p), table), qt, [k64], [v64], [n], [p])
    got = accept_tree(cache, ints([n]), ints(p), ints([[0, 1, 2, 3, 4]]), ints([[2, 0, 3, 9, 0]]), table)
    assert got[0].tolist() == [[0, 2, 3, -1, -1]] and [int(t) for t in got[1:]] == [3, 9, n - 2]
    kr, vr = cache.read(cuda(slots[-5:-2].astype(np.int32)))
    keep = [n - 5, n - 3, n - 2]
    assert np.array_equal(kr.cpu().numpy(), k64[keep].astype(np.float32)) and np.array_equal(vr.cpu().numpy(), v64[keep].astype(np.float32))
    del cache
    torch.cuda.empty_cache()
