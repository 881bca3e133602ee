"""Attention of drafted trees where its steps meet their limits: scores and
values that rise from chunk to chunk, scales far apart, pages given back, the
row count at which the kernel changes."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests import kv4_ref as ref
from tests import tree_ref as tree
from tests.test_gpu_kv4 import fault_bits, make
from tests.test_gpu_kv4_tree import check, cuda, ints, tree_case, widen

pytestmark = pytest.mark.gpu


def one_sequence(k, v, ps=64, wide=True):
    """A cache that holds k, v [n][hkv][D] on pages in another order, its table, and the values it stands for."""
    n, hkv, D = k.shape
    per = -(-n // ps)
    order = np.random.default_rng(n).permutation(per)
    cache = make(per, ps, hkv, D)
    at = np.arange(n)
    cache.append(cuda(k), cuda(v), cuda((order[at // ps] * ps + at % ps).astype(np.int32)))
    table = order[None].astype(np.int32)
    return cache, cuda(widen(table, ps) if wide else table), ref.values(*ref.quantise(k)), ref.values(*ref.quantise(v))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rise", [6.0, 3.0, 40.0])
def test_scores_and_values_that_rise_from_chunk_to_chunk(D, rise):
    """Of 32 positions to the next the scores rise by 2^rise in the weights, and every 128 positions V's scales by 2^3, so
    that the running maximum is raised up to four times a tile and what is summed up is scaled on the way.

    The scores are exact: q is 1, K one value of a position in 32 dims, a multiple of a power of two.  So what may differ is fp32's
    rounding of a score (to 2^-22 of the largest, twice), P and V in fp16 (2^-11 each) and the output's 2^-8."""
    T, n = 72, 72 + 1024
    p = tree.grow(np.random.default_rng(D), T)
    rng = np.random.default_rng(60)
    k = np.zeros((n, 1, D), np.float32)
    unit = rise * np.log(2.0) / 32.0              # of a score without its scale; K takes 8 bits of it
    unit = 2.0 ** np.floor(np.log2(unit)) * np.round(256 * unit / 2.0 ** np.floor(np.log2(unit))) / 256
    level = np.minimum(np.arange(n) // 32, 32)
    k[:, 0, 32:64] = level[:, None]
    v = rng.normal(size=(n, 1, D)).astype(np.float32) * (2.0 ** (np.minimum(np.arange(n) // 128, 8) * 3 - 14.0))[:, None, None].astype(np.float32)
    cache, table, k64, v64 = one_sequence(k, v)
    assert np.array_equal(k64, k)                 # multiples of 1/8 of the level
    q = torch.ones(1, T, 1, D, device="cuda", dtype=torch.bfloat16)
    got = cache.attend_tree(q, ints([n]), ints([p]), table, scale=unit).double().cpu().numpy()[0, :, 0]
    for t, rows in enumerate(tree.visible(p, n)):
        s = (k64[rows, 0] @ np.ones(D)) * np.float64(np.float32(unit))
        w = np.exp(s - s.max())
        w /= w.sum()
        want, weight = w @ v64[rows, 0], w @ np.abs(v64[rows, 0])
        tol = weight * (2 * 2 * np.abs(s).max() * 2.0 ** -22 + 2.0 ** -10) + np.abs(want) * 2.0 ** -8 + n * 2.0 ** -24 * np.abs(v64[rows, 0]).max(0)
        err = np.abs(got[t] - want)
        assert np.all(err <= tol), (t, float((err / tol).max()))
    assert fault_bits() == 0


@pytest.mark.parametrize("nodes,G", [(32, 1), (33, 1), (16, 2), (17, 2), (4, 8), (5, 8)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_at_which_the_kernel_changes(D, nodes, G):
    """32 rows and the next count, in a table wide enough for either kernel."""
    lens = [700, nodes, 260]
    trees = [tree.grow(np.random.default_rng(63 + b), nodes, 1, nodes // 8) for b in range(3)]
    cache, q, sl, parents, table, k64, v64 = tree_case(64, D, 2, G, 16, lens, trees, torch.bfloat16, wide=True)
    for window in (0, 90):
        check(cache.attend_tree(q, sl, parents, table, window=window), q, k64, v64, lens, trees, window)
    assert fault_bits() == 0


@pytest.mark.parametrize("dtype,pad", [(torch.float32, 0), (torch.bfloat16, 0), (torch.bfloat16, 60)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("power,size", [(-8, 0), (-16, 0), (-20, 0), (-14, 12), (-20, 12)])
def test_groups_of_far_smaller_scales(D, power, size, dtype, pad):
    """V and K are of size 2^size, but their second 32 dims 2^power of that (at 2^0 scales of 2^-20 are fp16's last bits in the
    cache itself); the queries there are as much larger.  Outputs of those dims and scores are as near as any.  A score is
    off by 2^-11 of its products (bf16) and fp32's sums, P and V by 2^-11 each; the limits go by each dim's own values,
    with 2^-24 of its largest for weights at fp16's lower end.  fp32: a weight times its scale enters to 2^-28 of the largest
    V there is, whatever its dim's are, each position for itself."""
    bf16 = dtype == torch.bfloat16
    T, n, hkv, G = 21 + pad, 300 + pad, 2, 2
    rng = np.random.default_rng(D)
    p = tree.grow(rng, 21, 1, 2) + [-2] * pad
    k, v = (rng.normal(size=(n, hkv, D)).astype(np.float32) for _ in range(2))
    k, v = k * np.float32(2.0 ** size), v * np.float32(2.0 ** size)
    k[..., 32:64] *= np.float32(2.0 ** power)
    v[..., 32:64] *= np.float32(2.0 ** power)
    q = rng.normal(size=(1, T, hkv * G, D)).astype(np.float32) * np.float32(0.5 * 2.0 ** -size)
    q[..., 32:64] *= np.float32(2.0 ** -power)
    cache, table, k64, v64 = one_sequence(k, v, wide=pad > 0)
    qt = cuda(q, dtype)
    got = cache.attend_tree(qt, ints([n]), ints([p]), table).double().cpu().numpy()[0]
    qn = qt.double().cpu().numpy()[0]
    off, norm, floor = np.zeros(D // 32), np.zeros(D // 32), 0.0
    for t, rows in enumerate(tree.visible(p, n)):
        for h in range(hkv * G):
            if not rows:
                assert not got[t, h].any()
                continue
            kk, vv = k64[rows, h // G], v64[rows, h // G]
            s = kk @ qn[t, h] * D ** -0.5
            w = np.exp(s - s.max())
            w /= w.sum()
            want, weight = w @ vv, w @ np.abs(vv)
            # fp32: an element of q to 2^-23 of its group's largest, whose codes enter with the offset 8
            far = np.abs(kk) @ np.abs(qn[t, h]) if bf16 else (np.abs(qn[t, h]).reshape(-1, 32).max(-1).repeat(32) * (np.abs(kk) + 8 / 7 * np.abs(kk).reshape(len(kk), -1, 32).max(-1).repeat(32, -1))).sum(-1)
            delta = D ** -0.5 * far.max() * 2.0 ** (-11 if bf16 else -20) + np.abs(s).max() * 2.0 ** -20
            tol = weight * (np.expm1(2 * delta) + 2.0 ** (-10 if bf16 else -18)) + n * (2.0 ** -24 * np.abs(vv).max(0) if bf16 else 2.0 ** -28 * np.abs(vv).max())
            floor += 32 * len(rows) * (0.0 if bf16 else 2.0 ** -28 * np.abs(vv).max()) ** 2
            if bf16:
                tol = tol + np.abs(want) * 2.0 ** -8
            err = np.abs(got[t, h] - want)
            assert np.all(err <= tol), (t, h, int((err / tol).argmax()), float((err / tol).max()))
            off += (err ** 2).reshape(-1, 32).sum(-1)
            norm += (want ** 2).reshape(-1, 32).sum(-1)
    # by norm, each group for itself: rounding errors do not add up
    assert np.all(off <= norm * (2.0 ** -8 if bf16 else 2.0 ** -18) ** 2 + floor), np.sqrt(off / norm)
    assert fault_bits() == 0


@pytest.mark.parametrize("dtype,pad", [(torch.float32, 0), (torch.bfloat16, 0), (torch.bfloat16, 60)])
@pytest.mark.parametrize("D,ps,window", [(128, 16, 100), (64, 16, 33), (256, 16, 100), (128, 64, 1), (128, 48, 500)])
def test_pages_given_back_behind_the_window(D, ps, window, dtype, pad):
    """A server gives pages back that no window reaches any more; their entries are -1 or no page of this pool.  That is no
    fault, and one page further on it is."""
    lens = [1000 + pad, 300 + pad, 22 + pad]
    p = tree.grow(np.random.default_rng(61), 21, 2, 1) + [-2] * pad
    T = len(p)
    cache, q, sl, parents, table, k64, v64 = tree_case(62, D, 2, 2, ps, lens, [p] * 3, dtype, wide=pad > 0)
    want = cache.attend_tree(q, sl, parents, table, window=window)
    check(want, q, k64, v64, lens, [p] * 3, window)
    first = [max(0, n - T + 1 - window) // ps for n in lens]      # the first page that a root at the tree's base may see
    assert first[0] > 0 and fault_bits() == 0
    for gone in (-1, cache.pages, 2 ** 31 - 1):
        cut = table.clone()
        for b, f in enumerate(first):
            cut[b, :f] = gone
        assert torch.equal(cache.attend_tree(q, sl, parents, cut, window=window), want)
        assert fault_bits() == 0
        cut[0, first[0]] = gone
        cache.attend_tree(q, sl, parents, cut, window=window)
        assert fault_bits() & 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pages_given_back_behind_a_chain_s_window(dtype):
    lens, T, window, ps = [1000, 300, 40], 5, 100, 16
    cache, q, sl, _, table, _, _ = tree_case(65, 128, 2, 4, ps, lens, [list(range(-1, T - 1))] * 3, dtype)
    want = cache.attend(q, sl, table, window=window)
    cut = table.clone()
    for b, n in enumerate(lens):
        cut[b, :max(0, n - T + 1 - window) // ps] = 2 ** 31 - 1
    assert torch.equal(cache.attend(q, sl, cut, window=window), want) and fault_bits() == 0
