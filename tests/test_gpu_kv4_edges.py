"""Edges of the 4-bit cache's attention, against 64 bits: values, scores and
queries of very unequal size, and arguments at the ends of their ranges."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from aljabr_b200 import native
from tests import kv4_ref as ref
from tests.test_gpu_kv4 import attend_case, check, fault_bits, make

pytestmark = pytest.mark.gpu


def one_sequence(k, v, dtype=torch.float32):
    """A cache of one sequence of the rows k, v [n][hkv][D], its table and length, and the values it holds."""
    n, hkv, D = k.shape
    pages = -(-n // 16)
    cache = make(pages, 16, hkv, D, fill=0xFF)
    cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), torch.arange(n, dtype=torch.int32, device="cuda"))
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    return (cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"), ref.values(*ref.quantise(k)),
            ref.values(*ref.quantise(v)))


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 5000])
def test_a_window_longer_than_every_sequence_is_none(window):
    """Sequences shorter than their new tokens, empty ones among them, with a window that 32 bits barely hold."""
    for T in (1, 3, 7):
        lens = [0, 1, 2, 300, 4000]
        cache, q, sl, table, out, k64, v64 = attend_case(23, 128, 2, 2, T, 16, lens)
        assert torch.equal(cache.attend(q, sl, table, window=window), out)
        check(out, q, k64, v64, lens)
    assert fault_bits() == 0


def test_a_page_of_more_than_2_to_the_30_positions():
    """The scales of V lie page_size + position rows into their section: a sum beyond 31 bits.  77 GB."""
    from aljabr_b200.kv4 import Kv4Cache
    ps, D, n = 2 ** 30 + 16, 64, 20
    if torch.cuda.mem_get_info()[0] < ps * 72 + 2 ** 30:
        pytest.skip("needs 78 GB")
    cache = Kv4Cache(1, ps, 1, D, data=torch.empty(ps * 72, dtype=torch.uint8, device="cuda"))
    rng = np.random.default_rng(24)
    k, v = (rng.normal(size=(n, 1, D)).astype(np.float32) for _ in range(2))
    slots = torch.arange(ps - n, ps, dtype=torch.int32, device="cuda")
    cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), slots)
    k64, v64 = ref.values(*ref.quantise(k)), ref.values(*ref.quantise(v))
    for got, want in zip(cache.read(slots), (k64, v64)):
        assert np.array_equal(got.cpu().numpy(), want.astype(np.float32))
    q = torch.from_numpy(rng.normal(size=(1, 1, 2, D)).astype(np.float32)).cuda()
    out = cache.attend(q, torch.tensor([ps], dtype=torch.int32, device="cuda"), window=n)
    check(out, q, [k64], [v64], [n])
    del cache
    torch.cuda.empty_cache()
    assert fault_bits() == 0


def test_device_swap_gives_the_choice_back():
    import ctypes
    before, now = ctypes.c_int(7), ctypes.c_int(7)
    native.call("aljabr_blackwell_device_swap", -1, ctypes.byref(before))
    try:
        native.call("aljabr_blackwell_device_swap", 0, ctypes.byref(now))
        assert now.value == -1
        for bad in (torch.cuda.device_count(), -2):
            with pytest.raises(native.ProviderError):
                native.call("aljabr_blackwell_device_swap", bad, ctypes.byref(now))
        native.call("aljabr_blackwell_device_swap", -1, ctypes.byref(now))
        assert now.value == 0
    finally:
        native.call("aljabr_blackwell_device_swap", before.value, ctypes.byref(now))


def test_a_table_without_pages_is_refused():
    """[batch, 0]: an empty tensor has no address, which would stand for 'sequence b is page b'."""
    cache = make(2, 16, 1, 64)
    q, lens = torch.zeros(1, 1, 1, 64, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(native.ProviderError):
        cache.attend(q, lens, torch.zeros(1, 0, dtype=torch.int32, device="cuda"))


def test_scores_far_below_zero_still_sum_to_one():
    """Equal scores of -1.1e31: the output is the mean of V, not zero."""
    rng = np.random.default_rng(21)
    k, v = np.full((40, 1, 128), -1.0, np.float32), rng.normal(size=(40, 1, 128)).astype(np.float32)
    cache, table, n, k64, v64 = one_sequence(k, v)
    out = cache.attend(torch.full((1, 1, 2, 128), 1e30, device="cuda"), n, table).double().cpu().numpy()
    weight, want = np.abs(v64).mean(0)[0], v64.mean(0)[0]
    # equal scores carry equal errors: what is left is P in two parts and fp32 sums, 2^-18 of sum P |v|
    assert np.all(np.abs(out[0, 0] - want) <= weight * 2.0 ** -18)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("at", [5, 17])      # a tile that is seen whole, and the sequence's last one
def test_a_nan_group_of_v_leaves_a_large_neighbour_finite(at, dtype):
    """A V row with NaN in one group and a scale of 5000 in the next, among rows of scale 0.1."""
    rng = np.random.default_rng(20)
    k, v = (rng.normal(size=(20, 1, 128)).astype(np.float32) for _ in range(2))
    v[at, 0, 32:64] *= 2e4
    cache, table, n, k64, v64 = one_sequence(k, v)
    bad = v.copy()
    bad[at, 0, 7] = np.nan
    cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(bad).cuda(), torch.arange(20, dtype=torch.int32, device="cuda"))
    q = torch.from_numpy(rng.normal(size=(1, 1, 2, 128)).astype(np.float32)).cuda().to(dtype)
    out = cache.attend(q, n, table)
    assert torch.isnan(out[..., :32]).all()
    want, weight, delta = ref.attention(q.float().cpu().numpy()[0], k64, v64, 20)
    # the bound of check() in tests/test_gpu_kv4.py, for the dims outside the NaN group
    tol = weight * (2 * delta[..., None] * 2.0 ** -20 + 2.0 ** (-18 if dtype == torch.float32 else -10)) + 20 * 2.0 ** -28 * np.abs(v64).max()
    tol += np.abs(want) * (2.0 ** -8 if dtype == torch.bfloat16 else 0)
    assert np.all((np.abs(out[0].double().cpu().numpy() - want) <= tol)[..., 32:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_absent_pages_between_others_in_a_long_sequence(dtype):
    """A page outside the cache counts as zeros: score 0, value 0.  Every slot of the ring is then loaded again."""
    lens, ps = [9000], 16
    cache, q, sl, table, _, k64, v64 = attend_case(25, 128, 1, 2, 1, ps, lens, dtype=dtype)
    gone = [3, 40, 41, 200, 333, 561]
    for i in gone:
        table[0, i] = -7 if i % 2 else 10 ** 8
        k64[0][i * ps:(i + 1) * ps] = 0.0
        v64[0][i * ps:(i + 1) * ps] = 0.0
    out = cache.attend(q, sl, table)
    assert fault_bits() & 2
    check(out, q, k64, v64, lens)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_outliers_of_q_do_not_cost_the_other_groups_their_bits(D):
    """q 300 times larger in one group of 32 (where K is small), K 100 times larger in another (where q is small).

    Bound of a score: q is off by at most 2^-23 of the largest value of its group of 32, so
    e = 2^-23 scale sum_g max|q_g| sum_g |k|, plus NG + 8 fp32 roundings of the groups' sums.  The output is then off by
    at most 2 e + 2^-18 (exp2, P in two parts, sums) of sum P |v|."""
    rng = np.random.default_rng(22 + D)
    n, heads, NG = 60, 16, D // 32
    k, v = (rng.normal(size=(n, 1, D)).astype(np.float32) for _ in range(2))
    q = rng.normal(size=(1, 1, heads, D)).astype(np.float32)
    k[..., :32] *= 0.05
    k[..., D - 5] *= 100
    q[..., 3] *= 300
    q[..., D - 32:] *= 0.1
    cache, table, lens, k64, v64 = one_sequence(k, v)
    out = cache.attend(torch.from_numpy(q).cuda(), lens, table).double().cpu().numpy()[0]
    want, weight, _ = ref.attention(q[0], k64, v64, n)
    scale = D ** -0.5
    top = np.abs(q[0, 0].astype(np.float64)).reshape(heads, NG, 32).max(-1)
    size = np.abs(k64[:, 0]).reshape(n, NG, 32).sum(-1)
    sums = np.abs(np.einsum("hgj,ngj->hng", q[0, 0].astype(np.float64).reshape(heads, NG, 32), k64[:, 0].reshape(n, NG, 32)))
    e = scale * (2.0 ** -23 * (top @ size.T).max(-1) + (NG + 8) * 2.0 ** -24 * 2 * sums.sum(-1).max(-1))
    err, tol = np.abs(out[0] - want[0]), weight[0] * (2 * e[:, None] + 2.0 ** -18) + n * 2.0 ** -28 * np.abs(v64).max()
    assert np.all(err <= tol), float((err / tol).max())
