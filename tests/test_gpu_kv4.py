"""The 4-bit KV cache on the GPU against a plain 64-bit implementation
(tests/kv4_ref.py): bytes written, values read back, attention."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from aljabr_b200 import native
from tests import kv4_ref as ref

pytestmark = pytest.mark.gpu


def fault_bits():
    torch.cuda.synchronize()
    bits = ctypes.c_uint(0)
    native.call("aljabr_blackwell_device_status", ctypes.byref(bits))
    return bits.value


def make(pages, page_size, hkv, D, fill=None):
    from aljabr_b200.kv4 import Kv4Cache
    data = None
    if fill is not None:
        size = native.lib().aljabr_blackwell_kv4_cache_size(pages, page_size, hkv, D)
        data = torch.full((size,), fill, dtype=torch.uint8, device="cuda")
    return Kv4Cache(pages, page_size, hkv, D, data=data)


def rows(rng, n, hkv, D, dtype):
    """Rows with groups of unequal size, a zero group, a tie of extremes and tiny values."""
    x = rng.normal(size=(n, hkv, D)) * np.exp(rng.normal(size=(n, hkv, D // 32, 1)).repeat(32, -1).reshape(n, hkv, D))
    x[0, 0, :32] = 0.0
    if n > 1:
        x[1, 0, :32] = np.clip(x[1, 0, :32], -1, 1)
        x[1, 0, 3], x[1, 0, 9] = 2.0, -2.0
    if n > 2:
        x[2, -1, -32:] *= 1e-7
    t = torch.from_numpy(x.astype(np.float32)).cuda().to(dtype)
    return t, t.float().cpu().numpy()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,hkv,D,ps", [(1, 1, 64, 16), (5, 3, 128, 48), (33, 2, 256, 16), (130, 8, 128, 64)])
def test_append_writes_the_documented_bytes(n, hkv, D, ps, dtype):
    rng = np.random.default_rng(n * D)
    pages = -(-n // ps) + 2
    cache = make(pages, ps, hkv, D, fill=0xA5)
    want = ref.RefCache(pages, ps, hkv, D, fill=0xA5)
    (k, kn), (v, vn) = rows(rng, n, hkv, D, dtype), rows(rng, n, hkv, D, dtype)
    slots = rng.permutation(pages * ps)[:n].astype(np.int32)
    if n > 3:
        slots[3] = -1
    back = [torch.full_like(k, 7.0) for _ in range(2)]
    cache.append(k, v, torch.from_numpy(slots).cuda(), k_back=back[0], v_back=back[1])
    for i, s in enumerate(slots):
        for h in range(hkv if s >= 0 else 0):
            want.write(int(s), h, kn[i, h], vn[i, h])
    assert np.array_equal(cache.data.cpu().numpy(), want.data)
    # the values handed back and read back are the codes' exact products (bf16: rounded once)
    read = cache.read(torch.from_numpy(slots).cuda(), dtype=dtype)
    for x, b, r in zip((kn, vn), back, read):
        exact = ref.values(*ref.quantise(x))
        exact[slots < 0] = 0.0
        exact = torch.from_numpy(exact.astype(np.float32)).to(dtype)
        assert torch.equal(b.cpu(), exact) and torch.equal(r.cpu(), exact)
    assert fault_bits() == 0


def test_quantisation_error_is_half_a_step():
    """A value is off by at most d / 2 (nearest code) where codes -8..7 reach it, by at most d where the side
    opposite the extreme is cut at 7 d (values up to 8 d); d's own rounding to fp16 adds 2^-11 of 8 d."""
    rng = np.random.default_rng(1)
    cache = make(4, 64, 4, 128)
    x, xn = rows(rng, 200, 4, 128, torch.float32)
    slots = torch.arange(200, dtype=torch.int32, device="cuda")
    cache.append(x, x, slots)
    got = cache.read(slots)[0].double().cpu().numpy()
    d = np.abs(xn).reshape(200, 4, 4, 32).max(-1).repeat(32, -1).reshape(xn.shape) / 8
    assert np.all(np.abs(got - xn) <= d * (1 + 2.0 ** -8) + 2.0 ** -24)
    inside = np.abs(xn) <= 7 * d
    assert np.all(np.abs(got - xn)[inside] <= d[inside] * (0.5 + 2.0 ** -8) + 2.0 ** -24)


def test_non_finite_groups_read_back_as_nan_and_large_ones_saturate():
    cache = make(1, 16, 1, 64)
    k = torch.ones(3, 1, 64, device="cuda")
    k[0, 0, 5], k[1, 0, 40], k[2, 0, 1] = float("nan"), float("-inf"), 3e38
    cache.append(k, -k, torch.arange(3, dtype=torch.int32, device="cuda"))
    kr, vr = (t.cpu().numpy()[:, 0] for t in cache.read(torch.arange(3, dtype=torch.int32, device="cuda")))
    for r in (kr, vr):
        assert np.isnan(r[0, :32]).all() and np.isfinite(r[0, 32:]).all()
        assert np.isnan(r[1, 32:]).all() and np.isfinite(r[1, :32]).all()
    assert kr[2, 1] == 8 * 65504.0 and vr[2, 1] == -8 * 65504.0 and (kr[2, 2:32] == 0).all()


def test_strided_and_unaligned_rows():
    rng = np.random.default_rng(2)
    for dtype, cut in ((torch.float32, 0), (torch.float32, 1), (torch.float32, 4), (torch.bfloat16, 0), (torch.bfloat16, 3)):
        wide = torch.from_numpy(rng.normal(size=(20, 3 * 256 + 8)).astype(np.float32)).cuda().to(dtype)
        k, v = wide[:, cut:cut + 256], wide[:, 256 + cut:512 + cut]
        a, b = make(2, 16, 2, 128), make(2, 16, 2, 128)
        slots = torch.arange(20, dtype=torch.int32, device="cuda")
        a.append(k, v, slots)
        b.append(k.contiguous(), v.contiguous(), slots)
        assert torch.equal(a.data, b.data)


def test_slots_outside_the_cache_are_skipped_and_reported():
    cache = make(2, 16, 1, 64)
    k = torch.ones(3, 1, 64, device="cuda")
    slots = torch.tensor([31, 32, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    cache.append(k, k, slots)
    assert fault_bits() & 2
    kr, _ = cache.read(slots)
    assert fault_bits() & 2
    assert (kr[0] == 1).all() and (kr[1:] == 0).all()
    assert fault_bits() == 0


# ---------------------------------------------------------------- attention
def attend_case(seed, D, hkv, G, T, ps, lens, window=0, soft_cap=0.0, dtype=torch.float32, paged=True, fill=0xFF,
                spread=1.5, pages=None, page0=0):
    """A cache whose unused bytes are `fill` (0xFF: scales that are NaN), random rows in use."""
    rng = np.random.default_rng(seed)
    B = len(lens)
    per = max(1, -(-max(lens) // ps))
    pages = pages or (page0 + B * per + 1)
    cache = make(pages, ps, hkv, D, fill=fill)
    order = (page0 + rng.permutation(B * per)).reshape(B, per) if paged else np.arange(B).reshape(B, 1)
    k64, v64 = [], []
    for b, n in enumerate(lens):
        k = rng.normal(size=(n, hkv, D)).astype(np.float32) * (0.3 + 2 * rng.random((1, hkv, D)) ** 4).astype(np.float32)
        v = rng.normal(size=(n, hkv, D)).astype(np.float32)
        if n:
            pos = np.arange(n)
            slots = torch.from_numpy((order[b, pos // ps] * ps + pos % ps).astype(np.int32)).cuda()
            cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), slots)
        k64.append(ref.values(*ref.quantise(k)) if n else k.astype(np.float64))
        v64.append(ref.values(*ref.quantise(v)) if n else v.astype(np.float64))
    q = torch.from_numpy((rng.normal(size=(B, T, hkv * G, D)) * spread).astype(np.float32)).cuda().to(dtype)
    table = None
    if paged:
        t = order.astype(np.int32)
        for b, n in enumerate(lens):
            t[b, -(-n // ps):] = -1          # entries past a sequence are never followed
        table = torch.from_numpy(t).cuda()
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = cache.attend(q, sl, table, window=window, soft_cap=soft_cap)
    return cache, q, sl, table, out, k64, v64


def check(out, q, k64, v64, lens, window=0, soft_cap=0.0):
    """Bound of one output: score errors e (q in 22 bits of its row's largest value, fp32 sums of the offset codes and
    of the scaling: 2^-20 of delta, see attention()) change P by at most 2 e relative, hence the output by
    2 e sum P |v|; exp2, the two-part P' (2^-22) and fp32 sums add 2^-18 of it; P' keeps 2^-30 of the largest V, a
    position.  bf16: P' in one part and an output rounded to 8 bits: 2^-10 of sum P |v| and 2^-8 of the output."""
    qn = q.float().cpu().numpy()
    on = out.double().cpu().numpy()
    bf16 = q.dtype == torch.bfloat16
    for b, n in enumerate(lens):
        want, weight, delta = ref.attention(qn[b], k64[b], v64[b], n, window=window, soft_cap=soft_cap)
        floor = n * 2.0 ** -28 * (np.abs(v64[b]).max() if n else 0.0)
        tol = weight * (2 * delta[..., None] * 2.0 ** -20 + 2.0 ** (-10 if bf16 else -18)) + floor
        if bf16:
            tol = tol + np.abs(want) * 2.0 ** -8
        err = np.abs(on[b] - want)
        assert np.all(err <= tol), (b, n, float(err.max()), float((err / np.maximum(tol, 1e-300)).max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,hkv,G,T,ps,lens,window,cap", [
    (128, 2, 4, 1, 16, [1], 0, 0.0),
    (128, 8, 4, 1, 64, [0, 1, 15, 16, 17, 127, 128, 129, 257], 0, 0.0),
    (128, 1, 1, 1, 4096, [3000], 0, 0.0),
    (128, 2, 8, 1, 48, [700, 5000, 3], 0, 0.0),
    (128, 1, 16, 1, 32, [333, 64], 0, 0.0),
    (128, 2, 3, 5, 16, [5, 4, 200, 0, 1], 0, 0.0),
    (128, 1, 8, 7, 64, [900], 100, 0.0),
    (64, 4, 2, 1, 16, [77, 1024], 0, 30.0),
    (64, 3, 7, 3, 16, [40, 2, 513], 33, 0.0),
    (256, 2, 4, 1, 16, [19, 640], 0, 0.0),
    (256, 1, 5, 4, 80, [400, 33], 7, 50.0),
])
def test_attention_matches_64_bits(D, hkv, G, T, ps, lens, window, cap, dtype):
    _, q, _, _, out, k64, v64 = attend_case(D + G + T, D, hkv, G, T, ps, lens, window, cap, dtype)
    check(out, q, k64, v64, lens, window, cap)
    assert fault_bits() == 0


def test_attention_without_a_table_and_many_sequences():
    lens = [int(n) for n in np.random.default_rng(5).integers(0, 65, 300)]
    _, q, _, _, out, k64, v64 = attend_case(5, 64, 2, 2, 1, 64, lens, paged=False)
    check(out, q, k64, v64, lens)


def test_rows_that_see_nothing_are_zero():
    _, q, sl, table, out, _, _ = attend_case(6, 128, 2, 4, 4, 16, [0, 2, 4])
    o = out.cpu().numpy()
    assert (o[0] == 0).all() and (o[1, :2] == 0).all() and np.isfinite(o).all()
    assert np.abs(o[1, 2:]).max(-1).min() > 0 and np.abs(o[2]).max(-1).min() > 0


def test_masked_nan_rows_do_not_leak():
    """Rows outside the window, and rows later drafted tokens wrote, may hold NaN."""
    lens, T, window = [200], 3, 64
    cache, q, sl, table, _, k64, v64 = attend_case(7, 128, 2, 4, T, 16, lens, window)
    bad = torch.full((2, 2, 128), float("nan"), device="cuda")
    where = [100, 199]      # before every window; seen by the last query only
    slots = [int(table[0, p // 16]) * 16 + p % 16 for p in where]
    cache.append(bad, bad, torch.tensor(slots, dtype=torch.int32, device="cuda"))
    out = cache.attend(q, sl, table, window=window)
    assert torch.isnan(out[0, 2]).all()
    for t in (0, 1):
        want, weight, delta = ref.attention(q[0, t:t + 1].cpu().numpy(), k64[0], v64[0], 198 + t, window=window)
        assert np.all(np.abs(out[0, t].double().cpu().numpy() - want[0]) <= weight[0] * (2 * delta[0][:, None] * 2.0 ** -20 + 2.0 ** -9))


def test_nan_scales_stay_in_their_dims():
    cache, q, sl, table, _, _, _ = attend_case(8, 128, 1, 2, 1, 16, [40])
    k, v = cache.read(torch.tensor([int(table[0, 0]) * 16], dtype=torch.int32, device="cuda"))
    v[0, 0, 33] = float("inf")
    cache.append(k, v, torch.tensor([int(table[0, 0]) * 16], dtype=torch.int32, device="cuda"))
    o = cache.attend(q, sl, table).cpu().numpy()[0, 0]
    assert np.isnan(o[:, 32:64]).all() and np.isfinite(o[:, :32]).all() and np.isfinite(o[:, 64:]).all()


@pytest.mark.parametrize("factor", [0.0, 1e-30, 1e-6, 1e6])
def test_queries_of_any_size(factor):
    cache, q, sl, table, _, k64, v64 = attend_case(9, 128, 2, 2, 1, 16, [150])
    qf = q * factor
    check(cache.attend(qf, sl, table), qf, k64, v64, [150])


def test_non_finite_queries_stay_in_their_rows():
    for dtype in (torch.float32, torch.bfloat16):
        cache, q, sl, table, out, _, _ = attend_case(16, 128, 2, 4, 1, 16, [70], dtype=dtype)
        bad = q.clone()
        bad[0, 0, 1, 5], bad[0, 0, 6, 0] = float("nan"), float("inf")
        got = cache.attend(bad, sl, table)
        assert torch.isnan(got[0, 0, [1, 6]]).all()
        rest = [0, 2, 3, 4, 5, 7]
        assert torch.equal(got[0, 0, rest], out[0, 0, rest])


def test_wrapper_refusals():
    cache = make(4, 16, 2, 64)
    k = torch.zeros(3, 2, 64, device="cuda")
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 1, 4, 64, device="cuda")
    lens, table = torch.ones(1, dtype=torch.int32, device="cuda"), torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    bad = native.ProviderError
    for call in (lambda: cache.append(k.cpu(), k, slots), lambda: cache.append(k, k[:2], slots),
                 lambda: cache.append(k, k.bfloat16(), slots), lambda: cache.append(k.half(), k.half(), slots),
                 lambda: cache.append(k, k, slots.long()), lambda: cache.append(k, k, slots, k_back=torch.empty_like(k)),
                 lambda: cache.append(k.transpose(1, 2), k, slots), lambda: cache.read(slots, dtype=torch.float16),
                 lambda: cache.read(slots[::2]), lambda: cache.attend(q[0], lens, table),
                 lambda: cache.attend(q, lens.long(), table), lambda: cache.attend(q, lens, table[:, ::2]),
                 lambda: cache.attend(q, lens, table, out=torch.empty(1, 1, 4, 64, device="cuda", dtype=torch.bfloat16)),
                 lambda: cache.attend(torch.zeros(1, 1, 3, 64, device="cuda"), lens, table),
                 lambda: cache.attend(q, lens, table, window=-1)):
        with pytest.raises(bad):
            call()
    with pytest.raises(native.UnsupportedOperation):
        make(4, 16, 2, 96)


def test_values_of_very_different_size():
    """A first position with nearly all the weight and tiny values, as attention sinks have."""
    rng = np.random.default_rng(10)
    cache = make(64, 16, 1, 128)
    n = 1000
    k, v = rng.normal(size=(n, 1, 128)).astype(np.float32) * 0.1, rng.normal(size=(n, 1, 128)).astype(np.float32)
    k[0] = 4.0
    v[0] *= 1e-4
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    cache.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), slots)
    k64, v64 = ref.values(*ref.quantise(k)), ref.values(*ref.quantise(v))
    q = torch.full((1, 1, 4, 128), 0.25, device="cuda")
    table = torch.arange(64, dtype=torch.int32, device="cuda")[None]
    out = cache.attend(q, torch.tensor([n], dtype=torch.int32, device="cuda"), table)
    check(out, q, [k64], [v64], [n])


def test_results_repeat_and_leave_the_workspace_ready():
    cache, q, sl, table, out, k64, v64 = attend_case(11, 128, 2, 4, 1, 16, [4000, 100, 9000])
    for _ in range(3):
        assert torch.equal(cache.attend(q, sl, table), out)
    work, = cache._buffers.values()
    assert int(work[:1024].int().sum()) == 0
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = cache.attend(q, sl, table)
    s.synchronize()
    assert torch.equal(again, out) and len(cache._buffers) == 2


def test_call_replays_in_a_graph_with_growing_lengths():
    """Lengths and slots are read on the device, so one captured step serves every token."""
    cache, q, sl, table, _, k64, v64 = attend_case(12, 128, 2, 4, 1, 16, [500], fill=0)
    k, v = torch.randn(1, 2, 128, device="cuda"), torch.randn(1, 2, 128, device="cuda")
    slot = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)

    def one():
        cache.append(k, v, slot)
        cache.attend(q, sl, table, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        slot.fill_(int(table[0, 31]) * 16 + 15)
        one()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        one()
    for p in (500, 501):
        k.normal_(), v.normal_()
        slot.fill_(int(table[0, p // 16]) * 16 + p % 16)
        sl.fill_(p + 1)
        graph.replay()
        torch.cuda.synchronize()
        k64[0] = np.concatenate([k64[0][:p], ref.values(*ref.quantise(k.cpu().numpy()))])
        v64[0] = np.concatenate([v64[0][:p], ref.values(*ref.quantise(v.cpu().numpy()))])
        check(out, q, k64, v64, [p + 1])


def test_pages_and_lengths_outside_the_cache_are_not_followed():
    cache, q, sl, table, out, _, _ = attend_case(13, 128, 2, 4, 1, 16, [64, 64])
    broken = table.clone()
    broken[0, 1], broken[0, 2] = 10 ** 6, -5
    got = cache.attend(q, sl, broken)
    assert fault_bits() & 2
    assert torch.equal(got[1], out[1]) and torch.isfinite(got).all()
    got = cache.attend(q, torch.tensor([64, 10 ** 6], dtype=torch.int32, device="cuda"), table)
    assert fault_bits() & 2
    assert torch.equal(got, out)
    got = cache.attend(q, torch.tensor([-3, 64], dtype=torch.int32, device="cuda"), table)
    assert fault_bits() & 2
    assert (got[0] == 0).all() and torch.equal(got[1], out[1])


def test_cache_of_more_than_4_gib():
    """Pages behind the 2^32nd byte: 8 heads x 128 dims x 64 positions are 73,728 bytes a page."""
    pages = 2 ** 32 // 73728 + 200
    lens = [1000, 130]
    _, q, _, _, out, k64, v64 = attend_case(14, 128, 8, 4, 1, 64, lens, pages=pages, page0=pages - 60)
    check(out, q, k64, v64, lens)


def test_strided_queries():
    cache, q, sl, table, out, _, _ = attend_case(15, 128, 2, 4, 2, 16, [90, 33, 7])
    wide = torch.zeros(3, 2, 12 * 128, device="cuda")
    wide[..., :8 * 128] = q.flatten(2)
    view = wide[..., :8 * 128].unflatten(2, (8, 128))
    assert torch.equal(cache.attend(view, sl, table), out)
