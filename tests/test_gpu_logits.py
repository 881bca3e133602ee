"""The logits step on the GPU against numpy: fp32 operations in the documented
order give the same bits, and 64 bits bound them."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def reference(x, history, penalties, bias, allow, dtype):
    """x [vocab] of dtype; history: list of tokens; bias: list of (token, value); allow: bool [vocab] or None."""
    x = x.astype(dtype).copy()
    vocab = len(x)
    rep, freq, pres = (dtype(p) for p in penalties)
    tokens, counts = np.unique([t for t in history if 0 <= t < vocab], return_counts=True)
    with np.errstate(all="ignore"):
        for t, n in zip(tokens.astype(int), counts):
            v = x[t] / rep if x[t] > 0 else x[t] * rep
            x[t] = (v - freq * dtype(n)) - pres
        add = {}
        for t, b in bias:
            if 0 <= t < vocab:
                add[t] = add.get(t, dtype(0)) + dtype(b)
        for t, b in add.items():
            x[t] = x[t] + b
    ok = np.ones(vocab, bool) if allow is None else allow
    x[~ok] = -np.inf
    can = ok & ~np.isnan(x)
    token = int(np.flatnonzero(can & (x == x[can].max()))[0]) if can.any() else -1
    return x, token


def run(x, hist=None, pen=None, bias=None, allow=None, **kw):
    """Ragged lists -> padded tensors (padding: values that must not be read as live)."""
    from aljabr_b200.logits import process_logits
    rows, vocab = x.shape
    a = {}
    if hist is not None:
        n = max(1, max(len(h) for h in hist))
        m = np.full((rows, n), 1, np.int32)
        for i, h in enumerate(hist):
            m[i, :len(h)] = h
        a.update(history=m, history_len=np.array([len(h) for h in hist], np.int32), penalties=np.asarray(pen, np.float32))
    if bias is not None:
        n = max(1, max(len(b) for b in bias))
        t, w = np.full((rows, n), 2, np.int32), np.full((rows, n), 1e9, np.float32)
        for i, b in enumerate(bias):
            t[i, :len(b)], w[i, :len(b)] = [e[0] for e in b], [e[1] for e in b]
        a.update(bias_tokens=t, bias_values=w, bias_len=np.array([len(b) for b in bias], np.int32))
    if allow is not None:
        words = np.zeros((rows, (vocab + 31) // 32 + 1), np.uint32)
        for i in range(rows):
            bits = np.zeros(words.shape[1] * 32, np.uint8)
            bits[:vocab] = allow[i]
            bits[vocab:] = 1         # bits past the vocabulary mean nothing
            words[i] = np.packbits(bits, bitorder="little").view(np.uint32)
        a["allow"] = words.view(np.int32)
    out, token = process_logits(x, **{k: torch.from_numpy(v).cuda() for k, v in a.items()}, **kw)
    return out.cpu().numpy(), token.cpu().numpy()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 31), (3, 33), (1, 1000), (5, 32003), (2, 131077), (40, 4096), (1, 300001)])
def test_matches_the_formula(rows, vocab, dtype):
    rng = np.random.default_rng(vocab)
    x = torch.from_numpy((rng.normal(size=(rows, vocab)) * 4).astype(np.float32)).cuda().to(dtype)
    few = rng.integers(0, vocab, 20)
    hist = [list(rng.choice(few, rng.integers(0, 60))) + [-1, vocab, vocab + 7] for _ in range(rows)]
    pen = [[rng.uniform(0.8, 1.5), rng.uniform(-0.5, 1), rng.uniform(0, 1)] for _ in range(rows)]
    bias = [[(int(rng.integers(-1, vocab + 1)), float(rng.normal() * 3)) for _ in range(rng.integers(0, 70))] for _ in range(rows)]
    allow = rng.random((rows, vocab)) < 0.6
    out, token = run(x, hist, pen, bias, allow)
    xn = x.float().cpu().numpy()
    pen = np.asarray(pen, np.float32)
    for i in range(rows):
        b32 = [(t, np.float32(b)) for t, b in bias[i]]
        want, best = reference(xn[i], hist[i], pen[i], b32, allow[i], np.float32)
        assert np.array_equal(out[i], want) and token[i] == best
        # 64 bits: at most 5 roundings of values no larger than this
        exact, _ = reference(xn[i], hist[i], pen[i], b32, allow[i], np.float64)
        fine = np.isfinite(exact)
        size = np.abs(xn[i]) * 1.6 + 70 + sum(abs(b) for _, b in bias[i])
        assert np.all(np.abs(out[i] - exact)[fine] <= (5 + len(bias[i])) * 2.0 ** -24 * size[fine])


def test_repeated_biases_add_in_list_order():
    x = torch.zeros(1, 100, device="cuda")
    vals = [1e8, 1.0, -1e8, 3.0] * 20 + [0.5]
    out, token = run(x, bias=[[(7, b) for b in vals]])
    want = np.float32(0)
    for b in vals:
        want = np.float32(want + np.float32(b))
    assert out[0, 7] == want and np.all(out[0, np.arange(100) != 7] == 0)


def test_each_part_alone_and_in_place():
    from aljabr_b200.logits import process_logits
    rng = np.random.default_rng(3)
    x = rng.normal(size=(3, 5000)).astype(np.float32)
    t = torch.from_numpy(x).cuda()
    out, token = run(t)
    assert np.array_equal(out, x) and np.array_equal(token, x.argmax(1))
    out, token = run(t, hist=[[4, 4], [], [9]], pen=[[2, 0.5, 0.25]] * 3)
    for i, h in enumerate([[4, 4], [], [9]]):
        assert np.array_equal(out[i], reference(x[i], h, (2, 0.5, 0.25), [], None, np.float32)[0])
    mask = torch.from_numpy(rng.integers(-2 ** 31, 2 ** 31, (3, 157)).astype(np.int32)).cuda()
    apart, a = process_logits(t, allow=mask)
    same, b = process_logits(t, allow=mask, out=t)
    assert same.data_ptr() == t.data_ptr() and torch.equal(apart, same) and torch.equal(a, b)


def test_ties_nan_and_empty_rows():
    x = np.zeros((6, 40000), np.float32)
    x[0, [39000, 123, 20000]] = 5.0                     # ties go to the lowest index
    x[1] = np.nan
    x[1, 777] = -np.inf                                 # the only candidate
    x[2, 3] = np.nan
    x[2, 9] = 1.0
    x[3] = np.nan                                       # no candidate
    x[4] = -0.0
    x[4, 17] = 0.0                                      # -0 and +0 tie: index 0
    allow = np.ones((6, 40000), bool)
    allow[5] = False                                    # nothing allowed
    out, token = run(torch.from_numpy(x).cuda(), allow=allow)
    assert token.tolist() == [123, 777, 9, -1, 0, -1]
    assert np.isneginf(out[5]).all() and np.isnan(out[3]).all()


def test_rows_with_nothing_above_minus_infinity():
    """All allowed logits -inf: the lowest allowed index that is no listed token is as good as any, so the lowest of all
    allowed ones wins; in place too."""
    from aljabr_b200.logits import process_logits
    x = np.full((2, 20000), -np.inf, np.float32)
    allow = np.zeros((2, 20000), bool)
    allow[0, [13000, 400, 19999]] = True
    allow[1, [7, 9]] = True
    for in_place in (False, True):
        t = torch.from_numpy(x).cuda()
        out, token = run(t, hist=[[400], [9]], pen=[[1.1, 0.1, 0.1]] * 2, allow=allow, **({"out": t} if in_place else {}))
        assert token.tolist() == [400, 7] and np.isneginf(out).all()


def test_wrapper_refusals():
    from aljabr_b200 import native
    from aljabr_b200.logits import process_logits
    x = torch.zeros(2, 64, device="cuda")
    h, n, p = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.ones(2, 3, device="cuda")
    for kw in (dict(history=h), dict(history=h, history_len=n), dict(history=h, history_len=n[:1], penalties=p),
               dict(history=h.long(), history_len=n, penalties=p), dict(history=h, history_len=n, penalties=p.t()),
               dict(bias_tokens=h), dict(allow=h[:, :1]), dict(allow=h.cpu()), dict(out=x.bfloat16()), dict(token=n.long())):
        with pytest.raises(native.ProviderError):
            process_logits(x, **kw)
    with pytest.raises(native.ProviderError):
        process_logits(x.cpu())
    with pytest.raises(native.UnsupportedOperation):
        process_logits(x.half())


def test_strided_rows_and_long_histories():
    rng = np.random.default_rng(4)
    wide = torch.from_numpy(rng.normal(size=(4, 9001)).astype(np.float32)).cuda()
    x = wide[:, 1:8990]
    hist = [list(rng.integers(0, 50, 20000)) for _ in range(4)]
    out, token = run(x, hist=hist, pen=[[1.2, 0.01, 0.1]] * 4)
    for i in range(4):
        want, best = reference(x[i].cpu().numpy(), hist[i], np.float32([1.2, 0.01, 0.1]), [], None, np.float32)
        assert np.array_equal(out[i], want) and token[i] == best
