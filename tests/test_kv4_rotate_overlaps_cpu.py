"""Arguments of the rotated append that overlap: refused before the GPU is
touched, rows between other rows taken."""
import numpy as np
import pytest

from aljabr_b200 import native
from tests.test_kv4_tree_cpu import rotate

M = 1 << 24      # far apart
PLACES = dict(cache=M, qo=2 * M, q=3 * M, k=4 * M, v=5 * M, slots=6 * M, pos=7 * M, rope=8 * M + 8)
REFUSED = "must not", "may be written"


def refused(**kw):
    """Whether a call (fp32, 3 tokens, q rows of 4096 bytes, k and v rows of 1024) is refused for an overlap.  Every call here
    is refused, if for nothing else because rope is not aligned, which is looked at last."""
    args = dict(PLACES, **kw)
    assert args["rope"] % 16 == 8 and rotate(**args) == native.ALJ_ERR_BAD_ARG
    why = native.last_error()
    assert any(r in why for r in REFUSED) != ("aligned" in why)
    return "aligned" not in why


@pytest.mark.parametrize("kw,want", [
    (dict(), False),
    # q_out against q
    (dict(qo=3 * M), False), (dict(qo=3 * M + 4), True), (dict(qo=3 * M + 4096), True), (dict(qo=3 * M + 3 * 4096), False),
    (dict(qo=3 * M, qos=2048), True), (dict(qo=3 * M, qos=2048, n=1), False), (dict(qo=3 * M - 4096), True), (dict(qo=3 * M - 3 * 4096), False),
    (dict(qo=3 * M + 4096, qos=2048, qs=2048), False), (dict(qo=3 * M + 4092, qos=2048, qs=2048), True),
    (dict(qo=3 * M - 4096, qos=2048, qs=2048), False),
    # q_out against k and v, q in place: the columns of one buffer q | k | v, 6144 bytes a row
    (dict(qo=M * 3, q=M * 3, k=M * 3 + 4096, v=M * 3 + 5120, qs=1536, qos=1536, ks=1536, vs=1536), False),
    (dict(qo=M * 3, q=M * 3, k=M * 3 + 4092, v=M * 3 + 5120, qs=1536, qos=1536, ks=1536, vs=1536), True),
    (dict(qo=M * 3, q=M * 3, k=M * 3 + 4096, v=M * 3 + 6144 - 1020, qs=1536, qos=1536, ks=1536, vs=1536), True),
    (dict(qo=M * 4, k=M * 4), True), (dict(qo=5 * M - 3 * 4096), False), (dict(qo=5 * M - 3 * 4096 + 4), True), (dict(qo=5 * M + 2 * 1024 + 1020), True),
    (dict(qo=5 * M + 3 * 1024), False), (dict(qo=4 * M, n=1), True),
    # k_back and v_back
    (dict(kb=9 * M, vb=10 * M), False), (dict(kb=4 * M, vb=5 * M), False), (dict(kb=4 * M + 4, vb=10 * M), True),
    (dict(kb=4 * M, vb=10 * M, ks=512), True), (dict(kb=5 * M, vb=4 * M), True), (dict(kb=9 * M, vb=9 * M), True),
    (dict(kb=9 * M, vb=9 * M + 3 * 1024 - 4), True), (dict(kb=9 * M, vb=9 * M + 3 * 1024), False), (dict(kb=3 * M + 8, vb=9 * M), True),
    (dict(kb=9 * M, vb=2 * M + 3 * 4096 - 4), True), (dict(kb=9 * M, vb=2 * M + 3 * 4096), False),
    # what is read by all, and the cache (4 pages of 16 positions, 2 heads of 128: 18432 bytes)
    (dict(qo=6 * M), True), (dict(slots=2 * M + 12284), True), (dict(slots=2 * M + 12288), False), (dict(pos=9 * M, kb=9 * M, vb=10 * M), True),
    (dict(rope=2 * M - 100 * 128 * 4 - 8), False), (dict(rope=2 * M - 100 * 128 * 4 + 8), True), (dict(slots=M + 18428), True),
    (dict(qo=M + 18432), False), (dict(qo=M + 18428), True), (dict(kb=M - 3 * 1024, vb=10 * M), False), (dict(kb=M - 3 * 1024 + 4, vb=10 * M), True),
])
def test_overlaps(kw, want):
    assert refused(**kw) == want


def test_rows_of_any_strides_against_every_byte():
    """Random row sets of q_out, k and q, compared byte by byte."""
    rng = np.random.default_rng(80)

    def bytes_of(at, row, step, n):
        return {at + i * step * 4 + j for i in range(n) for j in range(0, row, 4)}
    hits = 0
    for _ in range(400):
        n = int(rng.integers(1, 9))
        qos, ks = int(rng.integers(64, 400)), int(rng.integers(64, 400))
        if rng.random() < 0.4:
            ks = qos
        k = 4 * M + 4 * int(rng.integers(-1600, 1600))
        kw = dict(hkv=1, hq=1, D=64, rot=64, n=n, qos=qos, qo=4 * M, qs=64, ks=ks, vs=64, k=k)
        want = bool(bytes_of(4 * M, 256, qos, n) & bytes_of(k, 256, ks, n))
        hits += want
        assert refused(**kw) == want, kw
    assert 50 < hits < 350
