"""Acceptance refuses outputs and caches that overlap; every call here is refused before the GPU is touched."""
import pytest

from aljabr_b200 import native
from tests.test_kv4_tree_cpu import P, accept

CACHE = 4 * 16 * 2 * (128 + 16)      # bytes of one: 4 pages of 16 positions, 2 heads of 128


# path of 2 x 5 (40 bytes) at P, count (8) at 2 P, token at 3 P, lens at 4 P; caches at 5 P and 6 P
@pytest.mark.parametrize("kw,what", [
    (dict(count=P), "one another"), (dict(count=P + 36), "one another"), (dict(token=2 * P), "one another"), (dict(new=3 * P + 4), "one another"),
    (dict(new=2 * P - 4), "one another"), (dict(path=4 * P - 36), "one another"),
    (dict(caches=(5 * P, 5 * P + 16)), "overlap"), (dict(caches=(5 * P, 5 * P + CACHE - 16)), "overlap"),
    (dict(caches=(5 * P + CACHE - 16, 6 * P, 5 * P)), "overlap"), (dict(caches=(5 * P, 5 * P)), "overlap"),
    (dict(caches=(5 * P, P - CACHE + 16)), "an output"), (dict(caches=(5 * P, 4 * P)), "an output"), (dict(token=5 * P + CACHE - 4), "an output"),
    # neighbours are taken: what is refused is the cache that is not aligned, behind them
    (dict(count=P + 40, caches=(5 * P, 5 * P + CACHE, 8)), "aligned"), (dict(token=2 * P + 8, caches=(5 * P + CACHE, 5 * P, 8)), "aligned"),
    (dict(caches=(P - CACHE, 5 * P, 8)), "aligned"), (dict(token=5 * P + CACHE, caches=(5 * P, 6 * P, 8)), "aligned"),
    (dict(table=None, width=0, batch=1, caches=(5 * P, 8)), "aligned")])
def test_overlaps(kw, what):
    assert accept(**kw) == native.ALJ_ERR_BAD_ARG and what in native.last_error(), native.last_error()
