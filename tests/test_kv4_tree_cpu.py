"""Refusals of the tree operators over the 4-bit cache, checked before the GPU
is touched, and the plain forms that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest

from aljabr_b200 import native
from tests import tree_ref as tree

P = 1 << 20      # a well-aligned address that is never followed
DIMS, UNSUP, ARG, OK = native.ALJ_ERR_BAD_DIMS, native.ALJ_ERR_UNSUPPORTED, native.ALJ_ERR_BAD_ARG, native.ALJ_OK


def rc(name, *args):
    return getattr(native.lib(), name)(*args)


def rotate(cache=P, pages=4, ps=16, hkv=2, D=128, qo=P, qos=1024, q=P, k=P, v=P, dt=native.KV_F32, qs=1024, ks=256, vs=256, hq=8,
           slots=P, pos=P, rope=P, far=100, rot=128, inter=0, n=3, kb=None, vb=None):
    return rc("aljabr_blackwell_kv4_rotate_append_dev", cache, pages, ps, hkv, D, qo, qos, q, k, v, dt, qs, ks, vs, hq, slots, pos,
              rope, far, rot, inter, n, kb, vb, None)


def attend(out=P, q=P, dt=native.KV_F32, qs=1024, cache=P, pages=4, ps=16, hkv=2, D=128, table=P, width=4, lens=P, batch=2,
           parents=P, pstride=5, nodes=5, hq=8, window=0, scale=0.1, cap=0.0, work=P, size=1 << 40):
    return rc("aljabr_blackwell_kv4_tree_attention_dev", out, q, dt, qs, cache, pages, ps, hkv, D, table, width, lens, batch,
              parents, pstride, nodes, hq, window, scale, cap, work, size, None)


def accept(path=P, count=2 * P, token=3 * P, new=4 * P, caches=(5 * P, 6 * P), layers=None, pages=4, ps=16, hkv=2, D=128, table=7 * P,
           width=4, lens=8 * P, batch=2, parents=9 * P, pstride=5, nodes=5, drafted=10 * P, picked=11 * P):
    arr = None if caches is None else (ctypes.c_void_p * len(caches))(*caches)
    return rc("aljabr_blackwell_kv4_accept_tree_dev", path, count, token, new, arr, len(caches) if layers is None else layers, pages,
              ps, hkv, D, table, width, lens, batch, parents, pstride, nodes, drafted, picked, None)


@pytest.mark.parametrize("kw,code", [
    (dict(pages=0), DIMS), (dict(D=96), UNSUP), (dict(ps=24), UNSUP), (dict(dt=2), UNSUP), (dict(n=-1), DIMS),
    (dict(cache=None), ARG), (dict(cache=P + 8), ARG), (dict(slots=None), ARG), (dict(slots=P + 2), ARG), (dict(k=None), ARG),
    (dict(v=P + 1), ARG), (dict(kb=P), ARG), (dict(ks=255), DIMS), (dict(hq=0), DIMS), (dict(hq=2 ** 30), DIMS),
    (dict(far=0), DIMS), (dict(rot=0), DIMS), (dict(rot=24), DIMS), (dict(rot=144), DIMS), (dict(rot=-16), DIMS),
    (dict(q=None), ARG), (dict(qo=None), ARG), (dict(pos=None), ARG), (dict(rope=None), ARG), (dict(qs=1023), DIMS),
    (dict(qos=1000), DIMS), (dict(q=P + 2), ARG), (dict(qo=P + 1, dt=native.KV_BF16), ARG), (dict(pos=P + 1), ARG),
    (dict(rope=P + 8), ARG)])
def test_rotated_append_refuses(kw, code):
    assert rotate(**kw) == code and native.last_error()


def test_rotated_append_of_no_tokens_is_nothing():
    assert rotate(n=0, q=None, k=None, slots=None, pos=None, rope=None) == OK


@pytest.mark.parametrize("kw,code", [
    (dict(D=80), UNSUP), (dict(ps=8), UNSUP), (dict(nodes=0), DIMS), (dict(nodes=257, pstride=257), DIMS), (dict(hq=7), DIMS),
    (dict(nodes=256, pstride=256, hq=10), UNSUP), (dict(dt=5), UNSUP), (dict(batch=-1), DIMS), (dict(batch=2049), DIMS),
    (dict(window=-1), ARG), (dict(cap=-1.0), ARG), (dict(cap=1e-35), ARG), (dict(out=None), ARG), (dict(q=None), ARG),
    (dict(lens=None), ARG), (dict(lens=P + 2), ARG), (dict(work=None), ARG), (dict(width=0), DIMS), (dict(table=None, batch=5), DIMS),
    (dict(qs=1023), DIMS), (dict(out=P + 8), ARG), (dict(q=P + 2), ARG), (dict(parents=None), ARG), (dict(parents=P + 2), ARG),
    (dict(pstride=4), DIMS), (dict(pstride=-5), DIMS)])
def test_tree_attention_refuses(kw, code):
    assert attend(**kw) == code and native.last_error()


def test_tree_attention_of_an_empty_batch_is_nothing():
    assert attend(batch=0, out=None, lens=None, parents=None) == OK


@pytest.mark.parametrize("kw,code", [
    (dict(D=80), UNSUP), (dict(pages=0), DIMS), (dict(nodes=0), DIMS), (dict(nodes=257, pstride=257), DIMS), (dict(layers=0), DIMS),
    (dict(layers=257), DIMS), (dict(batch=2049), DIMS), (dict(path=None), ARG), (dict(count=None), ARG), (dict(token=None), ARG),
    (dict(new=None), ARG), (dict(caches=None, layers=2), ARG), (dict(caches=(5 * P, None)), ARG), (dict(caches=(5 * P, 6 * P + 8)), ARG),
    (dict(caches=(5 * P, 6 * P, 5 * P)), ARG), (dict(lens=None), ARG), (dict(drafted=None), ARG), (dict(picked=None), ARG),
    (dict(parents=None), ARG), (dict(pstride=3), DIMS), (dict(width=0), DIMS), (dict(table=None, batch=5), DIMS),
    (dict(path=P + 2), ARG), (dict(new=4 * P + 1), ARG), (dict(drafted=10 * P + 3), ARG),
    (dict(new=8 * P), ARG), (dict(new=8 * P + 4), ARG), (dict(path=9 * P + 36), ARG), (dict(token=11 * P), ARG),
    (dict(count=7 * P + 28), ARG)])
def test_acceptance_refuses(kw, code):
    assert accept(**kw) == code and native.last_error()


def test_acceptance_of_an_empty_batch_is_nothing():
    assert accept(batch=0, path=None, lens=None, parents=None) == OK


def test_workspace_sizes():
    size = native.lib().aljabr_blackwell_kv4_tree_attention_workspace_size
    assert size(1, 32, 8, 128) > 0 and size(0, 32, 8, 128) == DIMS and size(257, 8, 8, 128) == DIMS and size(3, 9, 8, 128) == DIMS
    assert size(129, 64, 8, 128) == UNSUP and size(5, 8, 8, 96) == UNSUP
    # what the wrapper keeps serves every call
    most = max(size(native.KV4_MAX_NODES, native.KV4_MAX_ROWS // native.KV4_MAX_NODES, 1, D) for D in (64, 128, 256))
    assert all(size(n, g, 1, D) <= most for n in (1, 7, 64, 128, 256) for g in (1, 3, 4) for D in (64, 128, 256))
    assert all(size(n, 1024 // n, 1, D) <= most for n in (1, 2, 64, 128, 256) for D in (64, 128, 256))


def test_plain_trees():
    #      0
    #    1   2      6 (a second root)
    #   3   4       7
    parents = [-1, 0, 0, 1, 2, -2, -1, 6, 5]
    assert tree.chains(parents) == [[0], [0, 1], [0, 2], [0, 1, 3], [0, 2, 4], [], [6], [6, 7], []]
    rows = tree.visible(parents, 12)
    assert rows[0] == [0, 1, 2, 3] and rows[3] == [0, 1, 2, 3, 4, 6] and rows[5] == [] and rows[7] == [0, 1, 2, 9, 10]
    assert tree.visible(parents, 12, window=2)[3] == [4, 6] and tree.visible(parents, 12, window=5)[0] == [0, 1, 2, 3]
    assert tree.visible(parents, 12, window=3)[0] == [1, 2, 3] and tree.visible(parents, 8) == [[]] * 9
    assert tree.walk(parents, [9, 5, 5, 7, 7, 1, 5, 7, 0], [5, 7, 8, 7, 0, 0, 0, 0, 0]) == [0, 1, 3]
    assert tree.walk([-2, -1], [1, 1], [1, 1]) == []


def test_plain_rotation_keeps_lengths():
    rng = np.random.default_rng(3)
    x, a = rng.normal(size=(4, 2, 64)).astype(np.float32), rng.normal(size=(10, 24))
    table = np.stack((np.cos(a), np.sin(a)), -1).astype(np.float32)
    for inter in (False, True):
        y = tree.rotate(x, table, np.array([0, 9, 3, -1]), inter)
        assert np.allclose((y[:3] ** 2).sum(-1), (x[:3] ** 2).sum(-1), rtol=1e-5) and (y[3] == 0).all()
        assert np.array_equal(y[:3, :, 48:], x[:3, :, 48:]) and not np.allclose(y[:3, :, :48], x[:3, :, :48])
