"""Trees of drafted tokens in plain numpy, written from the description in include/aljabr_blackwell.h."""
import numpy as np

from tests import kv4_ref as ref


def chains(parents):
    """For each node its path from the root, itself last; empty where it is absent."""
    got = []
    for t, up in enumerate(parents):
        got.append([t] if up == -1 else got[up] + [t] if 0 <= up < t and got[up] else [])
    return got


def grow(rng, nodes, roots=1, absent=0):
    """Random parents, not level by level."""
    p = [-1 if t < roots else int(rng.integers(0, t)) for t in range(nodes)]
    for t in rng.choice(np.arange(1, nodes), absent, replace=False) if absent else ():
        p[t] = -2
    return p


def visible(parents, n, window=0):
    """Positions that each node sees, of n with the tree's; none where no tree is there."""
    base, paths = n - len(parents), chains(parents)
    rows = []
    for path in paths:
        if base < 0 or not path:
            rows.append([])
            continue
        at = list(range(base)) + [base + i for i in range(len(path))]      # the position a row stands for
        where = list(range(base)) + [base + u for u in path]
        mine = base + len(path) - 1
        rows.append([w for a, w in zip(at, where) if not window or mine - a < window])
    return rows


def attention(q, k, v, parents, n, window=0, scale=None, soft_cap=0.0):
    """q [nodes][Hq][D]; as kv4_ref.attention, for a tree."""
    parts = [np.zeros((3,) + q.shape), np.zeros(q.shape[:2])]
    for t, rows in enumerate(visible(parents, n, window)):
        if rows:
            o, w, d = ref.attention(q[t:t + 1], k[rows], v[rows], len(rows), scale=scale, soft_cap=soft_cap)
            parts[0][0][t], parts[0][1][t], parts[1][t] = o[0], w[0], d[0]
    return parts[0][0], parts[0][1], parts[1]


def walk(parents, drafted, picked):
    path = [0] if parents[0] == -1 else []
    while path:
        kids = [t for t, p in enumerate(parents) if p == path[-1] and drafted[t] == picked[path[-1]]]
        if not kids:
            break
        path.append(kids[0])
    return path


def rotate(x, table, positions, interleaved):
    """x [tokens][heads][D] fp32, table [positions][n][2] fp32; every product and sum rounded to fp32."""
    n, y = table.shape[1], np.array(x, np.float32)
    cs = table[np.maximum(positions, 0)][:, None]
    c, s = cs[..., 0], cs[..., 1]
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    lo, hi = a * c - b * s, a * s + b * c
    if interleaved:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = lo, hi
    else:
        y[..., :n], y[..., n:2 * n] = lo, hi
    y[positions < 0] = 0
    return y
