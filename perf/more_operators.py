"""The operators of tree-drafted decoding over the 4-bit KV cache, as measured work.

Three operators of a speculative serving step: rotating a batch's queries and
keys by their positions while keys and values enter the 4-bit cache, attention
of a tree of drafted tokens over that cache, and accepting a drafted path (the
walk along the model's own greedy tokens, and the move of the accepted rows to
their final positions in every layer's cache).  Every case exists in two forms
with the same inputs: the plain form (elementary torch operations in fp32) and,
where `own` is true, the framework's own entry points.

Cache layout, as documented in include/aljabr_blackwell.h: `pages` pages of
`page_size` positions; a page holds, per kv head, K codes [page_size][D/2],
V codes [page_size][D/2], K scales [page_size][D/32] fp16, V scales
[page_size][D/32] fp16.  A group of 32 values is d * (c - 8), c in 0..15.

A tree of `nodes` drafted tokens is given by parents: parents[t] < t, -1 for a
root, -2 for a node that is absent.  Its nodes take the last `nodes` positions
of their sequence in the cache, in node order; a node sees every position
before the tree, its ancestors and itself.
"""
import math
import random

import torch

own = False


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the smallest: one new token of one sequence, fp32 activations as the decode step has them
        dict(name="rotate-token", kind="rotate", tokens=1, kv_heads=8, group=4, head_dim=128, rotary=128,
             interleaved=False, page_size=64, dtype="f32", fused=False, back=False, skip=0.0),
        # the drafted trees of a batch, q | k | v columns of one buffer, half of each head rotated in adjacent pairs
        dict(name="rotate-trees", kind="rotate", tokens=259, kv_heads=2, group=7, head_dim=64, rotary=32,
             interleaved=True, page_size=16, dtype="bf16", fused=True, back=False, skip=0.1),
        # a long prompt of one layer, the rounded rows returned for the prompt's own attention
        dict(name="rotate-prompt", kind="rotate", tokens=16384, kv_heads=8, group=4, head_dim=128, rotary=128,
             interleaved=False, page_size=64, dtype="bf16", fused=True, back=True, skip=0.0),
        # a chain of five drafted tokens on a short context
        dict(name="tree-short", kind="tree", batch=1, nodes=5, kv_heads=8, group=4, head_dim=128, page_size=64,
             max_len=257, ragged=False, window=0, soft_cap=0.0, dtype="f32"),
        # one sequence at the framework's decode context, a tree of 64
        dict(name="tree-4096", kind="tree", batch=1, nodes=64, kv_heads=8, group=4, head_dim=128, page_size=64,
             max_len=4096, ragged=False, window=0, soft_cap=0.0, dtype="bf16"),
        # odd sizes: sliding window and capped scores, small pages, fp32
        dict(name="tree-window", kind="tree", batch=5, nodes=21, kv_heads=4, group=3, head_dim=64, page_size=16,
             max_len=3001, ragged=True, window=1024, soft_cap=30.0, dtype="f32"),
        # a serving batch of sequences of very different lengths
        dict(name="tree-batch", kind="tree", batch=24, nodes=26, kv_heads=8, group=4, head_dim=128, page_size=64,
             max_len=16384, ragged=True, window=0, soft_cap=0.0, dtype="bf16"),
        # two long documents on 64 query heads, a wide tree
        dict(name="tree-long", kind="tree", batch=2, nodes=61, kv_heads=8, group=8, head_dim=128, page_size=128,
             max_len=65536, ragged=False, window=0, soft_cap=0.0, dtype="bf16"),
        # one sequence's step ends: 32 layers keep the accepted rows
        dict(name="accept-one", kind="accept", batch=1, nodes=26, layers=32, kv_heads=8, head_dim=128, page_size=64,
             max_len=300),
        # a serving batch's step ends, the trees as large as they come
        dict(name="accept-batch", kind="accept", batch=64, nodes=64, layers=32, kv_heads=8, head_dim=128, page_size=16,
             max_len=200),
        # one layer's whole step for a small batch: rows in, attention, accepted rows kept
        dict(name="step", kind="step", batch=4, nodes=16, kv_heads=8, group=4, head_dim=128, page_size=64, max_len=2047,
             ragged=True, window=0, soft_cap=0.0, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotate", "rotate", "tree", "tree", "tree", "accept", "step"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "rotate":
        kv_heads, head_dim, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128, 256]), rng.choice([1, 2, 4, 5, 8])
        most = 16384 * 6144 // (kv_heads * head_dim * (group + 2)) // (2 if dtype == "f32" else 1)
        return dict(kind=kind, tokens=_log(rng, 1, min(most, 65536)), kv_heads=kv_heads, group=group, head_dim=head_dim,
                    rotary=rng.choice([head_dim, head_dim, head_dim // 2, 16, 48]), interleaved=rng.random() < 0.4,
                    page_size=rng.choice([16, 32, 48, 64, 128]), dtype=dtype, fused=rng.random() < 0.5,
                    back=rng.random() < 0.5, skip=rng.choice([0.0, 0.0, 0.2]))
    if kind == "accept":
        kv_heads, head_dim, batch = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256]), _log(rng, 1, 64)
        nodes = _log(rng, 1, 128)
        return dict(kind=kind, batch=batch, nodes=nodes, layers=rng.randint(1, max(1, 32 * 8 * 128 // (kv_heads * head_dim) // 4)),
                    kv_heads=kv_heads, head_dim=head_dim, page_size=rng.choice([16, 48, 64]),
                    max_len=nodes + rng.randint(0, 100))
    head_dim = rng.choice([64, 128, 128, 256])
    kv_heads, group = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 7, 8])
    batch = _log(rng, 1, 32)
    nodes = _log(rng, 1, 100)
    # positions: no more than the longest listed case reads, and its products no more than that case's
    most = 2 * 65536 * 8 * 128 // (kv_heads * head_dim * batch)
    most = min(65536, most * 61 * 8 // (group * nodes) if group * nodes > 61 * 8 else most)
    if dtype == "f32":
        most //= 4
    return dict(kind=kind, batch=batch, nodes=nodes, kv_heads=kv_heads, group=group, head_dim=head_dim,
                page_size=rng.choice([16, 48, 64, 256]), max_len=_log(rng, nodes, max(nodes + 1, most)),
                ragged=batch > 1 and rng.random() < 0.7, window=rng.choice([0, 0, 0, 100, 1024]),
                soft_cap=rng.choice([0.0, 0.0, 50.0]), dtype=dtype)


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _lens(case):
    """Positions of each sequence, the tree's among them: fixed by the case, so that its work is."""
    n, most = case["batch"], case["max_len"]
    if not case.get("ragged", True):
        return [most] * n
    r = random.Random(1000003 * n + most)
    lens = [min(most, max(case["nodes"], int(most * r.random() ** 2))) for _ in range(n)]
    lens[0] = most
    if n > 3:
        lens[1], lens[2] = 0, case["nodes"]   # a slot of the batch that holds no sequence, and a tree without context
    return lens


def _trees(case):
    """parents [batch][nodes]: trees grown level by level, two or three children a node, the last nodes of some absent;
    fixed by the case."""
    n, nodes = case["batch"], case["nodes"]
    r = random.Random(7919 * n + nodes)
    got = []
    for b in range(n):
        live = nodes if b % 3 != 1 else max(1, nodes - r.randint(0, nodes // 4))
        p = sorted(r.randint(max(0, (t - 1) // 3), max(0, (t - 1) // 2)) for t in range(1, live))
        got.append([-1] + p + [-2] * (nodes - live))
    return got


def _ancestors(parents):
    """For each node the nodes that it sees, itself among them (none where it is absent)."""
    seen = []
    for t, p in enumerate(parents):
        seen.append([] if p == -2 else [t] if p == -1 else seen[p] + [t])
    return seen


def _page_count(case):
    return -(-case["max_len"] // case["page_size"])


# ------------------------------------------------------------------ work
def work(case):
    kind = case["kind"]
    row = case["kv_heads"] * case["head_dim"]           # values of K, or of V, of one position
    if kind == "accept":
        moved = 3 * case["batch"]                       # rows of an accepted path that are not in place yet
        ints = case["batch"] * (4 * 4 * case["nodes"] + 16)
        return {"bytes": 2 * moved * case["layers"] * row * 2 * 18 / 32 + ints, "flops": case["batch"] * case["nodes"]}
    e, G = 4 if case["dtype"] == "f32" else 2, case["group"]
    if kind == "rotate":
        n = case["tokens"]
        wide = n * row * e * (2 * G + 2 + (2 if case["back"] else 0))
        return {"bytes": wide + n * row * 2 * 18 / 32 + n * (8 + 4 * case["rotary"]),
                "flops": n * row * (3 * (G + 1) + 8)}
    D, T = case["head_dim"], case["nodes"]
    seen = pairs = 0
    for n, parents in zip(_lens(case), _trees(case)):
        if n < T:
            continue
        base, lows = n - T, []
        for nodes in _ancestors(parents):
            if nodes:
                lo = max(0, base + len(nodes) - case["window"]) if case["window"] else 0
                lows.append(lo)
                pairs += max(0, base - lo) + min(len(nodes), case["window"] or len(nodes))
        seen += n - min(lows)
    b = seen * row * 2 * 18 / 32 + 2 * case["batch"] * T * row * G * e + 4 * case["batch"] * T
    if kind == "step":
        b += case["batch"] * T * row * (2 * e * (G + 1) + 2 * 18 / 32)
    return {"bytes": b, "flops": 4 * pairs * row * G}


# ------------------------------------------------------------------ inputs
def _kv(tokens, kv_heads, D, g, dtype):
    """K rows with channels of unequal size, as the projections give them, and V rows."""
    amp = 0.3 + torch.rand(kv_heads, D, device="cuda", generator=g) ** 4 * 3.0
    k = torch.randn(tokens, kv_heads, D, device="cuda", generator=g) * amp
    v = torch.randn(tokens, kv_heads, D, device="cuda", generator=g) * 0.7
    return k.to(dtype), v.to(dtype)


def _fill(cache, page_size, kv_heads, D, g):
    """Quantises random K / V into every page of the cache, some pages at a time."""
    pages = cache.shape[0]
    step = max(1, (1 << 26) // (page_size * kv_heads * D))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        for which, x in enumerate(_kv(n * page_size, kv_heads, D, g, torch.float32)):
            codes, d = _quantise(x)
            _put(cache[p:p + n], which, codes.view(n, page_size, kv_heads, D),
                 d.view(n, page_size, kv_heads, D // 32), kv_heads, page_size, D)


def _rope(positions, rotary, theta=500000.0):
    """Table [positions][rotary / 2] of (cos, sin), from angles in 64 bits."""
    f = theta ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * f
    return torch.stack((a.cos(), a.sin()), -1).float()


def _draft(case, seed, parents):
    """Drafted and greedily picked tokens [batch][nodes]: the greedy tokens follow the draft down to some node, siblings
    drafted the same token now and then.  Accepted rows beyond the first lie past the accepted count, as in wide trees,
    so that a step can be repeated on its own result."""
    r = random.Random(seed)
    vocab = 128256
    drafted, picked = [], []
    for p in parents:
        d = [r.randrange(vocab) for _ in p]
        for t in range(2, len(p)):
            if p[t] >= 0 and p[t] == p[t - 1] and r.random() < 0.1:
                d[t] = d[t - 1]
        first = {}
        for t, up in enumerate(p):
            first.setdefault((up, d[t]), t)
        paths = []
        for a in _ancestors(p):
            if a and all(first[(p[t], d[t])] == t for t in a[1:]) and all(t == i or t >= len(a) for i, t in enumerate(a)):
                paths.append(a)
        want = max(1, min(max(map(len, paths)), 1 + int(r.expovariate(0.4))))
        path = r.choice([a for a in paths if len(a) <= want])
        g = [r.randrange(vocab) for _ in p]
        for up, t in zip(path, path[1:]):
            g[up] = d[t]
        at = path[-1]
        while any(p[t] == at and d[t] == g[at] for t in range(len(p))):
            g[at] = r.randrange(vocab)
        drafted.append(d)
        picked.append(g)
    return drafted, picked


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind = case["kind"]
    Hkv, D, ps = case["kv_heads"], case["head_dim"], case["page_size"]
    s = {"case": dict(case)}
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    if kind == "rotate":
        per, pages = 0, -(-case["tokens"] // ps) + 1
    else:
        per = _page_count(case)
        pages = case["batch"] * per
    layers = case.get("layers", 1)
    cache = torch.zeros(layers, pages, Hkv * ps * (D + D // 8), dtype=torch.uint8, device="cuda")
    order = torch.randperm(pages, device="cuda", generator=g).int()
    if kind == "rotate":
        n = case["tokens"]
        at = torch.arange(n, device="cuda")
        s["slots"] = (order[at // ps] * ps + at % ps).int()
        s["positions"] = (at + int(torch.randint(0, 1000, (1,), generator=g, device="cuda"))).int()
    else:
        _fill(cache.view(layers * pages, -1), ps, Hkv, D, g)
        B, T = case["batch"], case["nodes"]
        s["lens"], s["table"] = ints(_lens(case)), order.view(B, per)
        parents = _trees(case)
        s["parents"] = ints(parents)
        seen = torch.zeros(B, T, T, dtype=torch.bool)
        for b, p in enumerate(parents):
            for t, a in enumerate(_ancestors(p)):
                seen[b, t, a] = True
        s["seen"] = seen.cuda()
        if kind == "tree":
            n = B * T
        if kind in ("accept", "step"):
            s["drafted"], s["picked"] = map(ints, _draft(case, seed, parents))
        if kind == "step":                              # the tree's rows enter at its slots, rotated by their depth
            n = B * T
            base = s["lens"].long()[:, None] - T
            pos = (base + torch.arange(T, device="cuda")).clamp(min=0)
            live = (s["parents"] > -2) & (base >= 0)
            slots = s["table"].long().gather(1, pos // ps) * ps + pos % ps
            s["slots"] = torch.where(live, slots, -1).int().flatten()
            s["positions"] = torch.where(live, base + s["seen"].sum(-1) - 1, -1).int().flatten()
    if kind != "accept":
        Hq, dt = Hkv * case["group"], _dtype(case)
        q = (torch.randn(n, Hq, D, device="cuda", generator=g) * 1.2).to(dt)
        if kind == "tree":
            s["q"] = q.view(B, T, Hq, D)
            s["out"] = torch.empty_like(s["q"])
        else:
            k, v = _kv(n, Hkv, D, g, dt)
            if case.get("fused"):                       # the columns of a [tokens][q | k | v] buffer
                wide = torch.cat((q.flatten(1), k.flatten(1), v.flatten(1)), 1)
                q, k, v = (x.unflatten(1, (-1, D)) for x in wide.split([Hq * D, Hkv * D, Hkv * D], 1))
            s["q"], s["k"], s["v"] = q, k, v
            s["q_out"] = torch.empty(n, Hq, D, device="cuda", dtype=dt)
            s["k_back"] = s["v_back"] = None
            if case.get("back"):
                s["k_back"], s["v_back"] = (torch.empty(n, Hkv, D, device="cuda", dtype=dt) for _ in range(2))
            if case.get("skip"):                        # padding between the sequences of a batch
                s["slots"][torch.rand(n, device="cuda", generator=g) < case["skip"]] = -1
            far = case["max_len"] if kind == "step" else case["tokens"] + 1000
            s["rope"] = _rope(far, case.get("rotary", D))
            if kind == "step":
                s["out"] = torch.empty(B, T, Hq, D, device="cuda", dtype=dt)
    s["cache"] = cache
    if own:
        from aljabr_b200.kv4 import Kv4Cache
        s["kv4"] = [Kv4Cache(pages, ps, Hkv, D, data=cache[i]) for i in range(layers)]
    return s


# ------------------------------------------------------------------ plain forms
def _quantise(x):
    """x [.., D] fp32 -> codes [.., D] uint8, scales [.., D/32] fp16."""
    g = x.unflatten(-1, (-1, 32))
    top, bottom = g.amax(-1), g.amin(-1)
    ext = torch.where(-bottom >= top, bottom, top)
    d = torch.where(ext.isfinite(), (ext / -8).clamp(-65504.0, 65504.0), torch.nan).half()
    df = d.float()
    inv = torch.where(df == 0, torch.zeros_like(df), 1.0 / df)
    c = (torch.round(g * inv[..., None]) + 8).clamp(0, 15)
    c = torch.where(df.isfinite()[..., None], c, torch.full_like(c, 8.0))
    return c.to(torch.uint8).flatten(-2), d


def _values(codes, d):
    return ((codes.unflatten(-1, (-1, 32)).float() - 8) * d.float()[..., None]).flatten(-2)


def _parts(cache, kv_heads, page_size, D):
    """Views of a cache [pages][..]: code rows and scale rows of K and of V."""
    c = cache.view(cache.shape[0], kv_heads, page_size * (D + D // 8))
    n, k8 = page_size * D // 2, page_size * D // 16
    ends = ((0, n), (n, n), (2 * n, k8), (2 * n + k8, k8))
    return [c[:, :, at:at + size].unflatten(2, (page_size, -1)) for at, size in ends]


def _pack(codes, which):
    """codes [.., D] -> rows of D/2 bytes in the cache's order."""
    D = codes.shape[-1]
    if which == 0:   # K: word (c, g) holds dims 32 g + 8 c + 0..7
        x = codes.unflatten(-1, (D // 32, 4, 8)).transpose(-3, -2)
    else:            # V: halfword (r, g) holds dims 32 g + 4 r + 0..3
        x = codes.unflatten(-1, (D // 32, 8, 4)).transpose(-3, -2)
    x = x.flatten(-3).unflatten(-1, (-1, 2))
    return x[..., 0] | (x[..., 1] << 4)


def _unpack(rows, which):
    D = rows.shape[-1] * 2
    x = torch.stack((rows & 15, rows >> 4), -1).flatten(-2)
    x = x.unflatten(-1, (4, D // 32, 8) if which == 0 else (8, D // 32, 4)).transpose(-3, -2)
    return x.flatten(-3)


def _put(cache, which, codes, d, kv_heads, page_size, D):
    """Writes whole pages: codes [pages][page_size][kv_heads][D]."""
    parts = _parts(cache, kv_heads, page_size, D)
    parts[which].copy_(_pack(codes, which).transpose(1, 2))
    parts[2 + which].copy_(d.contiguous().view(torch.uint8).transpose(1, 2))


def _gather(cache, which, page, row, kv_heads, page_size, D):
    """Values [..][kv_heads][D] of the rows (page, row), in fp32."""
    parts = _parts(cache, kv_heads, page_size, D)
    codes = _unpack(parts[which][page, :, row], which)
    d = parts[2 + which][page, :, row].contiguous().view(torch.float16)
    return _values(codes, d)


def _rotate(x, cs, interleaved):
    """x [tokens][heads][D] fp32, the first 2 n dims of a head rotated by cs [tokens][n] of (cos, sin): dims i and
    i + n are a pair, or 2 i and 2 i + 1."""
    n = cs.shape[1]
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    if interleaved:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        y = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        y = torch.cat((a * c - b * s, a * s + b * c), -1)
    return torch.cat((y, x[..., 2 * n:]), -1)


def _plain_rotate(s):
    """Rotated q, and K and V rows as the cache now holds them."""
    c = s["case"]
    ps, Hkv, D = c["page_size"], c["kv_heads"], c["head_dim"]
    there = s["positions"] >= 0
    cs = s["rope"][s["positions"].clamp(min=0).long()]
    turn = lambda x: _rotate(x.float(), cs, c.get("interleaved", False))  # noqa: E731
    keep = (s["slots"] >= 0) & there
    at = s["slots"][keep].long()
    parts = _parts(s["cache"][0], Hkv, ps, D)

    def store(which, x, dtype):
        codes, d = _quantise(x)
        parts[which][at // ps, :, at % ps] = _pack(codes[keep], which)
        parts[2 + which][at // ps, :, at % ps] = d[keep].contiguous().view(torch.uint8)
        return torch.where(keep[:, None, None], _values(codes, d), 0.0).to(dtype)
    q = torch.where(there[:, None, None], turn(s["q"]), 0.0).to(s["q"].dtype)
    return q, store(0, turn(s["k"]), s["k"].dtype), store(1, s["v"].float(), s["v"].dtype)


def _plain_tree(s, q):
    c = s["case"]
    ps, Hkv, D, T, G, B = c["page_size"], c["kv_heads"], c["head_dim"], c["nodes"], c["group"], c["batch"]
    pos = torch.arange(c["max_len"], device="cuda")
    page = s["table"].long()[:, pos // ps]
    row = (pos % ps).expand(B, -1)
    k, v = (_gather(s["cache"][0], i, page, row, Hkv, ps, D) for i in (0, 1))        # [B][S][Hkv][D]
    q = q.float().view(B, T, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, T * G, D)
    sc = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(D))                # [B][Hkv][T G][S]
    if c["soft_cap"]:
        sc = torch.tanh(sc / c["soft_cap"]) * c["soft_cap"]
    base = s["lens"].long()[:, None] - T
    depth = s["seen"].sum(-1)                                                         # itself among them; 0: absent
    node = (pos - base).clamp(0, T - 1)                                               # [B][S]
    see = s["seen"].gather(2, node[:, None].expand(B, T, -1))
    in_tree = ((pos >= base) & (pos < base + T))[:, None]
    at = torch.where(in_tree, base[..., None] + depth.gather(1, node)[:, None] - 1, pos)  # position that a row stands for
    see = torch.where(in_tree, see, (pos < base)[:, None] & (depth > 0)[..., None]) & (base >= 0)[..., None]
    if c["window"]:
        see &= at > (base + depth - 1)[..., None] - c["window"]
    see = see.repeat_interleave(G, 1)[:, None]                                        # [B][1][T G][S]
    sc = torch.where(see, sc, -torch.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == -torch.inf, torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(l == 0, torch.ones_like(l), l)
    return o.view(B, Hkv, T, G, D).permute(0, 2, 1, 3, 4).reshape(B, T, Hkv * G, D).to(s["q"].dtype)


def _plain_accept(s):
    """Path, its length, the token after it and the new lengths; the accepted rows of every layer move in place."""
    c = s["case"]
    ps, Hkv, D, T, B = c["page_size"], c["kv_heads"], c["head_dim"], c["nodes"], c["batch"]
    parents, base = s["parents"].long(), s["lens"].long() - T
    node = torch.arange(T, device="cuda")
    up = parents.clamp(min=0)
    good = (parents >= 0) & (s["drafted"] == s["picked"].gather(1, up))
    twin = (parents[:, :, None] == parents[:, None]) & good[:, None]                  # good siblings of each node
    good &= ~(twin & (node < node[:, None])).any(-1)                                  # the first of them
    good |= (node == 0) & (parents == -1)
    on = (good[:, None] | ~s["seen"]).all(-1) & (parents > -2) & (base >= 0)[:, None]
    on &= s["seen"][:, :, 0]
    count = on.sum(1)
    path = torch.where(on, node, T).sort(1).values
    last = path.gather(1, (count - 1).clamp(min=0)[:, None])
    token = torch.where(count > 0, s["picked"].gather(1, last.clamp(max=T - 1))[:, 0], -1).int()
    lens = torch.where(base >= 0, base + count, s["lens"]).int()
    # row i of the tree's rows comes from path[i], or stays
    source = torch.where(node < count[:, None], path, node)
    first = base.clamp(min=0)[:, None]
    n_pages = s["cache"].shape[1]
    layer = torch.arange(s["cache"].shape[0], device="cuda")[:, None, None] * n_pages
    place = lambda p: (layer + s["table"].long().gather(1, p // ps), (p % ps).expand(len(layer), -1, -1))  # noqa: E731
    fits = _page_count(c) * ps - 1
    src, dst = place((first + source).clamp(max=fits)), place((first + node).clamp(max=fits))
    parts = _parts(s["cache"].flatten(0, 1), Hkv, ps, D)
    moved = (base >= 0)[None, :, None].expand(len(layer), -1, T)
    new = [x[src[0], :, src[1]][moved] for x in parts]
    parts[0][dst[0][moved], :, dst[1][moved]] = new[0]
    parts[1][dst[0][moved], :, dst[1][moved]] = new[1]
    parts[2][dst[0][moved], :, dst[1][moved]] = new[2]
    parts[3][dst[0][moved], :, dst[1][moved]] = new[3]
    return [torch.where(path < T, path, -1).int(), count.int(), token, lens]


def run(s):
    c = s["case"]
    kind = c["kind"]
    got = []
    if own:
        from aljabr_b200.kv4 import accept_tree
        cache = s["kv4"][0]
        if kind in ("rotate", "step"):
            q = cache.append_rotated(s["q"], s["k"], s["v"], s["slots"], s["positions"], s["rope"],
                                     interleaved=c.get("interleaved", False), q_out=s["q_out"], k_back=s["k_back"],
                                     v_back=s["v_back"])
            got += [q] if s["k_back"] is None else [q, s["k_back"], s["v_back"]]
        if kind in ("tree", "step"):
            q = s["q"] if kind == "tree" else q.view(s["out"].shape)
            got.append(cache.attend_tree(q, s["lens"], s["parents"], s["table"], window=c["window"],
                                         soft_cap=c["soft_cap"], out=s["out"]))
        if kind in ("accept", "step"):
            got += accept_tree(s["kv4"], s["lens"], s["parents"], s["drafted"], s["picked"], s["table"])
    else:
        if kind in ("rotate", "step"):
            q, k, v = _plain_rotate(s)
            got += [q] if s["k_back"] is None else [q, k, v]
        if kind in ("tree", "step"):
            got.append(_plain_tree(s, s["q"] if kind == "tree" else q))
        if kind in ("accept", "step"):
            got += _plain_accept(s)
    return got if kind == "tree" else got + [s["cache"]]


# ------------------------------------------------------------------ 64 bits
def _rows64(cache, which, page, row, kv_heads, page_size, D):
    """Values [n][kv_heads][D] of the rows (page, row), from each dimension's byte and shift."""
    per_head = page_size * (D + D // 8)
    dims = torch.arange(D, device="cuda")
    g, j = dims // 32, dims % 32
    if which == 0:
        byte, shift = 4 * ((j // 8) * (D // 32) + g) + (j % 8) // 2, 4 * (j % 2)
    else:
        byte, shift = 2 * ((j // 4) * (D // 32) + g) + (j % 4) // 2, 4 * (j % 2)
    flat = cache.reshape(-1)
    base = (page[:, None] * kv_heads + torch.arange(kv_heads, device="cuda")) * per_head
    code_at = base + which * page_size * D // 2 + row[:, None] * (D // 2)
    code = (flat[code_at[..., None] + byte].int() >> shift.int()) & 15
    scale_at = (base + page_size * D + which * page_size * D // 16) // 2 + row[:, None] * (D // 32)
    d = flat.view(torch.float16)[scale_at[..., None] + g].double()
    return (code.double() - 8.0) * d


def _round64(x):
    """A row's values after quantising, in 64 bits: x [.., D]."""
    g = x.unflatten(-1, (-1, 32))
    where = g.abs().argmax(-1, keepdim=True)
    ext = g.gather(-1, where)
    both = ((g == -ext).any(-1, keepdim=True)) & (ext > 0)   # +m and -m: the negative one sets the scale
    d = (torch.where(both, -ext, ext) / -8.0).clamp(-65504, 65504).half().double()
    c = torch.where(d == 0, torch.zeros_like(g), torch.round(g / torch.where(d == 0, torch.ones_like(d), d)))
    return (c.clamp(-8, 7) * d).flatten(-2)


def _turn64(x, s, interleaved):
    """Rotation as complex numbers."""
    pos = s["positions"].clamp(min=0).long()
    z = torch.view_as_complex(s["rope"].double())[pos][:, None]
    n, y = z.shape[-1], x.double().clone()
    if interleaved:
        w = torch.complex(y[..., 0:2 * n:2], y[..., 1:2 * n:2]) * z
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = w.real, w.imag
    else:
        w = torch.complex(y[..., :n], y[..., n:2 * n]) * z
        y[..., :n], y[..., n:2 * n] = w.real, w.imag
    return y * (s["positions"] >= 0)[:, None, None]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    ps, Hkv, D = case["page_size"], case["kv_heads"], case["head_dim"]
    got, new = [], None
    if kind in ("rotate", "step"):
        inter = case.get("interleaved", False)
        keep = ((s["slots"] >= 0) & (s["positions"] >= 0))[:, None, None]
        new = [torch.where(keep, _round64(x), 0.0) for x in (_turn64(s["k"], s, inter), s["v"].double())]
        q64 = _turn64(s["q"], s, inter)
        got = [q64] + (new if case.get("back") else [])
        if kind == "rotate":
            return got + [None]
        q64 = q64.to(_dtype(case)).double()              # what the attention is given
    if kind in ("tree", "step"):
        B, T, G = case["batch"], case["nodes"], case["group"]
        q = s["q"].double() if kind == "tree" else q64
        q = q.view(B, T, Hkv, G, D)
        out = torch.zeros(B, T, Hkv * G, D, device="cuda", dtype=torch.float64)
        for b, (n, parents) in enumerate(zip(_lens(case), _trees(case))):
            if n < T:
                continue
            base = n - T
            pos = torch.arange(n, device="cuda")
            page = s["table"][b].long()[pos // ps]
            k, v = (_rows64(s["cache"][0], i, page, pos % ps, Hkv, ps, D) for i in (0, 1))
            if kind == "step":
                k[base:], v[base:] = (x.view(B, T, Hkv, D)[b] for x in new)
            chains = _ancestors(parents)
            at = pos.clone()
            at[base:] = torch.tensor([base + len(a) - 1 for a in chains], device="cuda")
            for t, chain in enumerate(chains):
                if not chain:
                    continue
                lo = max(0, base + len(chain) - case["window"]) if case["window"] else 0
                lo = min(lo, base)
                rows = torch.cat((pos[lo:base], torch.tensor([base + u for u in chain], device="cuda")))
                if case["window"]:
                    rows = rows[at[rows] > base + len(chain) - 1 - case["window"]]
                sc = torch.einsum("hgd,shd->hgs", q[b, t], k[rows]) / math.sqrt(D)
                if case["soft_cap"]:
                    sc = torch.tanh(sc / case["soft_cap"]) * case["soft_cap"]
                out[b, t] = torch.einsum("hgs,shd->hgd", sc.softmax(-1), v[rows]).reshape(Hkv * G, D)
        got.append(out)
    if kind in ("accept", "step"):
        T = case["nodes"]
        drafted, picked = s["drafted"].tolist(), s["picked"].tolist()
        paths, tokens, lens = [], [], []
        for b, (n, p) in enumerate(zip(_lens(case), _trees(case))):
            path = [0] if n >= T and p[0] == -1 else []
            while path and (kids := [t for t in range(T) if p[t] == path[-1] and drafted[b][t] == picked[b][path[-1]]]):
                path.append(kids[0])
            paths.append(path + [-1] * (T - len(path)))
            tokens.append(picked[b][path[-1]] if path else -1)
            lens.append(n - T + len(path) if n >= T else n)
        counts = [sum(x >= 0 for x in p) for p in paths]
        got += [torch.tensor(x, dtype=torch.int32) for x in (paths, counts, tokens, lens)] + [None]
    return got
