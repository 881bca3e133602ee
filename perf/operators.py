"""The operators of the 4-bit KV cache and of the logits step, as measured work.

Four operators of the decode loop: quantising K and V rows as they enter the
4-bit cache, reading rows back, attention over that cache, and the logits
step (penalties, biases, grammar mask, greedy token).  Every case exists in
two forms with the same inputs: the plain form (elementary torch operations
in fp32) and, where `own` is true, the framework's own entry points.

Cache layout, as documented in include/aljabr_blackwell.h: `pages` pages of
`page_size` positions; a page holds, per kv head, K codes [page_size][D/2],
V codes [page_size][D/2], K scales [page_size][D/32] fp16, V scales
[page_size][D/32] fp16.  A group of 32 values is d * (c - 8), c in 0..15.
"""
import math
import random

import torch

own = False


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a prompt chunk of a small model, bf16 K / V in the rows of a fused q|k|v buffer, some rows padding
        dict(name="append-chunk", kind="append", tokens=513, kv_heads=2, head_dim=64, page_size=16, dtype="bf16",
             fused=True, skip=0.1),
        # a long prompt entering the cache of one layer, fp32 K / V as the projections leave them
        dict(name="append-prompt", kind="append", tokens=16384, kv_heads=8, head_dim=128, page_size=64, dtype="f32",
             fused=False, skip=0.0),
        # a short prefix read back for the attention of the next chunk
        dict(name="read-prefix", kind="read", tokens=1001, kv_heads=8, head_dim=128, page_size=16, dtype="bf16"),
        # a long session read back in fp32
        dict(name="read-session", kind="read", tokens=49152, kv_heads=8, head_dim=128, page_size=64, dtype="f32"),
        # the smallest serving step: one new token is quantised into the cache and attends to a short context
        dict(name="step-short", kind="step", batch=1, q_len=1, kv_heads=8, group=4, head_dim=128, page_size=64,
             max_len=257, ragged=False, window=0, soft_cap=0.0, dtype="f32"),
        # the framework's decode shape: 32 query heads on 8 kv heads, context 4096, fp32 activations
        dict(name="attend-4096", kind="attend", batch=1, q_len=1, kv_heads=8, group=4, head_dim=128, page_size=4096,
             max_len=4096, ragged=False, window=0, soft_cap=0.0, dtype="f32"),
        # a serving batch of sequences of very different lengths
        dict(name="attend-batch", kind="attend", batch=32, q_len=1, kv_heads=8, group=4, head_dim=128, page_size=64,
             max_len=16384, ragged=True, window=0, soft_cap=0.0, dtype="bf16"),
        # verifying five drafted tokens a sequence, sliding window and capped scores, odd lengths
        dict(name="attend-verify", kind="attend", batch=7, q_len=5, kv_heads=4, group=2, head_dim=64, page_size=16,
             max_len=3001, ragged=True, window=1024, soft_cap=30.0, dtype="f32"),
        # two long documents on 64 query heads
        dict(name="attend-long", kind="attend", batch=2, q_len=1, kv_heads=8, group=8, head_dim=128, page_size=128,
             max_len=131072, ragged=False, window=0, soft_cap=0.0, dtype="bf16"),
        # one sequence's logits with a grammar mask
        dict(name="logits-one", kind="logits", rows=1, vocab=128256, history=300, biases=16, grammar=True, dtype="f32"),
        # odd vocabulary, bf16 logits, no grammar
        dict(name="logits-odd", kind="logits", rows=5, vocab=32003, history=77, biases=3, grammar=False, dtype="bf16"),
        # a serving batch with long histories
        dict(name="logits-batch", kind="logits", rows=96, vocab=128256, history=4000, biases=64, grammar=True,
             dtype="f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "read", "step", "attend", "attend", "attend", "logits", "logits"])
    dtype = rng.choice(["f32", "bf16"])
    if kind in ("append", "read"):
        kv_heads, head_dim = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([64, 128, 256])
        most = {"append": 16384, "read": 49152}[kind] * 1024 // (kv_heads * head_dim)
        c = dict(kind=kind, tokens=_log(rng, 1, min(most, 65536)), kv_heads=kv_heads, head_dim=head_dim,
                 page_size=rng.choice([16, 32, 48, 64, 128]), dtype=dtype)
        if kind == "append":
            c.update(fused=rng.random() < 0.5, skip=rng.choice([0.0, 0.0, 0.2]))
        return c
    if kind == "logits":
        rows = _log(rng, 1, 96)
        return dict(kind=kind, rows=rows, vocab=_log(rng, 1000, 12_000_000 // rows if rows > 46 else 260_000),
                    history=_log(rng, 1, 4000), biases=rng.randint(0, 64), grammar=rng.random() < 0.5, dtype=dtype)
    head_dim = rng.choice([64, 128, 128, 256])
    kv_heads, group = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 7, 8, 16])
    batch = _log(rng, 1, 48)
    q_len = 1 if kind == "step" else rng.choice([1, 1, 1, 2, 4, 7])
    # positions: no more than the longest listed case reads, and its products no more than that case's
    most = 2 * 131072 * 8 * 128 // (kv_heads * head_dim * batch)
    most = min(131072, most // max(1, group * q_len // 8))
    return dict(kind=kind, batch=batch, q_len=q_len, kv_heads=kv_heads, group=group, head_dim=head_dim,
                page_size=rng.choice([16, 48, 64, 256]), max_len=_log(rng, 1, max(2, most)),
                ragged=batch > 1 and rng.random() < 0.7, window=rng.choice([0, 0, 0, 100, 1024]),
                soft_cap=rng.choice([0.0, 0.0, 50.0]), dtype=dtype)


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _lens(case):
    """Positions of each sequence: fixed by the case, so that its work is."""
    n, most = case["batch"], case["max_len"]
    if not case["ragged"]:
        return [most] * n
    r = random.Random(1000003 * n + most)
    lens = [min(most, max(case["q_len"], int(most * r.random() ** 2))) for _ in range(n)]
    lens[0] = most
    if n > 3 and case["kind"] == "attend":
        lens[1], lens[2] = 0, min(most, 1)   # a slot of the batch that holds no sequence yet, and one that just began
    return lens


def _page_count(case):
    return -(-case["max_len"] // case["page_size"])


# ------------------------------------------------------------------ work
def work(case):
    kind, e = case["kind"], 4 if case["dtype"] == "f32" else 2
    if kind in ("append", "read"):
        values = 2 * case["tokens"] * case["kv_heads"] * case["head_dim"]
        cached = values * 18 / 32
        wide = values * e * (2 if kind == "append" else 1)   # the rows in, and (append) the rounded rows out
        return {"bytes": wide + cached + 4 * case["tokens"], "flops": 4 * values}
    if kind == "logits":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (e + 4) + (n / 8 if case["grammar"] else 0) +
                case["rows"] * (4 * case["history"] + 8 * case["biases"] + 24), "flops": 4 * n}
    D, G, T = case["head_dim"], case["group"], case["q_len"]
    rows = case["batch"] * T * case["kv_heads"] * G
    seen = pairs = 0
    for n in _lens(case):
        per = [(max(0, p - case["window"] + 1) if case["window"] else 0, p) for p in range(n - T, n) if p >= 0]
        if per:
            seen += per[-1][1] - per[0][0] + 1
            pairs += sum(hi - lo + 1 for lo, hi in per)
    b = seen * case["kv_heads"] * D * 2 * 18 / 32 + 2 * rows * D * e
    if kind == "step":
        b += case["batch"] * case["kv_heads"] * D * 2 * 2 * e
    return {"bytes": b, "flops": 4 * pairs * case["kv_heads"] * G * D}


# ------------------------------------------------------------------ inputs
def _kv(tokens, kv_heads, D, g, dtype):
    """K rows with channels of unequal size, as rotary keys have them, and V rows."""
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


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, dt = case["kind"], _dtype(case)
    s = {"case": dict(case)}
    if kind == "logits":
        rows, vocab, hist, nb = case["rows"], case["vocab"], case["history"], case["biases"]
        s["logits"] = (torch.randn(rows, vocab, device="cuda", generator=g) * 3.0).to(dt)
        # tokens come back: half of a history is drawn from a few hundred tokens
        few = torch.randint(0, vocab, (rows, min(hist, 200)), device="cuda", generator=g)
        h = torch.randint(0, vocab, (rows, hist), device="cuda", generator=g)
        again = torch.gather(few, 1, torch.randint(0, few.shape[1], (rows, hist), device="cuda", generator=g))
        s["history"] = torch.where(torch.rand(rows, hist, device="cuda", generator=g) < 0.5, h, again).int()
        s["history_len"] = (hist - torch.arange(rows, device="cuda") * hist // (2 * rows)).int()
        s["penalties"] = torch.tensor([1.1, 0.3, 0.4], device="cuda").repeat(rows, 1) * \
            (1 + 0.1 * torch.rand(rows, 1, device="cuda", generator=g))
        s["bias_tokens"] = s["bias_values"] = s["bias_len"] = s["allow"] = None
        if nb:
            first = torch.randint(0, vocab, (rows, 1), device="cuda", generator=g)
            s["bias_tokens"] = ((first + torch.arange(nb, device="cuda") * max(1, vocab // (nb + 1))) % vocab).int()
            s["bias_values"] = torch.randn(rows, nb, device="cuda", generator=g) * 5.0
            s["bias_len"] = torch.full((rows,), nb, device="cuda", dtype=torch.int32)
        if case["grammar"]:
            s["allow"] = torch.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32), device="cuda", generator=g).int()
        s["out"] = torch.empty(rows, vocab, device="cuda")
        s["token"] = torch.empty(rows, device="cuda", dtype=torch.int32)
        return s
    Hkv, D, ps = case["kv_heads"], case["head_dim"], case["page_size"]
    if kind in ("append", "read"):
        tokens = case["tokens"]
        pages = -(-tokens // ps) + 1
    else:
        per = _page_count(case)
        pages = case["batch"] * per
    cache = torch.zeros(pages, Hkv * ps * (D + D // 8), dtype=torch.uint8, device="cuda")
    order = torch.randperm(pages, device="cuda", generator=g).int()
    if kind in ("append", "read"):
        at = torch.arange(tokens, device="cuda")
        s["slots"] = (order[at // ps] * ps + at % ps).int()
        if kind == "append":
            k, v = _kv(tokens, Hkv, D, g, dt)
            if case["fused"]:   # the K and V columns of a [tokens][q | k | v] buffer
                wide = torch.zeros(tokens, 4 * Hkv * D, device="cuda", dtype=dt)
                wide[:, 2 * Hkv * D:3 * Hkv * D] = k.view(tokens, -1)
                wide[:, 3 * Hkv * D:] = v.view(tokens, -1)
                k, v = (wide[:, i * Hkv * D:(i + 1) * Hkv * D].unflatten(1, (Hkv, D)) for i in (2, 3))
            s["k"], s["v"] = k, v
            if case["skip"]:
                s["slots"][torch.rand(tokens, device="cuda", generator=g) < case["skip"]] = -1
            s["k_back"], s["v_back"] = (torch.empty(tokens, Hkv, D, device="cuda", dtype=dt) for _ in range(2))
        else:
            _fill(cache, ps, Hkv, D, g)
            s["k_out"], s["v_out"] = (torch.empty(tokens, Hkv, D, device="cuda", dtype=dt) for _ in range(2))
    else:
        _fill(cache, ps, Hkv, D, g)
        B, T, Hq = case["batch"], case["q_len"], Hkv * case["group"]
        lens = torch.tensor(_lens(case), device="cuda", dtype=torch.int32)
        s["lens"], s["table"] = lens, order.view(B, per)
        s["q"] = (torch.randn(B, T, Hq, D, device="cuda", generator=g) * 1.2).to(dt)
        s["out"] = torch.empty(B, T, Hq, D, device="cuda", dtype=dt)
        if kind == "step":
            s["k"], s["v"] = _kv(B, Hkv, D, g, dt)
            s["k_back"], s["v_back"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
            last = (lens - 1).long()
            s["slots"] = (s["table"].long().gather(1, (last // ps)[:, None])[:, 0] * ps + last % ps).int()
    s["cache"] = cache
    if own:
        from aljabr_b200.kv4 import Kv4Cache
        s["kv4"] = Kv4Cache(pages, ps, Hkv, D, data=cache)
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
    n, at, got = page_size * D // 2, 0, []
    for size in (n, n, n // 8, n // 8):
        got.append(c[:, :, at:at + size].unflatten(2, (page_size, -1)))
        at += size
    return got


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


def _write(cache, which, page, row, codes, d, kv_heads, page_size, D):
    """Writes the rows (page, row) of every kv head."""
    parts = _parts(cache, kv_heads, page_size, D)
    parts[which][page, :, row] = _pack(codes, which)
    parts[2 + which][page, :, row] = d.contiguous().view(torch.uint8)


def _gather(cache, which, page, row, kv_heads, page_size, D):
    """Values [..][kv_heads][D] of the rows (page, row), in fp32."""
    parts = _parts(cache, kv_heads, page_size, D)
    codes = _unpack(parts[which][page, :, row], which)
    d = parts[2 + which][page, :, row].contiguous().view(torch.float16)
    return _values(codes, d)


def _plain_append(s, k, v):
    c = s["case"]
    ps, Hkv, D = c["page_size"], c["kv_heads"], c["head_dim"]
    keep = s["slots"] >= 0
    at = s["slots"][keep].long()
    back = []
    for which, x in enumerate((k, v)):
        codes, d = _quantise(x.float())
        _write(s["cache"], which, at // ps, at % ps, codes[keep], d[keep], Hkv, ps, D)
        back.append(torch.where(keep[:, None, None], _values(codes, d), 0.0).to(x.dtype))
    return back


def _plain_attend(s):
    c = s["case"]
    ps, Hkv, D, T, G, B = c["page_size"], c["kv_heads"], c["head_dim"], c["q_len"], c["group"], c["batch"]
    pos = torch.arange(c["max_len"], device="cuda")
    page = s["table"].long()[:, pos // ps]
    row = (pos % ps).expand(B, -1)
    k, v = (_gather(s["cache"], i, page, row, Hkv, ps, D) for i in (0, 1))           # [B][S][Hkv][D]
    q = s["q"].float().view(B, T, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, T * G, D)
    sc = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(D))                # [B][Hkv][T G][S]
    if c["soft_cap"]:
        sc = torch.tanh(sc / c["soft_cap"]) * c["soft_cap"]
    hi = s["lens"].long()[:, None] - T + torch.arange(T, device="cuda")              # last position of each query
    seen = pos <= hi[..., None]
    if c["window"]:
        seen &= pos > hi[..., None] - c["window"]
    seen = seen.repeat_interleave(G, 1)[:, None]                                      # [B][1][T G][S]
    sc = torch.where(seen, sc, -torch.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == -torch.inf, torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(l == 0, torch.ones_like(l), l)
    return o.view(B, Hkv, T, G, D).permute(0, 2, 1, 3, 4).reshape(B, T, Hkv * G, D).to(s["q"].dtype)


def _plain_logits(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    h = s["history"].long()
    live = torch.arange(h.shape[1], device="cuda") < s["history_len"][:, None]
    count = torch.zeros_like(x).scatter_add_(1, h, live.float())
    rep, freq, pres = (s["penalties"][:, i:i + 1] for i in range(3))
    hit = count > 0
    x = torch.where(hit, torch.where(x > 0, x / rep, x * rep) - freq * count - pres, x)
    if s["bias_tokens"] is not None:
        x = x.scatter_add(1, s["bias_tokens"].long(), s["bias_values"])
    allowed = torch.ones_like(hit)
    if s["allow"] is not None:
        bits = (s["allow"][..., None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        allowed = bits.flatten(1)[:, :vocab] != 0
        x = torch.where(allowed, x, -torch.inf)
    can = allowed & ~x.isnan()
    best = torch.where(can, x, -torch.inf).amax(1, keepdim=True)
    first = (can & (x == best)).int().argmax(1)
    token = torch.where(can.any(1), first, -1).int()
    return [x, token]


def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        if kind == "logits":
            from aljabr_b200.logits import process_logits
            return list(process_logits(s["logits"], history=s["history"], history_len=s["history_len"],
                                       penalties=s["penalties"], bias_tokens=s["bias_tokens"],
                                       bias_values=s["bias_values"], bias_len=s["bias_len"], allow=s["allow"],
                                       out=s["out"], token=s["token"]))
        cache = s["kv4"]
        if kind == "read":
            return list(cache.read(s["slots"], k_out=s["k_out"], v_out=s["v_out"]))
        got = []
        if kind in ("append", "step"):
            cache.append(s["k"], s["v"], s["slots"], k_back=s["k_back"], v_back=s["v_back"])
            got = [s["k_back"], s["v_back"]]
        if kind in ("attend", "step"):
            got.insert(0, cache.attend(s["q"], s["lens"], s["table"], window=c["window"], soft_cap=c["soft_cap"],
                                       out=s["out"]))
        return got
    if kind == "logits":
        return _plain_logits(s)
    if kind == "read":
        ps, Hkv, D = c["page_size"], c["kv_heads"], c["head_dim"]
        at = s["slots"].long()
        return [_gather(s["cache"], i, at // ps, at % ps, Hkv, ps, D).to(_dtype(c)) for i in (0, 1)]
    got = []
    if kind in ("append", "step"):
        got = _plain_append(s, s["k"], s["v"])
    if kind in ("attend", "step"):
        got.insert(0, _plain_attend(s))
    return got


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


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "logits":
        x = s["logits"].double()
        vocab = x.shape[1]
        for r in range(x.shape[0]):
            n = int(s["history_len"][r])
            tokens, times = torch.unique(s["history"][r, :n].long(), return_counts=True)
            rep, freq, pres = s["penalties"][r].double().tolist()
            y = x[r, tokens]
            x[r, tokens] = torch.where(y > 0, y / rep, y * rep) - freq * times.double() - pres
            if s["bias_tokens"] is not None:
                x[r].index_add_(0, s["bias_tokens"][r].long(), s["bias_values"][r].double())
            if s["allow"] is not None:
                at = torch.arange(vocab, device="cuda")
                bit = (s["allow"][r][at // 32] >> (at % 32).int()) & 1
                x[r, bit == 0] = -math.inf
        return [x, None]
    ps, Hkv, D = case["page_size"], case["kv_heads"], case["head_dim"]
    if kind == "read":
        at = s["slots"].long()
        return [_rows64(s["cache"], i, at // ps, at % ps, Hkv, ps, D) for i in (0, 1)]
    back = []
    if kind in ("append", "step"):
        back = [torch.where((s["slots"] >= 0)[:, None, None], _round64(x.double()), 0.0) for x in (s["k"], s["v"])]
        if kind == "append":
            return back
    B, T, G = case["batch"], case["q_len"], case["group"]
    out = torch.zeros(B, T, Hkv * G, D, device="cuda", dtype=torch.float64)
    for b, n in enumerate(_lens(case)):
        if n == 0:
            continue
        pos = torch.arange(n, device="cuda")
        page = s["table"][b].long()[pos // ps]
        k, v = (_rows64(s["cache"], i, page, pos % ps, Hkv, ps, D) for i in (0, 1))
        if kind == "step":
            k[n - 1], v[n - 1] = back[0][b], back[1][b]
        for t in range(T):
            hi = n - T + t
            if hi < 0:
                continue
            lo = max(0, hi - case["window"] + 1) if case["window"] else 0
            q = s["q"][b, t].double().view(Hkv, G, D)
            sc = torch.einsum("hgd,shd->hgs", q, k[lo:hi + 1]) / math.sqrt(D)
            if case["soft_cap"]:
                sc = torch.tanh(sc / case["soft_cap"]) * case["soft_cap"]
            out[b, t] = torch.einsum("hgs,shd->hgd", sc.softmax(-1), v[lo:hi + 1]).reshape(Hkv * G, D)
    return [out] + back
