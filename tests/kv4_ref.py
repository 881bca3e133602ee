"""The 4-bit KV cache in plain numpy, written from the description in
include/aljabr_blackwell.h: quantiser, layout, and attention in 64 bits."""
import numpy as np


def quantise(x):
    """x [.., D] -> codes uint8 [.., D], scales float16 [.., D/32], in fp32 arithmetic."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        top, bottom = g.max(-1), g.min(-1)
        ext = np.where(-bottom >= top, bottom, top)
        finite = np.isfinite(g).all(-1)
        d = np.where(finite, np.clip(ext * np.float32(-0.125), -65504, 65504), np.nan).astype(np.float16)
        df = d.astype(np.float32)
        inv = np.where(df == 0, np.float32(0), np.float32(1) / df).astype(np.float32)
        c = np.clip(np.rint(g * inv[..., None]) + np.float32(8), 0, 15)
        c = np.where(finite[..., None], c, 8)
    return c.astype(np.uint8).reshape(x.shape), d


def values(codes, d):
    g = codes.reshape(*codes.shape[:-1], -1, 32).astype(np.float64) - 8
    with np.errstate(all="ignore"):
        return (g * d.astype(np.float64)[..., None]).reshape(codes.shape)


class RefCache:
    """Byte-exact image of a cache, one row at a time."""

    def __init__(self, pages, page_size, kv_heads, head_dim, fill=0):
        self.pages, self.ps, self.hkv, self.D, self.NG = pages, page_size, kv_heads, head_dim, head_dim // 32
        self.block = page_size * (head_dim + head_dim // 8)
        self.data = np.full(pages * kv_heads * self.block, fill, np.uint8)

    def _places(self, slot, head):
        page, off = divmod(slot, self.ps)
        at = (page * self.hkv + head) * self.block
        row, sc = self.D // 2, 2 * self.NG
        k, v = at + off * row, at + self.ps * row + off * row
        ks = at + 2 * self.ps * row + off * sc
        return k, v, ks, ks + self.ps * sc

    def write(self, slot, head, k, v):
        kp, vp, ksp, vsp = self._places(slot, head)
        for which, (x, at, sat) in enumerate(((k, kp, ksp), (v, vp, vsp))):
            codes, d = quantise(x)
            self.data[sat:sat + 2 * self.NG] = np.frombuffer(d.tobytes(), np.uint8)
            row = np.zeros(self.D // 2, np.uint8)
            for dim in range(self.D):
                g, j = divmod(dim, 32)
                if which == 0:
                    bit = 8 * 4 * ((j // 8) * self.NG + g) + 4 * (j % 8)
                else:
                    bit = 8 * 2 * ((j // 4) * self.NG + g) + 4 * (j % 4)
                row[bit // 8] |= codes[dim] << (bit % 8)
            self.data[at:at + self.D // 2] = row


def attention(q, k, v, n, window=0, scale=None, soft_cap=0.0):
    """q [T][Hq][D], k / v [S][Hkv][D] (values, 64 bits), n cached positions.  Returns out [T][Hq][D] and
    |.|: sum_p P |v| and the largest scores error weight of each row (see the bound in the tests)."""
    T, Hq, D = q.shape
    G = Hq // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, weight = np.zeros((T, Hq, D)), np.zeros((T, Hq, D))
    delta = np.zeros((T, Hq))
    for t in range(T):
        hi = n - T + t
        lo = max(0, hi - window + 1) if window else 0
        if hi < 0:
            continue
        for h in range(Hq):
            kk, vv = k[lo:hi + 1, h // G], v[lo:hi + 1, h // G]
            qq = q[t, h].astype(np.float64)
            s = kk @ qq * scale
            if soft_cap:
                s = np.tanh(s / soft_cap) * soft_cap
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, h], weight[t, h] = p @ vv, p @ np.abs(vv)
            # the scale of a group is at most its largest value / 7; codes enter with the offset -8
            top = np.abs(kk).reshape(len(kk), -1, 32).max(-1).repeat(32, -1)
            delta[t, h] = scale * np.abs(qq).max() * (np.abs(kk) + 8 / 7 * top).sum(-1).max() + np.abs(s).max() + soft_cap
    return out, weight, delta
