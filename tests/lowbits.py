"""Plain 64-bit forms of the 4-bit weight and 8-bit cache operators, from the formats' definitions (numpy)."""
import numpy as np

E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6], np.float64)
E4M3 = np.array([np.nan if c & 127 == 127 else (-1) ** (c >> 7) * (
    (c & 7) * 2.0 ** -9 if (c >> 3) & 15 == 0 else (1 + (c & 7) / 8) * 2.0 ** (((c >> 3) & 15) - 7)) for c in range(256)])


def bf16_bits(a):
    u = np.ascontiguousarray(a, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r).astype(np.uint16)


def bf16_value(h):
    return (np.asarray(h, np.uint16).astype(np.uint32) << 16).view(np.float32)


def _nearest(table, x):
    """Index of the nearest table value (ascending, codes 0..), ties to the even code; x >= 0, at most the last."""
    hi = np.searchsorted(table, x).clip(1, len(table) - 1)
    lo = hi - 1
    mid = (table[lo] + table[hi]) / 2
    up = (x > mid) | ((x == mid) & (hi % 2 == 0))
    return np.where(up, hi, lo)


def mx_quantize(x):
    """f32 rows -> (packed codes [rows, G * 64], scales [rows, G * 4])."""
    rows, k = x.shape
    g = -(-k // 128)
    w = np.zeros((rows, g * 128), np.float64)
    w[:, :k] = x
    w = w.reshape(rows, g * 4, 32)
    with np.errstate(invalid="ignore"):
        amax = np.abs(w).max(2)
    bad = ~np.isfinite(amax)
    _, ex = np.frexp(np.where(bad | (amax == 0), 1.0, amax))
    e = np.where(amax == 0, -127, (ex - 1 - 2).clip(-127, 127))
    a = np.where(bad[..., None], 0.0, np.abs(np.where(bad[..., None], 0.0, w)) * np.exp2(-e.astype(np.float64))[..., None])
    code = _nearest(E2M1, np.minimum(a, 6.0)) | (np.signbit(w) << 3)
    code = np.where(bad[..., None], 0, code).astype(np.uint8).reshape(rows, -1, 2)
    return code[..., 0] | code[..., 1] << 4, np.where(bad, 255, e + 127).astype(np.uint8)


def mx_values(q, s, k):
    c = np.stack([q & 15, q >> 4], -1).reshape(q.shape[0], -1, 32)
    v = np.where(c & 8, -E2M1[c & 7], E2M1[c & 7])
    sc = np.where(s == 255, np.nan, np.exp2(s.astype(np.float64) - 127))
    return (v * sc[..., None]).reshape(q.shape[0], -1)[:, :k]


def e4m3_codes(x):
    """f64 values of at most 448 in magnitude (or NaN) -> codes, to nearest even."""
    mag = _nearest(E4M3[:127], np.where(np.isnan(x), 0, np.abs(x)))
    return np.where(np.isnan(x), 127, mag | (np.signbit(x) << 7)).astype(np.uint8)


def cache_scale(x):
    """The byte of the least 2^e with max |finite x| <= 448 * 2^e."""
    f = np.abs(np.where(np.isfinite(x), x, 0)).astype(np.float64)
    amax = f.max() if f.size else 0.0
    if amax == 0:
        return 0
    e = int(np.ceil(np.log2(amax / 448)))
    while 448 * 2.0 ** e < amax:
        e += 1
    while 448 * 2.0 ** (e - 1) >= amax:
        e -= 1
    return max(-127, e) + 127


class Cache:
    """A pool of pages on the host, kept as the device keeps it."""

    def __init__(self, pages, heads, page, dim, rng=None):
        shape_k, shape_v = (pages, heads, page, dim), (pages, heads, dim, page)
        fill = (lambda s: rng.integers(0, 256, s, dtype=np.uint8)) if rng else (lambda s: np.zeros(s, np.uint8))
        self.k, self.v = fill(shape_k), fill(shape_v)
        self.ks, self.vs = fill((pages, heads)), fill((pages, heads))
        self.pages, self.heads, self.page, self.dim = pages, heads, page, dim

    def append(self, table, lens, starts, nk, nv):
        """nk, nv [rows, heads, dim] f32."""
        for b, length in enumerate(lens):
            n = starts[b + 1] - starts[b]
            if length < n:
                continue
            at = length - n
            while at < length:
                slot, a = divmod(at, self.page)
                c = min(self.page - a, length - at)
                p = table[b][slot] if slot < len(table[b]) else -1
                row = starts[b] + at - (length - n)
                if 0 <= p < self.pages:
                    for h in range(self.heads):
                        for codes, scales, new in ((self.k[p, h], self.ks, nk), (self.v[p, h].T, self.vs, nv)):
                            x = new[row:row + c, h].astype(np.float64)
                            had = int(scales[p, h])
                            s = max(cache_scale(x), had if a else 0)
                            if a and s > had:
                                old = codes[:a]
                                r = e4m3_codes(E4M3[old] * 2.0 ** (had - s))
                                codes[:a] = np.where(old & 127 == 127, old, r)
                            codes[a:a + c] = e4m3_codes(np.where(np.isfinite(x), x, np.nan) * 2.0 ** (127 - s))
                            scales[p, h] = s
                at += c

    def tokens(self, row, length):
        """(k, v [length, heads, dim] values, present [length])."""
        slots = np.arange(length) // self.page
        ids = np.array([row[s] if s < len(row) else -1 for s in slots], np.int64).reshape(-1)
        there = (ids >= 0) & (ids < self.pages)
        p, t = np.where(there, ids, 0), np.arange(length) % self.page
        k = E4M3[self.k[p, :, t]] * np.exp2(self.ks[p].astype(np.float64) - 127)[..., None]
        v = E4M3[self.v[p, :, :, t]] * np.exp2(self.vs[p].astype(np.float64) - 127)[..., None]
        return k, v, there

    def attend(self, table, lens, starts, q, scale, window=0):
        """(out, bound of an output's |V| times the scores' condition) for q [rows, q_heads, dim]."""
        rows, qh, _ = q.shape
        out, vmax, cond = np.zeros(q.shape), np.zeros((rows, qh)), np.zeros((rows, qh))
        group = qh // self.heads
        for b, length in enumerate(lens):
            n = starts[b + 1] - starts[b]
            k, v, there = self.tokens(table[b], max(length, 0))
            for i in range(n):
                t = length - n + i
                sees = there & (np.arange(len(there)) <= t)
                if window:
                    sees &= np.arange(len(there)) > t - window
                if not sees.any():
                    continue
                for h in range(qh):
                    kk, vv, x = k[sees, h // group], v[sees, h // group], q[starts[b] + i, h].astype(np.float64)
                    with np.errstate(invalid="ignore", over="ignore"):
                        s = (kk @ x) * scale
                        w = np.exp(s - s.max())
                        o = (w[:, None] * vv).sum(0) / w.sum()
                        cond[starts[b] + i, h] = (np.abs(kk) @ np.abs(x)).max() * scale
                    out[starts[b] + i, h] = o
                    vmax[starts[b] + i, h] = np.nanmax(np.abs(vv), initial=0.0)
        return out, vmax, cond
