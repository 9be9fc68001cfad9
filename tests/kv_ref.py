"""The paged 4-bit K/V cache in numpy: its format, and attention and appending in 64 bits (tests of ha_kv_*)."""
import numpy as np

EPS, THETA = 1e-6, 1e7


def nibble_of(HD):
    """The nibble in which each channel of a row stands."""
    c, G = np.arange(HD), HD // 4
    return 16 * ((c % G) // 4) + 4 * (c // G) + c % 4


def quantise(x):
    """(codes, scales, zeros) of f32 rows [..., HD]; scales and zeros f16 [..., 4]. Each operation rounds to f32."""
    f = np.float32
    v = np.asarray(x, f).reshape(x.shape[:-1] + (4, x.shape[-1] // 4))
    with np.errstate(all="ignore"):
        lo, hi = v.min(-1), v.max(-1)
        z = (lo + (hi - lo) * f(8 / 15)).astype(np.float16)
        s = np.maximum((hi - z.astype(f)) * f(1 / 7), (z.astype(f) - lo) * f(0.125)).astype(np.float16)
        bad = ~(np.isfinite(s) & np.isfinite(z) & np.isfinite(v).all(-1))
        s, z = np.where(bad, np.float16(np.nan), s), np.where(bad, np.float16(0), z)
        r = np.rint((v - z.astype(f)[..., None]) / s.astype(f)[..., None]) + f(8)
        c = np.where(s[..., None] > 0, np.clip(r, 0, 15), 8)
    return np.nan_to_num(c, nan=8).astype(np.int64).reshape(x.shape), s, z


def values(c, s, z):
    """What codes stand for, f64."""
    v = c.reshape(c.shape[:-1] + (4, c.shape[-1] // 4)).astype(np.float64) - 8
    return (v * s.astype(np.float64)[..., None] + z.astype(np.float64)[..., None]).reshape(c.shape)


class Pool:
    """Pages [n_pages][HK][2] blocks as bytes."""

    def __init__(self, n_pages, page, HK, HD, fill=None):
        self.n_pages, self.page, self.HK, self.HD = n_pages, page, HK, HD
        self.data = np.zeros((n_pages, HK, 2, page * (HD // 2 + 16)), np.uint8) if fill is None else fill

    def codes(self):
        return self.data[..., :self.page * self.HD // 2].reshape(self.n_pages, self.HK, 2, self.page, self.HD // 2)

    def params(self):
        """f16 [n_pages][HK][2][page / 4][4 groups][s, z][4 tokens]"""
        p = np.ascontiguousarray(self.data[..., self.page * self.HD // 2:]).view(np.float16)
        return p.reshape(self.n_pages, self.HK, 2, self.page // 4, 4, 2, 4)

    def put(self, page, slot, kh, which, row):
        c, s, z = quantise(row.astype(np.float32))
        nib = np.zeros(self.HD, np.uint8)
        nib[nibble_of(self.HD)] = c
        blk = self.data[page, kh, which]
        blk[slot * self.HD // 2:(slot + 1) * self.HD // 2] = nib[0::2] | nib[1::2] << 4
        par = blk[self.page * self.HD // 2:].view(np.float16).reshape(self.page // 4, 4, 2, 4)
        par[slot // 4, :, 0, slot % 4], par[slot // 4, :, 1, slot % 4] = s, z

    def put_rows(self, page, slot, kh, which, rows):
        """put() of rows [n][HD] at (page[n], slot[n])."""
        c, s, z = quantise(rows.astype(np.float32))
        nib = np.zeros(rows.shape, np.uint8)
        nib[:, nibble_of(self.HD)] = c
        self.codes()[page, kh, which, slot] = nib[:, 0::2] | nib[:, 1::2] << 4
        half = self.data[..., self.page * self.HD // 2:].view(np.float16)
        par = half.reshape(half.shape[:-1] + (self.page // 4, 4, 2, 4))
        assert np.shares_memory(par, self.data)
        par[page, kh, which, slot // 4, :, 0, slot % 4], par[page, kh, which, slot // 4, :, 1, slot % 4] = s, z

    def read(self, page, slot, kh, which):
        """Values [n][HD] (f64) of tokens at (page[n], slot[n])."""
        b = self.codes()[page, kh, which, slot].astype(np.int64)
        nib = np.stack([b & 15, b >> 4], -1).reshape(len(page), self.HD)[:, nibble_of(self.HD)]
        par = self.params()[page, kh, which, slot // 4, :, :, slot % 4]
        return values(nib, par[:, :, 0], par[:, :, 1])


def prep(x, w, pos, rot):
    """x [n][HD] (f64) normed with gain w, rotated at pos[n]."""
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * w.astype(np.float64)
    h = rot // 2
    a = pos[:, None] / THETA ** (2 * np.arange(h) / max(rot, 1))
    c, s = np.cos(a).astype(np.float32).astype(np.float64), np.sin(a).astype(np.float32).astype(np.float64)
    return np.concatenate([x[:, :h] * c - x[:, h:rot] * s, x[:, h:rot] * c + x[:, :h] * s, x[:, rot:]], -1)


def attend(pool, table, lens, start, q, gate, HQ, scale=None, rows=None):
    """f64 outputs {row: [HQ][HD]} of q [n_rows][HQ][HD] over the pool; rows: those asked for (default all)."""
    HK, HD, ps = pool.HK, pool.HD, pool.page
    scale = 1 / np.sqrt(HD) if scale is None else scale
    out = {}
    for b in range(len(lens)):
        n = start[b + 1] - start[b]
        mine = [t for t in range(start[b], start[b + 1]) if rows is None or t in rows]
        if not mine:
            continue
        tok = np.arange(lens[b])
        page = table[b][tok // ps]
        kv = [[pool.read(page, tok % ps, h, w) for w in (0, 1)] for h in range(HK)]
        for t in mine:
            m = lens[b] - n + (t - start[b]) + 1
            o = np.empty((HQ, HD))
            for h in range(HQ):
                K, V = kv[h // (HQ // HK)]
                s = K[:m] @ q[t, h].astype(np.float64) * scale
                p = np.exp(s - s.max())
                o[h] = p @ V[:m] / p.sum()
            out[t] = o / (1 + np.exp(-gate[t].astype(np.float64))) if gate is not None else o
    return out
