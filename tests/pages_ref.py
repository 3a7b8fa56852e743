"""The paged 8-bit cache in plain 64-bit numpy: the page format, append,
attention and fork from their definitions, for the tests of the kernels."""
import numpy as np

MOST = {"int8": 127.0, "e4m3": 448.0}


def padded(d):
    return -(-d // 64) * 64


def decode_table(kind):
    """The values of the 256 codes."""
    if kind == "int8":
        return np.arange(256, dtype=np.uint8).view(np.int8).astype(np.float64)
    c = np.arange(256)
    e, m = c >> 3 & 15, c & 7
    x = np.where(e > 0, (8.0 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)
    x[(e == 15) & (m == 7)] = np.nan
    return np.where(c & 128, -x, x)


def encode(y, kind):
    """The codes nearest to y (ties to even), clamped to the largest."""
    y = np.clip(y, -MOST[kind], MOST[kind])
    if kind == "int8":
        return np.rint(y).astype(np.int8).view(np.uint8)
    a = np.abs(y)
    e = np.maximum(np.floor(np.log2(np.maximum(a, 2.0 ** -30))), -6)
    e = np.where(a >= 2.0 ** (e + 1), e + 1, np.where((a < 2.0 ** e) & (e > -6), e - 1, e))
    n = np.rint(a / 2.0 ** (e - 3))  # steps of 2^(e - 3); 8..16 for a normal number
    up = n == 16
    e, n = np.where(up, e + 1, e), np.where(up, 8, n)
    code = np.where(n < 8, n, (e + 7) * 8 + n - 8).astype(np.uint8)
    return code | np.where(np.signbit(y), 128, 0).astype(np.uint8)


def offsets(page, hd, vd):
    """Byte of (token, dim) within a head's page: of the keys, of the values."""
    dk, dv = padded(hd), padded(vd)
    t, d = np.arange(page)[:, None], np.arange(dk)
    k = (t // 16 * (dk // 64) + d // 64) * 1024 + d % 64 // 16 * 256 + t % 16 * 16 + d % 16
    d = np.arange(dv)
    u = t % 32
    v = (t // 32 * (dv // 32) + d // 32) * 1024 + u % 16 // 4 * 256 + d % 16 * 16 + d % 32 // 16 * 8 + u // 16 * 4 + u % 4
    return k, page * dk + v


class Pool:
    """codes [layers][pages][kv_heads][bytes], scales [layers][pages][kv_heads][2]."""

    def __init__(self, kind, layers, n_pages, page, kv_heads, hd, vd=None, fill=0x25):
        self.kind, self.layers, self.n_pages, self.page, self.kv_heads = kind, layers, n_pages, page, kv_heads
        self.hd, self.vd = hd, hd if vd is None else vd
        self.bytes = page * (padded(self.hd) + padded(self.vd))
        self.codes = np.full((layers, n_pages, kv_heads, self.bytes), fill, dtype=np.uint8)
        self.scales = np.full((layers, n_pages, kv_heads, 2), 7.0, dtype=np.float32)
        self.off = offsets(page, self.hd, self.vd)
        self.values = decode_table(kind)

    def copy(self):
        p = Pool(self.kind, self.layers, self.n_pages, self.page, self.kv_heads, self.hd, self.vd)
        p.codes, p.scales = self.codes.copy(), self.scales.copy()
        return p

    def tokens(self, layer, page, which):
        """f64 values [kv_heads][page][dim] of a page's keys (0) or values (1)."""
        x = self.values[self.codes[layer, page][:, self.off[which]]]
        with np.errstate(invalid="ignore"):
            return (x * self.scales[layer, page, :, which].astype(np.float64)[:, None, None])[
                ..., :self.vd if which else self.hd]


def rotate(x, pos, cos, sin, style):
    """x [n][heads][dim] f64 at positions pos."""
    half = cos.shape[1]
    x = x.astype(np.float64)
    c, s = cos[pos].astype(np.float64)[:, None], sin[pos].astype(np.float64)[:, None]
    y = x.copy()
    a, b = (slice(0, half), slice(half, 2 * half)) if style == "neox" else (slice(0, 2 * half, 2),
                                                                             slice(1, 2 * half, 2))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def append(pool, layer, table, starts, pos, k, v, rope=None):
    """Appends in place; k, v [n][heads][dim]. Returns the pages and tokens that were written:
    {(page, head): live tokens}."""
    touched = {}
    for b in range(len(pos)):
        lo, n = int(starts[b]), int(starts[b + 1]) - int(starts[b])
        if n <= 0:
            continue
        at = int(pos[b]) + np.arange(n)
        kk = k[lo:lo + n].astype(np.float64)
        if rope:
            kk = rotate(kk, at, *rope)
        vv = v[lo:lo + n].astype(np.float64)
        for pi in range(int(pos[b]) // pool.page, (int(pos[b]) + n - 1) // pool.page + 1):
            page = int(table[b, pi])
            if not 0 <= page < pool.n_pages:
                continue
            sel = (at // pool.page) == pi
            t = at[sel] % pool.page
            keep = int(t[0])
            for h in range(pool.kv_heads):
                for which, x in ((0, kk), (1, vv)):
                    x = x[sel, h]
                    off = pool.off[which]
                    width = off.shape[1]
                    before = pool.scales[layer, page, h, which] if keep else np.float32(0)
                    most = np.max(np.abs(x)) if np.isfinite(x).all() else np.inf
                    with np.errstate(over="ignore"):
                        after = max(before, np.float32(most) * np.float32(1 / np.float32(MOST[pool.kind])))
                    if not np.isfinite(before) or not np.isfinite(after):
                        after = np.float32(np.nan)
                    pool.scales[layer, page, h, which] = after
                    inverse = 1 / np.float64(after) if after > 0 else 0.0
                    codes = pool.codes[layer, page, h]
                    if keep and after > before:
                        old = pool.values[codes[off[:keep]]]
                        codes[off[:keep]] = encode(old * (np.float64(before) * inverse), pool.kind)
                    full = np.zeros((len(t), width))
                    if not np.isnan(after):
                        full[:, :x.shape[1]] = x * inverse
                    codes[off[t]] = encode(full, pool.kind)
                touched[page, h] = int(t[-1]) + 1
    return touched


def sequence(pool, layer, row, n):
    """Keys and values f64 [kv_heads][n][dim] of a sequence's first n tokens (NaN where a page is none)."""
    out = [np.full((pool.kv_heads, -(-n // pool.page) * pool.page, d), np.nan) for d in (pool.hd, pool.vd)]
    for i in range(-(-n // pool.page)):
        if 0 <= row[i] < pool.n_pages:
            for which in (0, 1):
                out[which][:, i * pool.page:(i + 1) * pool.page] = pool.tokens(layer, int(row[i]), which)
    return out[0][:, :n], out[1][:, :n]


def attention(pool, layer, table, starts, pos, q, scale, window=0, sinks=0):
    """f64 out [n][heads][vd] and what the tests' tolerances are made of: per output the weighted mean of |v|, per
    head the largest score's sum of |q k|, the spread of the scores, and the largest code's value under the key that
    weighs most."""
    n, heads = q.shape[:2]
    group = heads // pool.kv_heads
    out = np.full((n, heads, pool.vd), np.nan)
    mass, size, spread, top = np.zeros((n, heads, pool.vd)), *(np.zeros((n, heads, 1)) for _ in range(3))
    for b in range(len(pos)):
        for i in range(int(starts[b + 1]) - int(starts[b])):
            r, t = int(starts[b]) + i, int(pos[b]) + i
            k, v = sequence(pool, layer, table[b], t + 1)
            j = np.arange(t + 1)
            seen = (t - j < window) | (j < sinks) if window else j <= t
            k, v = k[:, seen], v[:, seen]
            vs = np.stack([pool.scales[layer, max(table[b, x], 0) % pool.n_pages, :, 1] for x in j[seen] // pool.page], 1)
            for h in range(heads):
                kk, vv, qq = k[h // group], v[h // group], q[r, h].astype(np.float64)
                s = kk @ qq * scale
                if np.isnan(s).any() or np.isnan(vv).any():
                    continue
                w = np.exp(s - s.max())
                w /= w.sum()
                out[r, h], mass[r, h] = w @ vv, w @ np.abs(vv)
                size[r, h] = (np.abs(kk) @ np.abs(qq)).max() * abs(scale)
                spread[r, h] = s.max() - s.min()
                top[r, h] = (w * vs[h // group]).max() * MOST[pool.kind]
    return out, mass, size, spread, top


def fork(table, parents, spare, lens, page, beams):
    """(table_out, spare_out, [(source page, copy)])."""
    t_out, s_out, copies = table.copy(), spare.copy(), []
    for g in range(len(lens)):
        full, part = int(lens[g]) // page, int(lens[g]) % page
        first = g * beams
        par = [int(parents[first + c]) if 0 <= parents[first + c] < beams else c for c in range(beams)]
        has = part and full < table.shape[1]
        free = [table[first + p, full] for p in range(beams) if has and p not in par]
        for c, p in enumerate(par):
            t_out[first + c, :full] = table[first + p, :full]
            if not has:
                continue
            t_out[first + c, full] = table[first + p, full]
            if p in par[:c]:
                t_out[first + c, full] = spare[first + c]
                s_out[first + c] = free.pop(0)
                copies.append((int(table[first + p, full]), int(spare[first + c])))
    return t_out, s_out, copies
