"""The head's losses and the gated block over rows in 64 bits, with bounds on
what the kernels may be off by.

Products: operands are sums of bf16 terms. Terms that are left out weigh at
most 2^-13 of a product for 16-bit rows (the second of two times the second,
each below 2^-7 of its value), 2^-19 for f32 ones (the second times the third
and the third times the second, 2^-21 each); beside 16-bit rows a weight has two
terms at most, cut at 2^-7 and rounded at 2^-8, so that Q8_0 and f32 ones are off by
2^-15 more. Where every pair is multiplied and the weight whole nothing is left out. Sums are f32: a matrix instruction adds 32
products to a running sum and rounds once, by 2^-23 of what it has at most.
Exponentials are the hardware's, 2^-22, of an argument rounded by 2^-24 twice.
A value held as T terms between two products is off by 2^-8 (one), 2^-15 (two:
cut at 2^-7, rounded at 2^-8) or 2^-22 of itself. Results are rounded by half a
step of their type."""
import math

import numpy as np

from ditch_amd import hipmem

TERMS = {"bf16": 1, "f16": 2, "f32": 3}
W_TERMS = {"bf16": 1, "fp8": 1, "mxfp4": 1, "int4": 1, "f16": 2, "q8_0": 3, "f32": 3}
HELD = {1: 2.0 ** -8, 2: 2.0 ** -15, 3: 2.0 ** -22}
HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
LEAST = {"bf16": 2.0 ** -133, "f16": 2.0 ** -25, "f32": 2.0 ** -149}
LEFT_OUT = {1: 2.0 ** -13, 2: 2.0 ** -13, 3: 2.0 ** -19}


def to_rows(a, dtype):
    """a as the row type's own numbers: the stored array and its values in 64 bits."""
    a = np.asarray(a, dtype=np.float32)
    if dtype == "f32":
        return a, a.astype(np.float64)
    if dtype == "f16":
        h = a.astype(np.float16)
        return h, h.astype(np.float64)
    b = a.view(np.uint32)
    b = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return b, from_rows(b, "bf16")


def from_rows(a, dtype):
    if dtype == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


STORE = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}
FILL = 0x5A


class Rows:
    """Rows in device memory, `gap` elements wider than their width, with a
    pattern between the rows and behind the last."""

    def __init__(self, dev, n, width, dtype, values=None, gap=0):
        self.n, self.width, self.dtype, self.stride = n, width, dtype, width + gap
        raw = np.full((n * self.stride + 64) * STORE[dtype]().itemsize, FILL, dtype=np.uint8).view(STORE[dtype])
        if values is not None:
            stored, self.values = to_rows(values, dtype)
            raw[:n * self.stride].reshape(n, self.stride)[:, :width] = stored
        self.buf = hipmem.Buffer.from_array(raw)
        self.size = raw.size
        used = ((n - 1) * self.stride + width) if n else 0
        self.desc = dev.kv_rows(self.buf.ptr, used * raw.itemsize, self.stride)

    def get(self):
        """The rows' values; checks that nothing else was written."""
        raw = self.buf.download(STORE[self.dtype], (self.size,))
        rows = raw[:self.n * self.stride].reshape(self.n, self.stride)
        pattern = np.full(raw.itemsize, FILL, dtype=np.uint8).view(STORE[self.dtype])[0]
        same = lambda v: (v.view(np.uint16 if v.itemsize == 2 else np.uint32) ==  # noqa: E731
                          np.asarray(pattern).view(np.uint16 if v.itemsize == 2 else np.uint32)).all()
        assert same(np.ascontiguousarray(rows[:, self.width:])) and same(raw[self.n * self.stride:])
        return from_rows(rows[:, :self.width], self.dtype)


class Floats:
    """n floats in device memory with a pattern behind them."""

    def __init__(self, n, values=None):
        raw = np.full((n + 16) * 4, FILL, dtype=np.uint8).view(np.float32)
        if values is not None:
            raw[:n] = values
        self.n, self.buf = n, hipmem.Buffer.from_array(raw)

    @property
    def ptr(self):
        return self.buf.ptr

    def get(self):
        raw = self.buf.download(np.float32, (self.n + 16,))
        assert (raw[self.n:].view(np.uint8) == FILL).all()
        return raw[:self.n].astype(np.float64)


class Workspace:
    """Scratch of NaN patterns with a pattern behind it."""

    def __init__(self, need):
        self.need = int(need)
        self.buf = hipmem.Buffer.from_array(np.full(self.need + 64, 0xFF, dtype=np.uint8))

    @property
    def args(self):
        return self.buf.ptr, self.need

    def check(self):
        tail = self.buf.download(np.uint8, (self.need + 64,))[self.need:]
        assert (tail == 0xFF).all()


def _pairs(order, a, b):
    return sum(1 for i in range(a) for j in range(b) if i + j < order)


def product_off(size, k, dtype, fmt, order=None):
    """How far a product whose absolute terms sum to `size` may be off."""
    a, full = TERMS[dtype], W_TERMS[fmt] if fmt in W_TERMS else int(fmt)
    b = full if a == 3 else min(full, 2)
    order = max(a, b) if order is None else order
    left = 0 if _pairs(order, a, b) == a * b and b == full else LEFT_OUT[a]
    return size * (left + (_pairs(order, a, b) * (k // 32 + 2) + 1) * 2.0 ** -23)


def _lse(l):
    m = l.max(1)
    return m + np.log(np.exp(l - m[:, None]).sum(1))


def logits(x, w, dtype, fmt):
    """Logits and their bounds."""
    return x @ w.T, product_off(np.abs(x) @ np.abs(w).T, x.shape[1], dtype, fmt)


def _softmax(l, off):
    """Log sums, their bounds, probabilities, their bounds."""
    lse = _lse(l)
    p = np.exp(l - lse[:, None])
    e = 2.0 ** -21 + np.abs(l - l.max(1, keepdims=True)) * 2.0 ** -23
    lse_off = (p * (off + e)).sum(1) + 2.0 ** -22
    lse_off += np.abs(lse) * 2.0 ** -24
    e = off + lse_off[:, None] + 2.0 ** -21 + np.abs(l - lse[:, None]) * 2.0 ** -22
    return lse, lse_off, p, p * e


def loss(x, w, targets, dtype, fmt):
    """{name: (value, bound)} of loss and lse."""
    l, off = logits(x, w, dtype, fmt)
    lse, lse_off, _, _ = _softmax(l, off)
    live, at = targets >= 0, np.clip(targets, 0, w.shape[0] - 1)
    r = np.arange(len(x))
    v = np.where(live, lse - l[r, at], 0.0)
    v[targets >= w.shape[0]] = np.nan
    return {"loss": (v, np.where(live, lse_off + off[r, at] + np.abs(v) * 2.0 ** -24, 0)), "lse": (lse, lse_off)}


def _back(d, d_off, other, k, dtype, fmt, order):
    """d @ other and its bound, d held as the row type's terms."""
    held = np.abs(d) * HELD[TERMS[dtype]] + LEAST["bf16"]
    v = d @ other
    off = (d_off + held) @ np.abs(other) + product_off(np.abs(d) @ np.abs(other), k, dtype, fmt, order) * 2
    return v, off + np.abs(v) * HALF[dtype] + LEAST[dtype]


def _order(dtype, fmt):
    return max(TERMS[dtype], W_TERMS[fmt] if dtype == "f32" else min(W_TERMS[fmt], 2))


def loss_grad(x, w, targets, g, dtype, fmt):
    l, off = logits(x, w, dtype, fmt)
    _, _, p, p_off = _softmax(l, off)
    live = targets >= 0
    one = np.zeros_like(p)
    one[np.arange(len(x))[live], np.minimum(targets[live], w.shape[0] - 1)] = 1
    g = np.where(live, g, 0.0)
    d, d_off = (p - one) * g[:, None], (p_off + 2.0 ** -24) * np.abs(g)[:, None]
    return {"dx": _back(d, d_off, w, w.shape[0], dtype, fmt, _order(dtype, fmt)),
            "dw": _back(d.T, d_off.T, x, len(x), dtype, TERMS[dtype], TERMS[dtype])}


def kl(base, trial, w, dtype, fmt):
    lb, ob = logits(base, w, dtype, fmt)
    lt, ot = logits(trial, w, dtype, fmt)
    sb, sb_off, p, _ = _softmax(lb, ob)
    st, st_off, q, _ = _softmax(lt, ot)
    u = (lb - sb[:, None]) - (lt - st[:, None])
    v = (p * u).sum(1)
    # its derivatives by the logits are p (u - kl) and q - p; phi's sums and the log sums enter by their relative
    # accuracy times c = lse_trial - lse_base where that is small, whole where it is not
    off = (p * np.abs(u - v[:, None]) * ob + np.abs(q - p) * ot).sum(1)
    c, e = np.abs(st - sb), 2.0 ** -19 + 2.0 ** -22 * np.abs(lb - lb.max(1, keepdims=True))
    far = ((np.abs(lb - lt)) * p * e).sum(1)
    D = lb - lt
    phi0 = np.where(np.abs(D) < 1e-3, D * D / 2 - D ** 3 / 6, D + np.expm1(-np.clip(D, -700, None)))
    near = (p * phi0 * e).sum(1) + np.expm1(np.minimum(c, 1)) * 2.0 ** -20
    off += np.where(c > 0.99, far + 2.0 ** -20 * (1 + c), near) + np.abs(v) * 2.0 ** -20
    # products of the two logits' errors: second order
    off += (p * (ob + ot) ** 2).sum(1) + (q * (ob + ot) ** 2).sum(1)
    return {"kl": (v, off), "lse_base": (sb, sb_off), "lse_trial": (st, st_off)}


def kl_grad(base, trial, w, g, dtype, fmt):
    _, _, p, p_off = _softmax(*logits(base, w, dtype, fmt))
    _, _, q, q_off = _softmax(*logits(trial, w, dtype, fmt))
    d, d_off = (q - p) * g[:, None], (p_off + q_off) * np.abs(g)[:, None]
    return {"dx": _back(d, d_off, w, w.shape[0], dtype, fmt, _order(dtype, fmt))}


_erf = np.vectorize(math.erf)


def act(a, g):
    """Activation, its derivative, a bound on its second derivative."""
    with np.errstate(over="ignore"):
        if a in (0, 5):
            c = 1.0 if a == 0 else 1.702
            s = 1 / (1 + np.exp(-c * g))
            return g * s, s * (1 + c * g * (1 - s)), 0.5 * c * np.ones_like(g)
        if a == 1:
            k = math.sqrt(2 / math.pi)
            t = np.tanh(k * (g + 0.044715 * g ** 3))
            return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g), \
                np.ones_like(g)
        if a == 2:
            c = 0.5 * (1 + _erf(g / math.sqrt(2)))
            return g * c, c + g * np.exp(-g * g / 2) / math.sqrt(2 * math.pi), np.ones_like(g)
        r = np.maximum(g, 0)
        return (r, (g > 0) * 1.0, np.zeros_like(g)) if a == 3 else (r * r, 2 * r, 2 * np.ones_like(g))


def _gate_up(x, wg, wu, a, dtype, fmt):
    g, g_off = logits(x, wg, dtype, fmt)
    u, u_off = logits(x, wu, dtype, fmt)
    y, dy, curve = act(a, g)
    # the functions themselves: a few f32 roundings of values of the size of g and of 1
    own = 2.0 ** -20 * (np.abs(g) + (g * g if a == 4 else 0))
    y_off = own + (np.abs(dy) + curve * g_off) * g_off
    dy_off = 2.0 ** -20 * (1 + np.abs(g) + g * g) + curve * g_off + (1.0 * (np.abs(g) <= g_off) if a == 3 else 0)
    return y, y_off, dy, dy_off, u, u_off


def glu(x, wg, wu, a, dtype, fmt):
    y, y_off, _, _, u, u_off = _gate_up(x, wg, wu, a, dtype, fmt)
    v = y * u
    off = y_off * np.abs(u) + (np.abs(y) + y_off) * u_off + np.abs(v) * 2.0 ** -23
    return v, off + np.abs(v) * HALF[dtype] + LEAST[dtype]


def glu_grad(x, wg, wu, dout, a, dtype, fmt):
    y, y_off, dy, dy_off, u, u_off = _gate_up(x, wg, wu, a, dtype, fmt)
    dg, du = dout * u * dy, dout * y
    dg_off = np.abs(dout) * (np.abs(u) * dy_off + (np.abs(dy) + dy_off) * u_off) + np.abs(dg) * 2.0 ** -22
    du_off = np.abs(dout) * y_off + np.abs(du) * 2.0 ** -23
    k, order = wg.shape[0], _order(dtype, fmt)
    a1, a2 = _back(dg, dg_off, wg, 2 * k, dtype, fmt, order), _back(du, du_off, wu, 2 * k, dtype, fmt, order)
    # one sum over both: each part's running sums hold the other's too
    more = product_off(np.abs(dg) @ np.abs(wg) + np.abs(du) @ np.abs(wu), 2 * k, dtype, fmt, order)
    n = len(x)
    return {"dx": (a1[0] + a2[0], a1[1] + a2[1] + more),
            "dgate": _back(dg.T, dg_off.T, x, n, dtype, TERMS[dtype], TERMS[dtype]),
            "dup": _back(du.T, du_off.T, x, n, dtype, TERMS[dtype], TERMS[dtype])}


def check(got, want, off, what=""):
    """Every value within its bound; NaN and infinities where they are expected."""
    got, want = np.asarray(got), np.asarray(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=what)
    fine = np.isfinite(want)
    far = np.abs(got[fine] - want[fine]) - np.broadcast_to(off, want.shape)[fine]
    assert (far <= 0).all(), f"{what}: off by {far.max():.3g} more than allowed at {int(far.argmax())} of {far.size}"
