"""Pages of 8-bit keys and values on the GPU: append, read, attention and
fork against the plain 64-bit form of pages_ref.py.

Append forms each value in 64 bits and rounds it once, so codes and scales
are compared for equality. Attention's tolerance per output, with
p the softmax weights and S = max_j scale * sum_d |q_d k_jd|:
  a score is off by at most d = (DK / 32 + 8) * 2^-23 * S + 2^-22 * spread
    (f32 accumulation over DK / 32 matrix products of 32, the split of q, the
    products with the scales; the exponent's rounding grows with the scores'
    spread), and a weight by a factor exp(+-d);
  numerator and denominator each follow, and their f32 sums over n keys add
    (n / 256 + 16) * 2^-24 each, so |out - exact| <= (2 d + (n / 256 + 16) *
    2^-23) * sum p |v|;
  weights enter the products as f16 with the largest (times its value scale)
    at 2^12 or above: what lies below f16's least step, 2^-24, may be dropped,
    2^-36 of the largest weight's code value a key: n * 2^-36 * top;
  16-bit rows: weights of 11 bits add 2^-12 * sum p |v|, the rounding of the
    output half a step, eps / 2 * |out|.
"""
import ctypes

import numpy as np
import pytest
import torch

import pages_ref as ref
from ditch_amd import abi, hipmem
from ditch_amd.hip import DeviceError

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _raw(x, dtype):
    """The bytes of x in a row type, and the values they stand for."""
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(TORCH[dtype])
    return t.view(torch.uint8 if dtype == "f32" else torch.int16).numpy() if dtype != "f32" else t.numpy(), \
        t.float().numpy()


def _values(raw, dtype):
    if dtype == "f32":
        return raw.view(np.float32)
    return torch.from_numpy(raw.view(np.int16)).view(TORCH[dtype]).float().numpy()


class Rows:
    """A row buffer [n][width] with a stride, a guard behind every row and after the last."""

    def __init__(self, dev, n, width, dtype, x=None, stride=None, fill=0x77):
        self.n, self.width, self.dtype, self.e = n, width, dtype, 4 if dtype == "f32" else 2
        self.stride = width if stride is None else stride
        self.nbytes = ((max(n, 1) - 1) * self.stride + width) * self.e
        self.host = np.full((max(n, 1) * self.stride + 64) * self.e, fill, dtype=np.uint8)
        if x is not None:
            raw, self.x = _raw(x.reshape(n, width), dtype)
            view = self.host[:n * self.stride * self.e].reshape(n, self.stride * self.e)
            view[:, :width * self.e] = raw.view(np.uint8).reshape(n, width * self.e)
        self.buf = hipmem.Buffer.from_array(self.host)
        self.desc = dev.kv_rows(self.buf.ptr.value, self.nbytes, self.stride)

    def get(self):
        """f32 values [n][width]; the guards must hold what they held."""
        got = self.buf.download(np.uint8, self.host.shape)
        rows = got[:self.n * self.stride * self.e].reshape(self.n, self.stride * self.e)
        was = self.host[:self.n * self.stride * self.e].reshape(self.n, self.stride * self.e)
        np.testing.assert_array_equal(rows[:, self.width * self.e:], was[:, self.width * self.e:])
        np.testing.assert_array_equal(got[self.n * self.stride * self.e:], self.host[self.n * self.stride * self.e:])
        return _values(np.ascontiguousarray(rows[:, :self.width * self.e]).reshape(-1), self.dtype).reshape(self.n,
                                                                                                          self.width)


class Setup:
    """A pool, some sequences' tables and their device copies."""

    def __init__(self, dev, pool, table):
        self.dev, self.pool, self.table = dev, pool, np.ascontiguousarray(table, dtype=np.int32)
        self.codes, self.scales = hipmem.Buffer.from_array(pool.codes), hipmem.Buffer.from_array(pool.scales)
        self.d_table = hipmem.Buffer.from_array(self.table)
        self.pages = dev.kv_pages(self.codes.ptr.value, pool.codes.nbytes, self.scales.ptr.value, pool.scales.nbytes,
                                  pool.kind, pool.layers, pool.n_pages, pool.page, pool.kv_heads, pool.hd, pool.vd)
        self.keep = []

    def batch(self, starts, pos, n_rows=None, max_rows=None, max_len=None):
        starts, pos = np.asarray(starts), np.asarray(pos)
        n = np.diff(starts)
        bs, bp = (hipmem.Buffer.from_array(a.astype(np.uint32)) for a in (starts, pos))
        self.keep += [bs, bp]
        return self.dev.kv_batch(self.d_table.ptr.value, self.table.shape[1], bs.ptr.value, bp.ptr.value, len(pos),
                                 int(starts[-1]) if n_rows is None else n_rows,
                                 int(n.max()) if max_rows is None else max_rows,
                                 int((pos + n).max()) if max_len is None else max_len)

    def download(self):
        self.dev.sync()
        p = self.pool.copy()
        p.codes = self.codes.download(np.uint8, p.codes.shape)
        p.scales = self.scales.download(np.float32, p.scales.shape)
        return p

    def attention(self, layer, batch, dtype, out, q, heads, scale, window=0, sinks=0, stream=None, ws=None):
        need = self.dev.kv_pages_attention_workspace(self.pages, batch, heads, dtype, window, sinks)
        if ws is None:
            ws = hipmem.Buffer(max(need, 1))
            ws.upload(np.full(max(need, 1), 0xFF, dtype=np.uint8))  # what it holds does not matter
            self.keep.append(ws)
        self.dev.kv_pages_attention(self.pages, layer, batch, dtype, out.desc, q.desc, heads, scale, ws.ptr.value,
                                    need, window=window, sinks=sinks, stream=stream)


def _tables(rng, pool, seqs, cols):
    return rng.permutation(pool.n_pages)[:seqs * cols].reshape(seqs, cols)


def _rope(rng, n, half):
    angle = np.arange(n)[:, None] * 1e4 ** (-np.arange(half) / max(half, 1))
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def _starts(n):
    return np.concatenate([[0], np.cumsum(n)])


def _compare_pools(got, want, touched, layer):
    """Live tokens of the touched pages, their scales, and every byte of every other page."""
    same_scales = want.scales.copy()
    np.testing.assert_array_equal(got.scales, same_scales)
    rest = np.ones(want.codes.shape[:2], dtype=bool)
    for (page, h), live in touched.items():
        rest[layer, page] = False
        for which in (0, 1):
            at = want.off[which][:live]
            a, b = want.values[got.codes[layer, page, h][at]], want.values[want.codes[layer, page, h][at]]
            np.testing.assert_array_equal(a, b)
    np.testing.assert_array_equal(got.codes[rest], want.codes[rest])


# ---------------------------------------------------------------------------
# append and read

APPEND = [
    # kind, dtype, heads, kv_heads, hd, vd, page, rotated, style, [(rows, pos)]
    ("int8", "f32", 4, 2, 64, 64, 32, 64, "neox", [(1, 0), (1, 31), (1, 32), (1, 45)]),
    ("e4m3", "bf16", 8, 8, 128, 128, 64, 128, "neox", [(70, 0), (0, 9), (5, 62), (1, 100), (130, 33)]),
    ("int8", "f16", 7, 1, 80, 80, 32, 40, "gptj", [(33, 1), (64, 32), (2, 31)]),
    ("e4m3", "f32", 2, 2, 192, 128, 128, 64, "neox", [(3, 126), (200, 60)]),
    ("int8", "bf16", 3, 3, 256, 256, 256, 0, "neox", [(1, 255), (17, 250), (300, 4)]),
    ("e4m3", "f16", 3, 1, 1, 1, 32, 0, "neox", [(5, 30)]),
    ("int8", "f32", 6, 3, 30, 30, 64, 30, "gptj", [(97, 63), (1, 0)]),
    ("e4m3", "bf16", 2, 1, 160, 160, 64, 160, "neox", [(1, 7), (100, 40)]),
    ("int8", "bf16", 3, 1, 64, 64, 32, 64, "neox", [(b % 3, 11 * b % 90) for b in range(200)]),
]


@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append_and_read(dev, case):
    kind, dtype, heads, kvh, hd, vd, page, rot, style, seqs = APPEND[case]
    rng = np.random.default_rng(case)
    cols = 8
    pool = ref.Pool(kind, 2, len(seqs) * cols + 3, page, kvh, hd, vd)
    table = _tables(rng, pool, len(seqs), cols)
    s = Setup(dev, pool, table)
    half = rot // 2
    rope = _rope(rng, 600, half) + (style,)
    d_cos, d_sin = (hipmem.Buffer.from_array(x if x.size else np.zeros(1, np.float32)) for x in rope[:2])
    desc = dev.kv_rope(d_cos.ptr.value, d_sin.ptr.value, 600, half, style)
    # what the pages hold in front of the new rows, then the rows, twice with growing and shrinking sizes
    touched = {}
    for step, size in enumerate((1.0, 2.5, 0.5)):
        rows = [p for _, p in seqs] if step == 0 else [r for r, _ in seqs]
        pos = [0] * len(seqs) if step == 0 else [p for _, p in seqs]
        starts = _starts(rows)
        n = int(starts[-1])
        if n == 0:
            continue
        b = s.batch(starts, pos, max_len=max(r + p for r, p in zip(rows, pos)))
        x = [rng.standard_normal((n, h * d)) * size for h, d in ((kvh, hd), (kvh, vd), (heads, hd))]
        k, v, q = Rows(dev, n, kvh * hd, dtype, x[0]), Rows(dev, n, kvh * vd, dtype, x[1], kvh * vd + 5), \
            Rows(dev, n, heads * hd, dtype, x[2])
        q_out = Rows(dev, n, heads * hd, dtype, stride=heads * hd + 3)
        dev.kv_pages_append(s.pages, 1, b, dtype, k.desc, v.desc, rope=desc, q=q.desc, q_out=q_out.desc, heads=heads)
        touched |= ref.append(pool, 1, table, starts, pos, k.x.reshape(n, kvh, hd), v.x.reshape(n, kvh, vd),
                              rope if half else None)
        _compare_pools(s.download(), pool, touched, 1)
        at = np.concatenate([np.arange(p, p + r) for r, p in zip(rows, pos)])
        want = q.x.reshape(n, heads, hd).astype(np.float64)
        want = ref.rotate(want, at, *rope) if half else want
        got = q_out.get().reshape(n, heads, hd)
        eps = torch.finfo(TORCH[dtype]).eps / 2
        # (from 64 bits through f32 to the row type: half a step of each)
        assert (np.abs(got - want) <= (eps + 2.0 ** -24) * np.abs(want) * 1.01 + 2.0 ** -25).all()
        # read back what each sequence holds
        ends = [r + p for r, p in zip(rows, pos)]
        rs = _starts(ends)
        ko, vo = Rows(dev, int(rs[-1]), kvh * hd, "f32", stride=kvh * hd + 1), Rows(dev, int(rs[-1]), kvh * vd, "f32")
        dev.kv_pages_read(s.pages, 1, s.batch(rs, [0] * len(seqs)), "f32", ko.desc, vo.desc)
        dev.sync()
        gk, gv = ko.get().reshape(-1, kvh, hd), vo.get().reshape(-1, kvh, vd)
        for i in range(len(seqs)):
            if ends[i]:
                wk, wv = ref.sequence(pool, 1, table[i], ends[i])
                np.testing.assert_array_equal(gk[rs[i]:rs[i + 1]], wk.transpose(1, 0, 2).astype(np.float32))
                np.testing.assert_array_equal(gv[rs[i]:rs[i + 1]], wv.transpose(1, 0, 2).astype(np.float32))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_read_rounds_to_the_row_type(dev, dtype):
    rng = np.random.default_rng(8)
    pool = ref.Pool("int8", 1, 2, 32, 2, 64)
    pool.codes[:] = rng.integers(-127, 128, pool.codes.shape).astype(np.int8).view(np.uint8)
    pool.scales[:] = rng.uniform(0.01, 0.02, pool.scales.shape)
    s = Setup(dev, pool, [[1, 0]])
    k, v = Rows(dev, 40, 128, dtype), Rows(dev, 40, 128, dtype)
    dev.kv_pages_read(s.pages, 0, s.batch([0, 40], [3]), dtype, k.desc, v.desc)
    dev.sync()
    wk, wv = ref.sequence(pool, 0, [1, 0], 43)
    for got, want in ((k, wk), (v, wv)):
        want = _raw(want[:, 3:].transpose(1, 0, 2).reshape(40, 128), dtype)[1]
        np.testing.assert_array_equal(got.get(), want)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_value_that_is_not_finite_poisons_its_page_and_head(dev, kind, bad):
    rng = np.random.default_rng(4)
    pool = ref.Pool(kind, 1, 3, 32, 2, 64)
    table = np.array([[2, 0]])
    s = Setup(dev, pool, table)
    for step, (lo, hi) in enumerate(((0, 10), (10, 12), (12, 40), (0, 5))):
        n = hi - lo
        x, y = rng.standard_normal((n, 2, 64)), rng.standard_normal((n, 2, 64))
        if step == 1:
            x[1, 1, 7] = bad
        k, v = Rows(dev, n, 128, "f32", x), Rows(dev, n, 128, "f32", y)
        dev.kv_pages_append(s.pages, 0, s.batch([0, n], [lo]), "f32", k.desc, v.desc)
        touched = ref.append(pool, 0, table, [0, n], [lo], k.x.reshape(n, 2, 64), v.x.reshape(n, 2, 64))
        got = s.download()
        np.testing.assert_array_equal(got.scales, pool.scales)
        assert np.isnan(got.scales[0, 2, 1, 0]) == (step in (1, 2)) and np.isfinite(got.scales[0, 2, 0]).all()
        for (page, h), live in touched.items():
            for which in (0, 1):
                if np.isfinite(pool.scales[0, page, h, which]):
                    at = pool.off[which][:live]
                    np.testing.assert_array_equal(pool.values[got.codes[0, page, h][at]],
                                                  pool.values[pool.codes[0, page, h][at]])


def test_values_of_zero_and_of_extreme_size(dev):
    for kind in ("int8", "e4m3"):
        for size in (0.0, 1e-42, 1e-38, 1e37, 3e38):
            rng = np.random.default_rng(2)
            pool = ref.Pool(kind, 1, 1, 32, 1, 64)
            s = Setup(dev, pool, [[0]])
            x = (rng.uniform(-1, 1, (9, 64)) * size).astype(np.float32)
            k, v = Rows(dev, 9, 64, "f32", x), Rows(dev, 9, 64, "f32", x[::-1].copy())
            dev.kv_pages_append(s.pages, 0, s.batch([0, 9], [0]), "f32", k.desc, v.desc)
            touched = ref.append(pool, 0, np.array([[0]]), [0, 9], [0], k.x.reshape(9, 1, 64), v.x.reshape(9, 1, 64))
            _compare_pools(s.download(), pool, touched, 0)


def test_bounds_far_above_what_there_is(dev):
    """max_rows and max_len up to their limits cost nothing but idle workgroups, or are refused."""
    rng = np.random.default_rng(18)
    pool = ref.Pool("int8", 1, 3, 32, 1, 64)
    s = Setup(dev, pool, [[2, 0, 1]])
    k = Rows(dev, 5, 64, "f32", rng.standard_normal((5, 64)))
    out = Rows(dev, 5, 64, "f32")
    for bound in (1 << 10, (1 << 31) - 1):
        b = s.batch([0, 5], [30], max_rows=bound, max_len=96)
        dev.kv_pages_append(s.pages, 0, b, "f32", k.desc, k.desc)
        touched = ref.append(pool, 0, np.array([[2, 0, 1]]), [0, 5], [30], k.x.reshape(5, 1, 64), k.x.reshape(5, 1, 64))
        got = s.download()
        for (page, h), live in touched.items():
            lo = 30 if page == 2 else 0
            np.testing.assert_array_equal(got.codes[0, page, h][got.off[0][lo:live]],
                                          pool.codes[0, page, h][pool.off[0][lo:live]])
        dev.kv_pages_read(s.pages, 0, b, "f32", out.desc, out.desc)
        dev.sync()
        if bound > 1 << 30:
            with pytest.raises(DeviceError, match="max_rows"):
                s.attention(0, b, "f32", out, k, 1, 0.1)


def test_offsets_past_32_bits(dev):
    """The same calls on pages at the start of a small pool and at the end of one of 4.7 GB: the same bytes."""
    rng = np.random.default_rng(19)
    heads, kvh, hd, page, cols = 16, 8, 128, 64, 3
    small = ref.Pool("e4m3", 1, 8, page, kvh, hd)
    n_big = 36000
    codes, scales = hipmem.Buffer(n_big * kvh * small.bytes), hipmem.Buffer(n_big * kvh * 8)
    x = [rng.standard_normal((150, h * hd)) for h in (kvh, kvh, heads)]
    results = []
    for first, n_pages in ((0, 8), (n_big - 8, n_big)):
        table = np.array([[5, 1, 3], [2, 7, 6]], dtype=np.int32) + first
        s = Setup(dev, small, table)
        if first:
            s.pages = dev.kv_pages(codes.ptr.value, codes.nbytes, scales.ptr.value, scales.nbytes, "e4m3", 1, n_pages,
                                   page, kvh, hd)
        b = s.batch([0, 100, 150], [0, 0])
        k, v, q = (Rows(dev, 150, a.shape[1], "bf16", a) for a in x)
        out, ko, vo = Rows(dev, 150, heads * hd, "bf16"), Rows(dev, 150, kvh * hd, "f32"), Rows(dev, 150, kvh * hd, "f32")
        dev.kv_pages_append(s.pages, 0, b, "bf16", k.desc, v.desc)
        s.attention(0, b, "bf16", out, q, heads, 0.1)
        # the second sequence continues the first: its copy of the last page goes to a spare one
        d = [hipmem.Buffer.from_array(np.array(a, dtype=np.int32)) for a in ([0, 0], [first, first + 4], [100])]
        t_out, s_out = hipmem.Buffer.from_array(table * 0), hipmem.Buffer.from_array(table[:, 0] * 0)
        dev.kv_pages_fork(s.pages, t_out.ptr, s_out.ptr, s.d_table.ptr, cols, d[0].ptr, d[1].ptr, d[2].ptr, 1, 2)
        b2 = s.batch([0, 100, 150], [0, 50])
        b2.table = t_out.ptr.value
        dev.kv_pages_read(s.pages, 0, b2, "f32", ko.desc, vo.desc)
        dev.sync()
        results.append((out.get(), ko.get(), vo.get(), t_out.download(np.int32, (2, cols)) - first,
                        s_out.download(np.int32, (2,)) - first))
        assert results[-1][3][1, 1] == 4 and np.array_equal(results[-1][1][100:], results[-1][1][50:100])
    for a, b in zip(*results):
        np.testing.assert_array_equal(a, b)


def test_append_within_its_bounds(dev):
    """Pages outside the pool, positions past max_len, rows past max_rows and n_rows, starts that run backwards:
    nothing is written for them."""
    rng = np.random.default_rng(6)
    pool = ref.Pool("int8", 1, 6, 32, 2, 64)
    table = np.array([[0, -1, 1], [2, 6, 3], [4, 1 << 30, 5]])
    s = Setup(dev, pool, table)
    n = 150
    k, v = Rows(dev, n, 128, "bf16", rng.standard_normal((n, 128))), Rows(dev, n, 128, "bf16",
                                                                           rng.standard_normal((n, 128)))
    kx, vx = k.x.reshape(n, 2, 64), v.x.reshape(n, 2, 64)
    # sequence 0: 70 rows from 20, only 60 of them within max_rows; 1: past max_len from row 36 on; 2: none (backwards)
    dev.kv_pages_append(s.pages, 0, s.batch([0, 70, 130, 90], [20, 50, 0], n_rows=n, max_rows=60, max_len=86), "bf16",
                        k.desc, v.desc)
    touched = ref.append(pool, 0, table, [0, 60], [20], kx, vx)
    touched |= ref.append(pool, 0, table[1:], [0, 36], [50], kx[70:], vx[70:])
    _compare_pools(s.download(), pool, touched, 0)
    # rows that the buffers do not hold
    dev.kv_pages_append(s.pages, 0, s.batch([140, 200], [0], n_rows=n, max_rows=60, max_len=60), "bf16", k.desc, v.desc)
    touched |= ref.append(pool, 0, table, [0, 10], [0], kx[140:], vx[140:])
    _compare_pools(s.download(), pool, touched, 0)
    # the read-back of a page outside the pool
    ko, vo = Rows(dev, 70, 128, "f32"), Rows(dev, 70, 128, "f32")
    dev.kv_pages_read(s.pages, 0, s.batch([0, 70], [0]), "f32", ko.desc, vo.desc)
    dev.sync()
    for got in (ko.get(), vo.get()):
        assert np.isnan(got[32:64]).all() and np.isfinite(got[:32]).all() and np.isfinite(got[64:]).all()


def test_queries_rotate_in_place(dev):
    rng = np.random.default_rng(9)
    pool = ref.Pool("e4m3", 1, 4, 64, 2, 128)
    s = Setup(dev, pool, [[3, 1]])
    cos, sin = _rope(rng, 100, 64)
    dc, ds = hipmem.Buffer.from_array(cos), hipmem.Buffer.from_array(sin)
    k, q = Rows(dev, 7, 256, "f32", rng.standard_normal((7, 256))), Rows(dev, 7, 640, "f32",
                                                                          rng.standard_normal((7, 640)))
    for style in ("neox", "gptj"):
        want = ref.rotate(q.get().reshape(7, 5, 128), np.arange(60, 67), cos, sin, style)
        dev.kv_pages_append(s.pages, 0, s.batch([0, 7], [60]), "f32", k.desc, k.desc,
                            rope=dev.kv_rope(dc.ptr.value, ds.ptr.value, 100, 64, style), q=q.desc, q_out=q.desc,
                            heads=5)
        dev.sync()
        np.testing.assert_array_equal(q.get().reshape(7, 5, 128), want.astype(np.float32))


# ---------------------------------------------------------------------------
# attention

def _filled(rng, kind, layers, n_pages, page, kvh, hd, vd):
    """A pool of normal keys and values of about unit size; zeros in the padded dims."""
    pool = ref.Pool(kind, layers, n_pages, page, kvh, hd, vd)
    spread = 30.0 if kind == "int8" else 100.0
    for which, d in ((0, hd), (1, vd)):
        x = np.zeros((layers, n_pages, kvh, page, ref.padded(d)))
        x[..., :d] = rng.standard_normal((layers, n_pages, kvh, page, d)) * spread
        pool.codes[..., pool.off[which]] = ref.encode(x, kind)
    pool.scales[:] = rng.uniform(0.7, 1.4, pool.scales.shape) / spread
    return pool


def _tolerance(pool, n, dtype, want, mass, size, spread, top):
    d = (ref.padded(pool.hd) / 32 + 8) * 2.0 ** -23 * size + 2.0 ** -22 * spread
    tol = (2 * d + (n / 256 + 16) * 2.0 ** -23) * mass + n * 2.0 ** -36 * top
    if dtype != "f32":
        tol = tol + 2.0 ** -12 * mass + torch.finfo(TORCH[dtype]).eps / 2 * np.abs(want) * 1.01
    return tol + 1e-30


def _check_attention(dev, pool, table, seqs, heads, dtype, window=0, sinks=0, layer=0, size=1.0, seed=0, stride=0,
                     max_rows=None, max_len=None, stream=None):
    rng = np.random.default_rng(seed + 100)
    s = Setup(dev, pool, table)
    rows, pos = [r for r, _ in seqs], [p for _, p in seqs]
    starts = _starts(rows)
    n = int(starts[-1])
    b = s.batch(starts, pos, max_rows=max_rows, max_len=max_len)
    q = Rows(dev, n, heads * pool.hd, dtype, rng.standard_normal((n, heads * pool.hd)) * size,
             heads * pool.hd + stride)
    out = Rows(dev, n, heads * pool.vd, dtype, stride=heads * pool.vd + stride)
    scale = pool.hd ** -0.5
    s.attention(layer, b, dtype, out, q, heads, scale, window, sinks, stream=stream)
    if stream:
        hipmem.check(hipmem.hip().hipStreamSynchronize(stream), "hipStreamSynchronize")
    dev.sync()
    got = out.get().reshape(n, heads, pool.vd)
    want, *sizes = ref.attention(pool, layer, table, starts, pos, q.x.reshape(n, heads, pool.hd), scale,
                                           window, sinks)
    tol = _tolerance(pool, max(r + p for r, p in seqs), dtype, want, *sizes)
    nan = np.isnan(want)
    np.testing.assert_array_equal(np.isnan(got), nan)
    worst = np.max(np.abs(got - want)[~nan] / tol[~nan]) if (~nan).any() else 0
    assert worst <= 1, worst
    return got


ATTENTION = [
    # kind, dtype, heads, kv_heads, hd, vd, page, [(rows, pos)], window, sinks
    ("int8", "f32", 8, 2, 128, 128, 64, [(1, 0), (1, 63), (1, 64), (1, 500)], 0, 0),
    ("e4m3", "f32", 8, 2, 128, 128, 64, [(1, 31), (1, 32), (0, 40), (2, 200)], 0, 0),
    ("int8", "bf16", 32, 4, 128, 128, 32, [(1, 777), (3, 95)], 0, 0),
    ("e4m3", "bf16", 6, 6, 64, 64, 128, [(1, 300), (1, 5)], 0, 0),
    ("int8", "f16", 14, 2, 64, 64, 64, [(1, 129), (5, 61)], 0, 0),
    ("e4m3", "f16", 4, 4, 192, 128, 64, [(1, 200), (4, 0)], 0, 0),
    ("int8", "f32", 2, 1, 256, 256, 256, [(1, 600), (2, 254)], 0, 0),
    ("e4m3", "f32", 3, 1, 80, 80, 32, [(1, 70), (9, 30)], 0, 0),
    ("int8", "f32", 1, 1, 1, 1, 32, [(3, 40)], 0, 0),
    ("int8", "bf16", 40, 2, 64, 64, 64, [(1, 100), (2, 64)], 0, 0),
    # windows: of one key, inside a page, over pages, longer than the sequence; sinks inside and outside of it
    ("int8", "f32", 4, 2, 64, 64, 32, [(1, 100), (40, 0)], 1, 0),
    ("e4m3", "bf16", 4, 2, 128, 128, 64, [(1, 300), (1, 3), (70, 100)], 20, 4),
    ("int8", "f32", 8, 2, 128, 128, 32, [(1, 900), (100, 250)], 100, 33),
    ("int8", "f16", 2, 2, 64, 64, 64, [(1, 90), (33, 31)], 5000, 7),
    ("e4m3", "f32", 2, 1, 64, 64, 64, [(1, 1000), (2, 64)], 64, 200),
    ("int8", "f32", 4, 2, 64, 64, 32, [(1, 100), (40, 0)], 17, 5000),
    # chunks
    ("int8", "f32", 4, 2, 128, 128, 64, [(150, 0), (65, 33)], 0, 0),
    ("e4m3", "bf16", 8, 2, 128, 128, 64, [(200, 100), (0, 0), (17, 250)], 0, 0),
    ("int8", "bf16", 14, 2, 64, 64, 32, [(129, 7)], 0, 0),
    ("e4m3", "f16", 2, 1, 256, 256, 64, [(90, 20)], 0, 0),
    ("int8", "f32", 3, 3, 192, 128, 64, [(100, 1)], 30, 2),
    ("int8", "bf16", 7, 1, 80, 80, 128, [(140, 300), (1, 20)], 128, 4),
    # the largest heads, every column of a tile a query
    ("int8", "f32", 16, 1, 256, 256, 64, [(1, 90), (2, 40)], 0, 0),
    ("e4m3", "bf16", 32, 1, 160, 160, 64, [(1, 200)], 0, 0),
    ("e4m3", "f32", 20, 1, 192, 128, 32, [(2, 70)], 50, 1),
]


# the bound that the call gives for a sequence's rows: what there are, or one
# that thousands of workgroups find nothing behind (the chunk kernel's choice)
BOUNDS = (None, 50000)


@pytest.mark.parametrize("bound", BOUNDS)
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention(dev, case, bound):
    kind, dtype, heads, kvh, hd, vd, page, seqs, window, sinks = ATTENTION[case]
    rng = np.random.default_rng(case)
    cols = max(-(-(r + p) // page) for r, p in seqs) + 1
    pool = _filled(rng, kind, 2, len(seqs) * cols + 2, page, kvh, hd, vd)
    _check_attention(dev, pool, _tables(rng, pool, len(seqs), cols), seqs, heads, dtype, window, sinks, layer=1,
                     size=2.0, seed=case, stride=case % 3 * 4 + case % 2, max_rows=bound)


@pytest.mark.parametrize("bound", BOUNDS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,pos,heads,kvh", [(1, 4500, 4, 1), (1, 9000, 2, 2), (2, 3000, 8, 1)])
def test_long_contexts(dev, dtype, rows, pos, heads, kvh, bound):
    """Lengths whose keys are split over workgroups and joined."""
    rng = np.random.default_rng(pos)
    cols = -(-(rows + pos) // 64)
    pool = _filled(rng, "int8", 1, cols + 2, 64, kvh, 64, 64)
    _check_attention(dev, pool, _tables(rng, pool, 1, cols), [(rows, pos)], heads, dtype, size=3.0, seed=pos,
                     max_rows=bound)


@pytest.mark.parametrize("bound", BOUNDS)
@pytest.mark.parametrize("rows", [1, 70])
def test_scores_far_apart(dev, rows, bound):
    """Scores of hundreds: one key takes everything, the others' weights underflow to zero."""
    rng = np.random.default_rng(1)
    pool = _filled(rng, "int8", 1, 12, 32, 2, 64, 64)
    _check_attention(dev, pool, _tables(rng, pool, 1, 12), [(rows, 250)], 4, "f32", size=150.0, max_rows=bound)


@pytest.mark.parametrize("bound", BOUNDS)
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("rows", [1, 64])
def test_scales_of_every_size(dev, kind, rows, bound):
    """Pages whose value scales differ by powers of ten, and one with a scale of zero (a page of zeros)."""
    rng = np.random.default_rng(12)
    pool = _filled(rng, kind, 1, 9, 64, 2, 128, 128)
    pool.scales[0, :, :, 1] *= 10.0 ** rng.integers(-6, 7, (9, 2))
    table = _tables(rng, pool, 1, 8)
    pool.scales[0, table[0, 2]] = 0
    pool.codes[0, table[0, 2]] = 0
    _check_attention(dev, pool, table, [(rows, 400)], 4, "f32", seed=5, max_rows=bound)


@pytest.mark.parametrize("bound", BOUNDS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_dead_tokens_and_unseen_pages_do_not_matter(dev, dtype, bound):
    """NaN scales, pages outside the pool and garbage codes where no query looks: behind the last token, in
    front of the window, in other layers."""
    rng = np.random.default_rng(13)
    pool = _filled(rng, "e4m3", 2, 20, 32, 2, 64, 64)
    table = _tables(rng, pool, 2, 9)
    seqs, window, sinks = [(1, 200), (40, 160)], 40, 3
    clean = _check_attention(dev, pool, table, seqs, 4, dtype, window, sinks, max_rows=bound)
    # between the sinks and every window: pages 1 and 2 of both sequences, pages 3 and 4 of the first
    for b in range(2):
        pool.scales[0, table[b, 1]] = np.nan
        pool.codes[0, table[b, 2]] = 0x7F
    table[0, 3] = -1
    table[0, 7:] = 77
    pool.scales[1] = np.nan
    # the dead tokens of the last page of sequence 0 (position 200 is token 8 of it): large, but codes
    for which in (0, 1):
        pool.codes[0, table[0, 6]][:, pool.off[which][9:]] = 0x7E
    s = _check_attention(dev, pool, table, seqs, 4, dtype, window, sinks, max_rows=bound)
    np.testing.assert_array_equal(s, clean)


@pytest.mark.parametrize("bound", BOUNDS)
@pytest.mark.parametrize("rows", [3, 80])
@pytest.mark.parametrize("which", [0, 1])
def test_poison_reaches_the_rows_that_see_it_only(dev, rows, which, bound):
    rng = np.random.default_rng(14)
    pool = _filled(rng, "int8", 1, 8, 32, 2, 64, 64)
    table = _tables(rng, pool, 1, 8)
    at = (95 + rows) // 32  # the page that only the last rows see
    pool.scales[0, table[0, at], 1, which] = np.nan
    got = _check_attention(dev, pool, table, [(rows, 96)], 4, "f32", max_rows=bound)
    assert np.isnan(got[-1, 2:]).all() and np.isfinite(got[:, :2]).all()
    if rows > 3:
        assert np.isfinite(got[0]).all()


@pytest.mark.parametrize("bound", BOUNDS)
@pytest.mark.parametrize("rows", [2, 80])
def test_attention_within_its_bounds(dev, rows, bound):
    """A visible page outside the pool gives NaN, rows past max_len NaN, rows past max_rows and rows of no sequence
    keep what they held."""
    rng = np.random.default_rng(15)
    pool = _filled(rng, "int8", 1, 8, 32, 1, 64, 64)
    table = np.array([[0, 1, 2, 3, 4, 5], [6, 9999, 7, 0, 1, 2]])
    got = _check_attention(dev, pool, table, [(rows, 70), (rows, 20)], 2, "f32", max_rows=bound)
    assert np.isfinite(got[:rows]).all() and np.isnan(got[rows + 12:]).all()
    s = Setup(dev, pool, table)
    n = 2 * rows + 5
    q, out = Rows(dev, n, 128, "f32", rng.standard_normal((n, 128))), Rows(dev, n, 128, "f32")
    s.attention(0, s.batch([0, rows], [70], n_rows=n, max_len=71, max_rows=bound), "f32", out, q, 2, 0.1)
    dev.sync()
    got = out.get()
    sentinel = out.host[:4].view(np.float32)[0]
    assert np.isfinite(got[0]).all() and np.isnan(got[1:rows]).all() and (got[rows:] == sentinel).all()
    out = Rows(dev, n, 128, "f32")
    s.attention(0, s.batch([2, 2 + rows], [70], n_rows=n, max_rows=rows - 1), "f32", out, q, 2, 0.1)
    dev.sync()
    got = out.get()
    assert (got[:2] == sentinel).all() and np.isfinite(got[2:1 + rows]).all() and (got[1 + rows:] == sentinel).all()


@pytest.mark.parametrize("bound", BOUNDS)
def test_a_query_that_is_not_finite_gives_nan(dev, bound):
    rng = np.random.default_rng(16)
    pool = _filled(rng, "int8", 1, 4, 64, 1, 64, 64)
    s = Setup(dev, pool, [[0, 1, 2, 3]])
    for rows in (1, 40):
        for bad in (np.nan, np.inf):
            x = rng.standard_normal((rows, 3, 64))
            x[0, 1, 5] = bad
            q, out = Rows(dev, rows, 192, "f32", x), Rows(dev, rows, 192, "f32")
            s.attention(0, s.batch([0, rows], [100], max_rows=bound), "f32", out, q, 3, 0.125)
            dev.sync()
            got = out.get().reshape(rows, 3, 64)
            assert np.isnan(got[0, 1]).all() and np.isfinite(got[:, 0]).all() and np.isfinite(got[:, 2]).all()
            assert np.isfinite(got[1:]).all()


@pytest.mark.parametrize("bound", BOUNDS)
def test_queries_of_zero_and_of_extreme_size(dev, bound):
    rng = np.random.default_rng(17)
    pool = _filled(rng, "e4m3", 1, 4, 64, 1, 64, 64)
    for size in (0.0, 1e-30, 1e30):
        pool.scales[0, :, :, 0] = 1e-30 if size > 1 else 0.01
        for rows in (1, 40):
            _check_attention(dev, pool, np.array([[2, 0, 1, 3]]), [(rows, 90)], 2, "f32", size=size, max_rows=bound)


# ---------------------------------------------------------------------------
# fork

@pytest.mark.parametrize("groups,beams,page,cols,lens", [
    (1, 4, 64, 4, [100]), (3, 8, 32, 3, [95, 64, 1]), (2, 1, 64, 2, [5, 128]), (2, 5, 128, 2, [0, 200]),
    (1, 64, 32, 2, [40]), (2, 3, 32, 2, [64, 63])])
def test_fork(dev, groups, beams, page, cols, lens):
    rng = np.random.default_rng(groups * beams)
    n = groups * beams
    pool = ref.Pool("int8", 3, n * (cols + 1) + 1, page, 2, 64)
    pool.codes[:] = rng.integers(0, 256, pool.codes.shape)
    pool.scales[:] = rng.uniform(0.1, 1, pool.scales.shape)
    ids = rng.permutation(pool.n_pages)
    table, spare = ids[:n * cols].reshape(n, cols).astype(np.int32), ids[n * cols:n * cols + n].astype(np.int32)
    for turn in range(3):
        parents = rng.integers(0, beams, n).astype(np.int32) if turn else np.tile(np.arange(beams, dtype=np.int32),
                                                                                  groups)
        if turn == 2:
            parents[rng.integers(0, n)] = [-1, beams, 1 << 30][beams % 3]
        s = Setup(dev, pool, table)
        d = [hipmem.Buffer.from_array(x) for x in (parents, spare, np.asarray(lens, dtype=np.uint32),
                                                    np.zeros_like(table), np.zeros_like(spare))]
        dev.kv_pages_fork(s.pages, d[3].ptr, d[4].ptr, s.d_table.ptr, cols, d[0].ptr, d[1].ptr, d[2].ptr, groups, beams)
        got = s.download()
        t, sp, copies = ref.fork(table, parents, spare, lens, page, beams)
        np.testing.assert_array_equal(d[3].download(np.int32, table.shape), t)
        np.testing.assert_array_equal(d[4].download(np.int32, spare.shape), sp)
        for src, dst in copies:
            pool.codes[:, dst], pool.scales[:, dst] = pool.codes[:, src], pool.scales[:, src]
        np.testing.assert_array_equal(got.codes, pool.codes)
        np.testing.assert_array_equal(got.scales, pool.scales)


def test_fork_with_pages_outside_the_pool(dev):
    """Such pages are neither read nor written; the tables come out as ever."""
    pool = ref.Pool("e4m3", 1, 4, 32, 1, 64)
    pool.codes[:] = np.random.default_rng(1).integers(0, 256, pool.codes.shape)
    table, spare = np.array([[0, -5], [1, 900]], dtype=np.int32), np.array([2, 1 << 30], dtype=np.int32)
    for parents, lens in (([0, 0], [40]), ([1, 1], [40]), ([0, 0], [10])):
        s = Setup(dev, pool, table)
        d = [hipmem.Buffer.from_array(np.asarray(x)) for x in (np.asarray(parents, np.int32), spare,
                                                               np.asarray(lens, np.uint32), table * 0, spare * 0)]
        dev.kv_pages_fork(s.pages, d[3].ptr, d[4].ptr, s.d_table.ptr, 2, d[0].ptr, d[1].ptr, d[2].ptr, 1, 2)
        got = s.download()
        t, sp, copies = ref.fork(table, np.asarray(parents), spare, lens, 32, 2)
        np.testing.assert_array_equal(d[3].download(np.int32, table.shape), t)
        np.testing.assert_array_equal(d[4].download(np.int32, spare.shape), sp)
        np.testing.assert_array_equal(got.codes, pool.codes)


# ---------------------------------------------------------------------------
# together, on other streams, in graphs, refused

def _beam_decode(dev, stream=None):
    """Beams that share a prompt: append, attend, fork, append, ...; every step against dense 64-bit states that are
    copied with their parents."""
    rng = np.random.default_rng(21)
    beams, kvh, heads, hd, page, cols, layers = 4, 2, 4, 64, 32, 6, 2
    pool = ref.Pool("int8", layers, 40, page, kvh, hd)
    prompt = 75
    shared = [30, 31]
    table = np.full((beams, cols), -1, dtype=np.int32)
    table[:, :2] = shared
    table[:, 2:] = np.arange(beams * 4).reshape(beams, 4)
    spare = np.arange(20, 24, dtype=np.int32)
    s = Setup(dev, pool, table)
    cos, sin = _rope(rng, 200, 32)
    dc, ds = hipmem.Buffer.from_array(cos), hipmem.Buffer.from_array(sin)
    rope = dev.kv_rope(dc.ptr.value, ds.ptr.value, 200, 32)
    d_spare = [hipmem.Buffer.from_array(spare), hipmem.Buffer.from_array(spare * 0)]
    d_table = [s.d_table, hipmem.Buffer.from_array(table * 0)]
    keep = []
    length = 0
    for step in range(30):
        rows = prompt if step == 0 else 1
        who = [0] if step == 0 else list(range(beams))
        n = rows * len(who)
        starts = _starts([rows] * len(who))
        s.d_table = d_table[0]
        s.table = table
        b = s.batch(starts, [length] * len(who))
        outs = []
        for layer in range(layers):
            k, v, q = (Rows(dev, n, h * hd, "f32", rng.standard_normal((n, h * hd))) for h in (kvh, kvh, heads))
            out = Rows(dev, n, heads * hd, "f32")
            dev.kv_pages_append(s.pages, layer, b, "f32", k.desc, v.desc, rope=rope, q=q.desc, q_out=q.desc,
                                heads=heads, stream=stream)
            s.attention(layer, b, "f32", out, q, heads, 0.125, stream=stream)
            ref.append(pool, layer, table, starts, [length] * len(who), k.x.reshape(n, kvh, hd),
                       v.x.reshape(n, kvh, hd), (cos, sin, "neox"))
            want = ref.attention(pool, layer, table, starts, [length] * len(who), ref.rotate(
                q.x.reshape(n, heads, hd), np.concatenate([length + np.arange(rows)] * len(who)), cos, sin,
                "neox").astype(np.float32), 0.125)
            outs.append((out, want))
            keep += [k, v, q, out]
        length += rows
        hipmem.synchronize()
        for out, (want, *sizes) in outs:
            got = out.get().reshape(n, heads, hd)
            assert (np.abs(got - want) <= _tolerance(pool, length, "f32", want, *sizes)).all(), step
        # the first step's page goes to every beam
        parents = np.zeros(beams, dtype=np.int32) if step == 0 else rng.integers(0, beams, beams).astype(np.int32)
        d_par, d_len = hipmem.Buffer.from_array(parents), hipmem.Buffer.from_array(np.array([length], dtype=np.uint32))
        dev.kv_pages_fork(s.pages, d_table[1].ptr, d_spare[1].ptr, d_table[0].ptr, cols, d_par.ptr, d_spare[0].ptr,
                          d_len.ptr, 1, beams, stream=stream)
        hipmem.synchronize()
        table, spare, copies = ref.fork(table, parents, spare, [length], page, beams)
        for src, dst in copies:
            pool.codes[:, dst], pool.scales[:, dst] = pool.codes[:, src], pool.scales[:, src]
        np.testing.assert_array_equal(d_table[1].download(np.int32, table.shape), table)
        np.testing.assert_array_equal(d_spare[1].download(np.int32, spare.shape), spare)
        d_table.reverse()
        d_spare.reverse()


def test_beams_decoded_together(dev):
    _beam_decode(dev)


def test_beams_decoded_on_another_stream(dev):
    lib = hipmem.hip()
    stream = ctypes.c_void_p()
    assert lib.hipStreamCreateWithFlags(ctypes.byref(stream), 1) == 0
    try:
        _beam_decode(dev, stream.value)
    finally:
        lib.hipStreamDestroy(stream)


def test_captured_calls_replay(dev):
    """A decode step of two sequences captured once and replayed with new rows, new positions and eager calls of
    other shapes in between: each replay equals the eager call on the same state."""
    lib = hipmem.hip()
    P = ctypes.c_void_p
    for name, args in {"hipStreamBeginCapture": [P, ctypes.c_int], "hipStreamEndCapture": [P, ctypes.POINTER(P)],
                       "hipGraphInstantiate": [ctypes.POINTER(P), P, P, P, ctypes.c_size_t],
                       "hipGraphLaunch": [P, P], "hipGraphExecDestroy": [P], "hipGraphDestroy": [P]}.items():
        getattr(lib, name).argtypes = args
        getattr(lib, name).restype = ctypes.c_int
    rng = np.random.default_rng(31)
    heads, kvh, hd = 8, 2, 128
    pool = _filled(rng, "e4m3", 1, 60, 64, kvh, hd, hd)
    table = _tables(rng, pool, 2, 30)
    s, eager = Setup(dev, pool, table), Setup(dev, pool, table)
    k, v, q = (Rows(dev, 2, h * hd, "bf16", rng.standard_normal((2, h * hd))) for h in (kvh, kvh, heads))
    out, out2 = Rows(dev, 2, heads * hd, "bf16"), Rows(dev, 2, heads * hd, "bf16")
    pos = np.array([900, 33], dtype=np.uint32)
    d_pos = hipmem.Buffer.from_array(pos)
    starts = hipmem.Buffer.from_array(np.array([0, 1, 2], dtype=np.uint32))
    b, b2 = (dev.kv_batch(x.d_table.ptr.value, 30, starts.ptr.value, d_pos.ptr.value, 2, 2, 1, 1800) for x in (s, eager))
    need = dev.kv_pages_attention_workspace(s.pages, b, heads, "bf16")
    ws = hipmem.Buffer(max(need, 1))
    stream, graph, exe = P(), P(), P()
    assert lib.hipStreamCreateWithFlags(ctypes.byref(stream), 1) == 0
    try:
        hipmem.synchronize()
        assert lib.hipStreamBeginCapture(stream, 0) == 0
        dev.kv_pages_append(s.pages, 0, b, "bf16", k.desc, v.desc, stream=stream.value)
        s.attention(0, b, "bf16", out, q, heads, 0.09, stream=stream.value, ws=ws)
        assert lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert lib.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
        for replay in range(4):
            for r in (k, v, q):
                r.host[:] = Rows(dev, 2, r.width, "bf16", rng.standard_normal((2, r.width))).host
                r.buf.upload(r.host)
            pos = pos + np.uint32(replay * 37)
            d_pos.upload(pos)
            hipmem.synchronize()
            assert lib.hipGraphLaunch(exe, stream) == 0
            hipmem.check(lib.hipStreamSynchronize(stream), "hipStreamSynchronize")
            dev.kv_pages_append(eager.pages, 0, b2, "bf16", k.desc, v.desc)
            eager.attention(0, b2, "bf16", out2, q, heads, 0.09)
            dev.sync()
            np.testing.assert_array_equal(out.get(), out2.get())
            np.testing.assert_array_equal(s.download().codes, eager.download().codes)
    finally:
        if exe.value:
            lib.hipGraphExecDestroy(exe)
        if graph.value:
            lib.hipGraphDestroy(graph)
        lib.hipStreamDestroy(stream)


def test_refusals(dev):
    """Every one is an error before anything is launched; the context works on."""
    pool = ref.Pool("int8", 2, 4, 32, 2, 64)
    s = Setup(dev, pool, [[0, 1]])
    n = 4
    k, q, out = Rows(dev, n, 128, "f32", np.ones((n, 128))), Rows(dev, n, 256, "f32", np.ones((n, 256))), \
        Rows(dev, n, 256, "f32")
    b = s.batch([0, n], [30])
    cos = hipmem.Buffer.from_array(np.ones((40, 32), dtype=np.float32))

    def changed(desc, **over):
        new = type(desc)()
        ctypes.memmove(ctypes.byref(new), ctypes.byref(desc), ctypes.sizeof(desc))
        for name, value in over.items():
            setattr(new, name, value)
        return new

    def append(pages=s.pages, layer=0, batch=b, dtype="f32", kd=k.desc, vd=k.desc, **more):
        dev.kv_pages_append(pages, layer, batch, dtype, kd, vd, **more)

    def attend(pages=s.pages, layer=0, batch=b, dtype="f32", o=out.desc, qd=q.desc, heads=4, **more):
        dev.kv_pages_attention(pages, layer, batch, dtype, o, qd, heads, 0.1, 0, 0, **more)

    refused = [
        lambda: append(pages=changed(s.pages, kind=3)), lambda: append(pages=changed(s.pages, page_tokens=33)),
        lambda: append(pages=changed(s.pages, codes=None)), lambda: append(pages=changed(s.pages, scales=None)),
        lambda: append(pages=changed(s.pages, codes=s.pages.codes + 8)),
        lambda: append(pages=changed(s.pages, codes_bytes=s.pages.codes_bytes - 1)),
        lambda: append(pages=changed(s.pages, scales_bytes=s.pages.scales_bytes - 1)),
        lambda: append(pages=changed(s.pages, n_pages=5)), lambda: append(pages=changed(s.pages, layers=3)),
        lambda: append(layer=2), lambda: append(pages=changed(s.pages, head_dim=300)),
        lambda: append(batch=changed(b, table=None)), lambda: append(batch=changed(b, starts=None)),
        lambda: append(batch=changed(b, pos=None)), lambda: append(batch=changed(b, max_len=65)),
        lambda: append(batch=changed(b, n_rows=5)), lambda: append(batch=changed(b, max_len=0xFFFFFFFF)),
        lambda: append(kd=None), lambda: append(vd=None), lambda: append(kd=changed(k.desc, data=None)),
        lambda: append(kd=changed(k.desc, bytes=k.desc.bytes - 1)), lambda: append(kd=changed(k.desc, stride=127)),
        lambda: append(kd=changed(k.desc, data=k.desc.data + 2)),
        lambda: append(vd=changed(k.desc, stride=1 << 62)),
        lambda: append(q=q.desc), lambda: append(q=q.desc, q_out=out.desc, heads=0),
        lambda: append(q=q.desc, q_out=out.desc, heads=5),
        lambda: append(rope=dev.kv_rope(cos.ptr.value, cos.ptr.value, 33, 32)),
        lambda: append(rope=dev.kv_rope(None, cos.ptr.value, 40, 32)),
        lambda: append(rope=dev.kv_rope(cos.ptr.value, cos.ptr.value, 40, 33)),
        lambda: append(rope=changed(dev.kv_rope(cos.ptr.value, cos.ptr.value, 40, 32), style=2)),
        lambda: attend(heads=3), lambda: attend(heads=0), lambda: attend(heads=6),
        lambda: attend(o=changed(out.desc, bytes=out.desc.bytes - 4)), lambda: attend(qd=None),
        lambda: attend(window=1 << 31), lambda: attend(pages=changed(s.pages, v_head_dim=0)),
        lambda: dev.kv_pages_read(s.pages, 0, b, "f32", changed(k.desc, bytes=8), k.desc),
        lambda: dev.kv_pages_fork(s.pages, 1, 2, 3, 0, 4, 5, 6, 1, 2),
        lambda: dev.kv_pages_fork(s.pages, 1, 2, 3, 2, 4, 5, 6, 1, 65),
        lambda: dev.kv_pages_fork(s.pages, 1, 2, 1, 2, 4, 5, 6, 1, 2),
        lambda: dev.kv_pages_fork(s.pages, 1, 2, 3, 2, 4, 2, 6, 1, 2),
        lambda: dev.kv_pages_fork(s.pages, 1, 2, 3, 2, None, 5, 6, 1, 2),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(DeviceError) as e:
            call()
        assert e.value.status == abi.INVALID_ARGUMENT and str(e.value), i
    with pytest.raises(DeviceError) as e:
        append(pages=changed(s.pages, v_head_dim=128, n_pages=1, layers=1))
    assert e.value.status == abi.UNSUPPORTED
    long = s.batch([0, n], [30], max_len=64)
    need = dev.kv_pages_attention_workspace(s.pages, long, 4, "f32")
    if need:
        with pytest.raises(DeviceError, match="workspace"):
            attend(batch=long)
    # no rows, no sequences: nothing to do
    append(batch=changed(b, n_rows=0))
    append(batch=changed(b, n_seqs=0))
    attend(batch=changed(b, max_rows=0))
    got = s.download()
    np.testing.assert_array_equal(got.codes, pool.codes)


# ---------------------------------------------------------------------------
# value scales of any size next to each other

def _check_scales(dev, pool, table, seqs, heads, dtype, bound, seed=3):
    """Attention against 64 bits, relative to the outputs themselves however small they are. On top of what the head
    of this file adds up: the logarithm of a value scale is off by 2^-23 of itself, and as much again for each of the
    two sums it goes into, a weight then by less than 2^-21 max |log2 scale|; of 16-bit rows a granule's part of the
    denominator comes from its f16 weights where its scale is at most 2^6 below the largest of those before it, which
    is n * 2^-31 of the whole."""
    rng = np.random.default_rng(seed)
    s = Setup(dev, pool, table)
    rows, pos = [r for r, _ in seqs], [p for _, p in seqs]
    starts, n = _starts(rows), sum(rows)
    keys = max(r + p for r, p in seqs)
    q = Rows(dev, n, heads * pool.hd, dtype, rng.standard_normal((n, heads * pool.hd)))
    out = Rows(dev, n, heads * pool.vd, dtype)
    scale = pool.hd ** -0.5
    s.attention(0, s.batch(starts, pos, max_rows=bound), dtype, out, q, heads, scale)
    dev.sync()
    got = out.get().reshape(n, heads, pool.vd)
    want, mass, size, spread, top = ref.attention(pool, 0, table, starts, pos, q.x.reshape(n, heads, pool.hd), scale)
    vs = pool.scales[0, :, :, 1]
    bias = np.abs(np.log2(vs[vs > 0])).max()
    d = (ref.padded(pool.hd) / 32 + 8) * 2.0 ** -23 * size + 2.0 ** -22 * spread + 2.0 ** -21 * bias
    tol = (2 * d + (keys / 256 + 16) * 2.0 ** -23) * mass + keys * 2.0 ** -36 * top + 2.0 ** -149
    if dtype != "f32":
        info = torch.finfo(TORCH[dtype])
        tol += 2.0 ** -12 * mass + (keys * 2.0 ** -31 + info.eps / 2 * 1.01) * np.abs(want) + info.smallest_normal * info.eps / 2
    worst = np.max(np.abs(got - want) / tol)
    assert worst <= 1, worst


# rows and position of one sequence: one workgroup a tile, a chunk, keys split over workgroups
REACHES = [(1, 400), (64, 400), (1, 4500)]


def _scaled(kind, pos, first, rest, page=64):
    rng = np.random.default_rng(pos)
    cols = -(-(pos + 64) // page)
    pool = _filled(rng, kind, 1, cols, page, 1, 64, 64)
    table = _tables(rng, pool, 1, cols)
    pool.scales[0, :, :, 1] *= np.where(np.arange(cols) == table[0, 0], first, rest)[:, None]
    return pool, table


@pytest.mark.parametrize("bound", BOUNDS)
@pytest.mark.parametrize("reach", REACHES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("first,rest", [(1e-35, 1.0), (1e-32, 1.0), (1.0, 1e-35), (1e-35, 1e-35), (1e-35, 1e30),
                                        (1e30, 1e-35), (1e-20, 1.0)])
def test_value_scales_at_the_ends_of_the_range(dev, first, rest, dtype, reach, bound):
    pool, table = _scaled("int8", reach[1], first, rest)
    _check_scales(dev, pool, table, [reach], 4, dtype, bound)


@pytest.mark.parametrize("bound", BOUNDS)
@pytest.mark.parametrize("reach", REACHES)
@pytest.mark.parametrize("rest", [1.0, 1e-33])
def test_a_page_of_zeros_in_front(dev, rest, reach, bound):
    pool, table = _scaled("e4m3", reach[1], rest, rest)
    pool.scales[0, table[0, 0]] = 0
    pool.codes[0, table[0, 0]] = 0
    _check_scales(dev, pool, table, [reach], 4, "f32", bound)


@pytest.mark.parametrize("bound", BOUNDS)
@pytest.mark.parametrize("reach", REACHES)
@pytest.mark.parametrize("kind,dtype", [("int8", "bf16"), ("e4m3", "f16"), ("int8", "f32")])
@pytest.mark.parametrize("apart", [7, 20, 33, 43])
@pytest.mark.parametrize("large_first", [True, False])
def test_value_scales_far_apart(dev, large_first, apart, kind, dtype, reach, bound):
    """One page of large values and the others 2^-apart of it, in front of them or behind."""
    low = 2.0 ** -apart
    pool, table = _scaled(kind, reach[1], 1.0 if large_first else low, low)
    if not large_first:
        pool.scales[0, table[0, reach[1] // 64 - 1], :, 1] /= np.float32(low)
    _check_scales(dev, pool, table, [reach], 4, dtype, bound)


@pytest.mark.parametrize("bound", BOUNDS)
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 64])
def test_scales_of_every_size_in_16_bits(dev, kind, dtype, rows, bound):
    rng = np.random.default_rng(12)
    pool = _filled(rng, kind, 1, 9, 64, 2, 128, 128)
    pool.scales[0, :, :, 1] *= 10.0 ** rng.integers(-8 if dtype == "f16" else -6, 1 if dtype == "f16" else 7, (9, 2))
    table = _tables(rng, pool, 1, 8)
    pool.scales[0, table[0, 2]] = 0
    pool.codes[0, table[0, 2]] = 0
    _check_scales(dev, pool, table, [(rows, 400)], 4, dtype, bound)


def test_the_last_positions(dev):
    """Positions up to the most that a batch may have, rows that run past them, pages named behind them: what lies
    there is as it was, and the rows' attention is that of the same page at the start of a sequence."""
    rng = np.random.default_rng(20)
    most, page, n = (1 << 31) - 257, 256, 700
    pool = ref.Pool("int8", 1, 8, page, 1, 64)
    table = np.full((1, most // page + 65), 5, dtype=np.int32)  # (page 5: where no row belongs)
    table[0, :most // page] = -1
    pos = most - 100
    table[0, pos // page] = 2
    s = Setup(dev, pool, table)
    k, v = (Rows(dev, n, 64, "f32", rng.standard_normal((n, 64))) for _ in range(2))
    b = s.batch([0, n], [pos], max_len=most)
    dev.kv_pages_append(s.pages, 0, b, "f32", k.desc, v.desc)
    touched = ref.append(pool, 0, table, [0, 100], [pos], k.x.reshape(n, 1, 64), v.x.reshape(n, 1, 64))
    _compare_pools(s.download(), pool, touched, 0)
    ko, vo = Rows(dev, n, 64, "f32"), Rows(dev, n, 64, "f32")
    dev.kv_pages_read(s.pages, 0, b, "f32", ko.desc, vo.desc)
    q, far = Rows(dev, n, 128, "f32", rng.standard_normal((n, 128))), Rows(dev, n, 128, "f32")
    s.attention(0, b, "f32", far, q, 2, 0.1, window=64)
    dev.sync()
    wk, wv = ref.sequence(pool, 0, [2], page)
    in_page = pos % page
    for got, want in ((ko.get(), wk), (vo.get(), wv)):
        np.testing.assert_array_equal(got[:100], want[0, in_page:in_page + 100].astype(np.float32))
        assert (got[100:] == np.full(4, 0x77, np.uint8).view(np.float32)).all()
    near_s = Setup(dev, pool, [[2]])
    near = Rows(dev, n, 128, "f32")
    near_s.attention(0, near_s.batch([0, n], [in_page], max_len=in_page + 100), "f32", near, q, 2, 0.1, window=64)
    dev.sync()
    far, near = far.get(), near.get()
    assert np.isfinite(far[:100]).all() and np.isnan(far[100:]).all()
    np.testing.assert_array_equal(far, near)


@pytest.mark.parametrize("parents,copier,spare", [([0, 0], 1, [2, 3]), ([1, 1], 1, [2, 3]), ([1, 1, 1], 2, [4, 2, 3])])
def test_a_copy_of_a_page_outside_the_pool_is_nan(dev, parents, copier, spare):
    """The child's copy has nothing in it that could pass for the parent's tokens; the codes stay."""
    beams = len(parents)
    pool = ref.Pool("int8", 2, 6, 32, 3, 64)
    pool.codes[:] = np.random.default_rng(3).integers(0, 256, pool.codes.shape)
    table = np.array([[0, -5], [1, 900], [0, 5]], dtype=np.int32)[:beams]
    spare = np.array(spare, dtype=np.int32)
    s = Setup(dev, pool, table)
    d = [hipmem.Buffer.from_array(np.asarray(x)) for x in (np.asarray(parents, np.int32), spare, np.array([40], np.uint32),
                                                           table * 0, spare * 0)]
    dev.kv_pages_fork(s.pages, d[3].ptr, d[4].ptr, s.d_table.ptr, 2, d[0].ptr, d[1].ptr, d[2].ptr, 1, beams)
    got = s.download()
    t, sp, copies = ref.fork(table, np.asarray(parents), spare, [40], 32, beams)
    np.testing.assert_array_equal(d[3].download(np.int32, table.shape), t)
    np.testing.assert_array_equal(d[4].download(np.int32, spare.shape), sp)
    np.testing.assert_array_equal(got.codes, pool.codes)
    assert t[copier, 1] == spare[copier]
    for _, dst in copies:
        pool.scales[:, dst] = np.nan
    np.testing.assert_array_equal(got.scales, pool.scales)
    s.table = t
    s.d_table = hipmem.Buffer.from_array(t)
    q, out = Rows(dev, beams, 192, "f32", np.ones((beams, 192))), Rows(dev, beams, 192, "f32")
    s.attention(0, s.batch(np.arange(beams + 1), [39] * beams), "f32", out, q, 3, 0.1)
    dev.sync()
    out = out.get()
    assert np.isnan(out[[c for c in range(beams) if parents[c] < 2]]).all()


@pytest.mark.parametrize("heads,hd,half,style", [(48, 256, 128, "neox"), (33, 100, 20, "gptj"), (40, 128, 0, "neox")])
def test_many_query_heads_of_few_rows(dev, heads, hd, half, style):
    """A row's heads over several workgroups, and over one that takes more than its threads hold at once."""
    rng = np.random.default_rng(heads)
    pool = ref.Pool("int8", 1, 2, 64, 1, hd)
    s = Setup(dev, pool, [[1, 0]])
    cos, sin = _rope(rng, 64, max(half, 1))
    dc, ds = hipmem.Buffer.from_array(cos), hipmem.Buffer.from_array(sin)
    for rows in (1, 3):
        k = Rows(dev, rows, hd, "f32", rng.standard_normal((rows, hd)))
        q, q_out = Rows(dev, rows, heads * hd, "f32", rng.standard_normal((rows, heads * hd))), Rows(dev, rows, heads * hd, "f32")
        dev.kv_pages_append(s.pages, 0, s.batch([0, rows], [60 - rows]), "f32", k.desc, k.desc,
                            rope=dev.kv_rope(dc.ptr.value, ds.ptr.value, 64, half, style), q=q.desc, q_out=q_out.desc,
                            heads=heads)
        dev.sync()
        want = q.x.reshape(rows, heads, hd).astype(np.float64)
        if half:
            want = ref.rotate(want, np.arange(60 - rows, 60), cos, sin, style)
        np.testing.assert_array_equal(q_out.get().reshape(rows, heads, hd), want.astype(np.float32))


@pytest.mark.parametrize("bound", BOUNDS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e5, 1e7, 1e9, 1e12, 1e20])
@pytest.mark.parametrize("reach", REACHES)
def test_scores_past_the_exponents_steps(dev, reach, size, dtype, bound):
    """Scores so large that f32 holds them in steps of a weight's whole range and more: where the largest lies further
    ahead of the others than they are off (d of the head of this file, and 200 for weights that vanish), its value
    comes out; elsewhere a mean of values."""
    rng = np.random.default_rng(22)
    rows, pos = reach
    cols = -(-(rows + pos) // 64)
    pool = _filled(rng, "int8", 1, cols, 64, 1, 64, 64)
    table = _tables(rng, pool, 1, cols)
    s = Setup(dev, pool, table)
    q = Rows(dev, rows, 256, dtype, rng.standard_normal((rows, 256)) * size)
    out = Rows(dev, rows, 256, dtype)
    s.attention(0, s.batch([0, rows], [pos], max_rows=bound), dtype, out, q, 4, 0.125)
    dev.sync()
    got = out.get().reshape(rows, 4, 64)
    k, v = (x[0] for x in ref.sequence(pool, 0, table[0], rows + pos))
    eps = 2.0 ** -20 if dtype == "f32" else 2.0 ** -8
    alone = 0
    for i in range(rows):
        n = pos + i + 1
        scores = q.x[i].reshape(4, 64).astype(np.float64) @ k[:n].T * 0.125
        off = 10 * 2.0 ** -23 * (np.abs(q.x[i].reshape(4, 64)).astype(np.float64) @ np.abs(k[:n]).T).max(1) * 0.125
        best, second = scores.argmax(1), np.sort(scores, 1)[:, -2]
        for h in range(4):
            assert np.isfinite(got[i, h]).all() and (np.abs(got[i, h]) <= np.abs(v[:n]).max(0) * (1 + eps)).all()
            if scores[h].max() - second[h] > 2 * off[h] + 200:
                alone += 1
                assert (np.abs(got[i, h] - v[best[h]]) <= eps * np.abs(v[best[h]]) + 1e-30).all()
    assert alone >= 2 * rows
