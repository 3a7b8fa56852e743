"""A model's cache in pages of 8-bit codes (ditch_hip_kv_cache_create_pages):
the cached forward and generation against a 64-bit forward whose keys and
values go through the plain pages of pages_ref.py.

Tolerance: the products behind a key or value are off by about 2^-18 of their
terms' sizes, some 2^-10 of a code's step, so about one code in a thousand
comes out a step away from the plain form's. A step is 1/127 of the page's
largest value (int8: about 3.5 / 127 = 0.03 of a value's usual size) or up to
1/8 of the value (e4m3). Worst off is a row with one key: one of a head's hd
output coordinates moves by a step, the head's output by 0.03 / sqrt(64) =
0.4 % (int8) or 0.125 / sqrt(128) = 1.1 % (e4m3) of its size, and the logits by
no larger part of theirs, as the residual holds the embedding and the other
heads too. Logits are held to 4e-3 and 1.2e-2 of the largest."""
import numpy as np
import pytest
import torch

import model_gen as mg
import pages_ref as ref
from ditch_amd import abi, hipmem
from ditch_amd.hip import DeviceError, Model

pytestmark = pytest.mark.gpu

TOLERANCE = {"int8": 4e-3, "e4m3": 1.2e-2}


class Plain:
    """The dense forward in 64 bits, keys and values through pools of pages."""

    def __init__(self, dev, spec, prompts, max_len, kind, page, window, sinks):
        c = self.c = spec.config
        self.w = {k: dev.dequant(w).astype(np.float64) if k[1] not in abi.VECTOR_SLOTS else
                  np.asarray(dev.dequant(w), dtype=np.float64).reshape(-1) for k, w in spec.tensors.items()}
        self.kind, self.window, self.sinks = kind, window, sinks
        cols = -(-max_len // page)
        self.table = np.arange(prompts * cols).reshape(prompts, cols)
        self.pool = ref.Pool(kind, c["layers"], prompts * cols, page, c["kv_heads"], c["head_dim"])
        half = c["rotary_dim"] // 2
        angle = np.arange(c["rope_len"])[:, None] * np.float64(np.float32(c["rope_theta"])) ** (-2.0 * np.arange(half) / c["rotary_dim"])
        self.rope = (np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32), "neox")

    def get(self, slot, layer=-1):
        return self.w.get((layer, abi.SLOT[slot], -1))

    def norm(self, x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.c["rms_eps"]) * w

    def forward(self, tokens, starts, pos):
        """tokens of every prompt's rows, one prompt after the other; logits of all rows."""
        c, hd = self.c, self.c["head_dim"]
        x = self.get("EMBED")[tokens]
        n = len(tokens)
        at = np.concatenate([pos[b] + np.arange(starts[b + 1] - starts[b]) for b in range(len(pos))])
        for li in range(c["layers"]):
            h = self.norm(x, self.get("ATTN_NORM", li))
            q, k, v = ((h @ self.get(s, li).T + (self.get(s + "_BIAS", li) if c["qkv_bias"] else 0)).reshape(n, -1, hd)
                       for s in "QKV")
            if c["qk_norm"]:
                q, k = self.norm(q, self.get("Q_NORM", li)), self.norm(k, self.get("K_NORM", li))
            ref.append(self.pool, li, self.table, starts, pos, k, v, self.rope)
            o = ref.attention(self.pool, li, self.table, starts, pos, ref.rotate(q, at, *self.rope), c["attn_scale"],
                              self.window, self.sinks)[0]
            x = x + o.reshape(n, -1) @ self.get("O", li).T
            h = self.norm(x, self.get("FFN_NORM", li))
            g = h @ self.get("GATE", li).T
            x = x + (g / (1 + np.exp(-g)) * (h @ self.get("UP", li).T)) @ self.get("DOWN", li).T
        return self.norm(x, self.get("FINAL_NORM")) @ self.get("EMBED").T


def _cached(dev, m, cache, tokens, rows, logit_rows, vocab):
    bt, br = hipmem.Buffer.from_array(np.asarray(tokens, np.uint32)), hipmem.Buffer.from_array(np.asarray(rows, np.uint32))
    bl, bo = hipmem.Buffer.from_array(np.asarray(logit_rows, np.uint64)), hipmem.Buffer(len(logit_rows) * vocab * 4)
    dev.check(dev.lib.ditch_hip_forward_cached(m.h, cache, bt.ptr, br.ptr, len(tokens), bl.ptr, len(logit_rows), bo.ptr,
                                               bo.nbytes))
    dev.sync()
    return bo.download(np.float32, (len(logit_rows), vocab))


CASES = [
    # kind, page, window, sinks, the model
    ("int8", 64, 0, 0, dict(hidden=256, heads=4, kv_heads=2, head_dim=64, qkv_bias=True)),
    ("e4m3", 32, 0, 0, dict(hidden=128, heads=4, kv_heads=1, head_dim=128, qk_norm=True)),
    ("int8", 32, 24, 3, dict(hidden=128, heads=2, kv_heads=2, head_dim=64)),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_cached_forward_over_pages(dev, case):
    kind, page, window, sinks, shape = CASES[case]
    spec = mg.dense("bf16", inter=256, layers=2, vocab=300, seed=case, **shape)
    m, vocab, lens = Model(dev, spec), 300, [70, 1, 33]
    cache = m.kv_cache_pages(3, 80, kind, page, window, sinks)
    plain = Plain(dev, spec, 3, 80, kind, page, window, sinks)
    rng = np.random.default_rng(case)
    try:
        pos = [0, 0, 0]
        # the prompts, a row of each, and two rows of the first with one of the last
        for rows in (lens, [1, 1, 1], [2, 0, 1], [1, 1, 1]):
            starts = np.concatenate([[0], np.cumsum(rows)])
            tokens = rng.integers(0, vocab, starts[-1])
            pairs = [(b, pos[b] + i) for b in range(3) for i in range(rows[b])]
            got = _cached(dev, m, cache, tokens, pairs, np.arange(len(tokens)), vocab)
            want = plain.forward(tokens, starts, pos)
            assert np.abs(got - want).max() <= TOLERANCE[kind] * np.abs(want).max()
            pos = [p + r for p, r in zip(pos, rows)]
    finally:
        m.kv_cache_free(cache)
        m.free()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_generation_past_1024_positions(dev, kind):
    """Greedy tokens of generate() over pages, each the plain forward's choice (or within the tolerance of it)."""
    spec = mg.dense("bf16", hidden=128, inter=128, heads=2, kv_heads=1, head_dim=64, layers=1, vocab=200, seed=5)
    spec.config["rope_len"] = 2048
    m = Model(dev, spec)
    with pytest.raises(DeviceError):
        m.kv_cache(2, 1300)  # the f32 cache ends at 1024
    cache = m.kv_cache_pages(2, 1300, kind)
    plain = Plain(dev, spec, 2, 1300, kind, 64, 0, 0)
    rng = np.random.default_rng(1)
    prompts = [list(rng.integers(0, 200, 1100)), list(rng.integers(0, 200, 40))]
    try:
        out, first = m.generate(cache, prompts, 4, first_logits=True)
        starts, pos = np.array([0, 1100, 1140]), [0, 0]
        logits = plain.forward(np.concatenate(prompts), starts, pos)[starts[1:] - 1]
        assert np.abs(first - logits).max() <= TOLERANCE[kind] * np.abs(logits).max()
        pos = [1100, 40]
        for step in range(4):
            for b in range(2):
                assert logits[b].max() - logits[b][out[b][step]] <= 2 * TOLERANCE[kind] * np.abs(logits[b]).max()
            logits = plain.forward(np.array([out[0][step], out[1][step]]), np.array([0, 1, 2]), pos)
            pos = [p + 1 for p in pos]
    finally:
        m.kv_cache_free(cache)
        m.free()


def test_rows_out_of_order_give_nan(dev):
    """A prompt whose rows do not follow each other; the other prompts are as ever."""
    spec = mg.dense("bf16", hidden=128, inter=128, heads=2, kv_heads=1, head_dim=64, layers=1, vocab=100, seed=6)
    m = Model(dev, spec)
    a, b = m.kv_cache_pages(2, 50), m.kv_cache_pages(2, 50)
    tokens = np.random.default_rng(2).integers(0, 100, 9)
    good = [(0, p) for p in range(5)] + [(1, p) for p in range(4)]
    bad = good[:5] + [(1, 0), (1, 2), (1, 1), (1, 3)]
    try:
        want = _cached(dev, m, a, tokens, good, np.arange(9), 100)
        got = _cached(dev, m, b, tokens, bad, np.arange(9), 100)
        np.testing.assert_array_equal(got[:5], want[:5])
        assert np.isnan(got[5:]).all() and np.isfinite(want).all()
    finally:
        m.kv_cache_free(a)
        m.kv_cache_free(b)
        m.free()


def test_refused_caches(dev):
    spec = mg.dense("bf16", hidden=128, inter=128, heads=2, kv_heads=1, head_dim=64, layers=1, vocab=100, seed=7)
    m, latent = Model(dev, spec), Model(dev, mg.mla("bf16", heads=2, layers=1, vocab=100))
    try:
        for args in ((0, 10), (1, 0), (1, spec.config["rope_len"] + 1), (1, 10, "int8", 16), (1, 10, "int8", 0),
                     (1, 10, "int8", 64, 1 << 31), (1 << 31, 100)):
            with pytest.raises(DeviceError):
                m.kv_cache_pages(*args)
        assert not dev.lib.ditch_hip_kv_cache_create_pages(m.h, 1, 10, 5, 64, 0, 0)
        assert not dev.lib.ditch_hip_kv_cache_create_pages(None, 1, 10, 0, 64, 0, 0)
        with pytest.raises(DeviceError, match="latent"):
            latent.kv_cache_pages(1, 10)
    finally:
        m.free()
        latent.free()


def _orders():
    whole = [[(0, p) for p in range(5)], [(1, p) for p in range(40)], [(2, 0)], [(3, p) for p in range(3)]]
    mixed = [(b, p) for p in range(3) for b in (0, 1)]
    return [
        # rows, those that have to come out as the sorted rows do (the others: NaN; None: whatever the positions in
        # front of them hold, which nothing was appended to)
        (sum(whole[::-1], []), lambda b, p: True),
        (whole[2] + whole[0] + whole[3] + whole[1], lambda b, p: True),
        (mixed + whole[2], lambda b, p: b == 2),
        (whole[1] + [(0, 0), (2, 0), (0, 1)], lambda b, p: b in (1, 2)),
        ([(7, 0)] + whole[1] + [(4, 0), ((1 << 32) - 1, 2)] + whole[0], lambda b, p: b in (0, 1)),
        (whole[3] + whole[3][:1] + whole[0], lambda b, p: b == 0),
        (whole[0][:3] + [(0, 4), (1, 0)], lambda b, p: b == 1),
        (whole[0] + [(1, p) for p in range(48, 53)], lambda b, p: b == 0 or (None if p < 50 else False)),
        (whole[0] + [(1, (1 << 32) - 1), (1, 0)], lambda b, p: b == 0),
        (whole[3] + [(0, p) for p in range(70)] + whole[2], lambda b, p: True),
    ]


@pytest.mark.parametrize("case", range(len(_orders())))
def test_prompts_in_any_order(dev, case):
    """Prompts one after the other in any order give what the sorted ones do; rows of a prompt that do not follow each
    other, of no prompt, or past the cache give NaN and leave the others alone."""
    rows, fine = _orders()[case]
    spec = mg.dense("bf16", hidden=128, inter=128, heads=4, kv_heads=2, head_dim=64, layers=2, vocab=100, seed=8)
    m = Model(dev, spec)
    a, b = m.kv_cache_pages(4, 50, page_tokens=32), m.kv_cache_pages(4, 50, page_tokens=32)
    token = {(x, y): (7 * x + 13 * y) % 100 for x, y in rows}
    good = sorted(r for r in set(rows) if fine(*r) and r[1] < 50)
    try:
        want = dict(zip(good, _cached(dev, m, a, [token[r] for r in good], good, np.arange(len(good)), 100)))
        for turn in range(2):  # (what the first left in the buffers must not show in the second)
            got = _cached(dev, m, b, [token[r] for r in rows], rows, np.arange(len(rows)), 100)
            for r, g in zip(rows, got):
                if fine(*r) is None:
                    continue
                if r in want:
                    assert np.abs(g - want[r]).max() <= 1e-5 * np.abs(want[r]).max(), r
                else:
                    assert np.isnan(g).all(), r
    finally:
        m.kv_cache_free(a)
        m.kv_cache_free(b)
        m.free()


MANY = [
    # heads, kv_heads, prompts, max_len, the calls: (prompt, rows) in the order of their rows
    (4, 1, 40, 300, [[(0, 20), (7, 1), (3, 13), (39, 2)], [(b, 1) for b in range(39, -1, -1)], [(7, 33), (0, 2)]]),
    (5, 1, 20, 100, [[(19, 4), (2, 7), (3, 1)], [(3, 1), (2, 1), (19, 3)]]),
    (20, 1, 33, 70, [[(5, 3), (4, 30)], [(b, 1) for b in range(33)], [(32, 2), (0, 1), (9, 5)]]),
    # more rows than prompts, a few of them in one prompt
    (4, 2, 300, 400, [[(b, 1) for b in range(299)] + [(299, 170)], [(299, 40)] + [(b, 1) for b in range(290)]]),
    # keys split over workgroups
    (4, 1, 3, 4000, [[(0, 1200), (1, 10)], [(2, 1), (0, 2)], [(0, 1), (1, 1)], [(0, 3)]]),
]


@pytest.mark.parametrize("case", range(len(MANY)))
def test_rows_of_some_of_many_prompts(dev, case):
    """Calls whose rows are those of few prompts or of many, no bound on a prompt's rows given, against the plain
    forward."""
    heads, kvh, prompts, max_len, calls = MANY[case]
    spec = mg.dense("bf16", hidden=128, inter=128, heads=heads, kv_heads=kvh, head_dim=64, layers=1, vocab=100, seed=case)
    spec.config["rope_len"] = max(max_len, spec.config["rope_len"])
    m = Model(dev, spec)
    cache = m.kv_cache_pages(prompts, max_len, page_tokens=32)
    plain = Plain(dev, spec, prompts, max_len, "int8", 32, 0, 0)
    rng = np.random.default_rng(case)
    pos = np.zeros(prompts, dtype=np.int64)
    try:
        for call in calls:
            rows = [(b, int(pos[b]) + i) for b, n in call for i in range(n)]
            tokens = rng.integers(0, 100, len(rows))
            got = _cached(dev, m, cache, tokens, rows, np.arange(len(rows)), 100)
            order = sorted(range(len(rows)), key=lambda i: rows[i])
            counts = np.bincount([b for b, _ in rows], minlength=prompts)
            want = plain.forward(tokens[order], np.concatenate([[0], np.cumsum(counts)]), pos)
            assert np.abs(got[order] - want).max() <= TOLERANCE["int8"] * np.abs(want).max()
            pos += counts
    finally:
        m.kv_cache_free(cache)
        m.free()


def test_a_step_of_thousands_of_prompts(dev):
    """A row for each of 2048 prompts with room for 2048 positions, and one for each of a few: the same logits."""
    spec = mg.dense("bf16", hidden=128, inter=128, heads=16, kv_heads=1, head_dim=64, layers=1, vocab=100, seed=9)
    spec.config["rope_len"] = 2048
    m = Model(dev, spec)
    n, some = 2048, [0, 1, 63, 700, 2047]
    big, small = m.kv_cache_pages(n, 2048, page_tokens=32), m.kv_cache_pages(len(some), 2048, page_tokens=32)
    rng = np.random.default_rng(3)
    try:
        for step in range(3):
            tokens, order = rng.integers(0, 100, n), rng.permutation(n)
            got = np.empty((n, 100), dtype=np.float32)
            got[order] = _cached(dev, m, big, tokens[order], [(b, step) for b in order], np.arange(n), 100)
            want = _cached(dev, m, small, tokens[some], [(i, step) for i in range(len(some))], np.arange(len(some)), 100)
            assert np.isfinite(got).all()
            assert np.abs(got[some] - want).max() <= TOLERANCE["int8"] * np.abs(want).max()
    finally:
        m.kv_cache_free(big)
        m.kv_cache_free(small)
        m.free()
