"""Calls of as many rows as they take, where a product or a norm has more threads
than a launch holds along one side."""
import numpy as np
import pytest

import model_gen as mg
import rows_ref as rr
from ditch_amd import hipmem
from ditch_amd.hip import Model
from test_gpu_head import _weight

pytestmark = pytest.mark.gpu

PERIOD = 4099  # rows that are different: a prime, so that none of a tile's rows repeats with the tiles


def test_losses_of_the_most_rows(dev):
    """2^24 rows on 40000 words: 10.3 million tiles of 256 x 256, 512 threads each. The rows repeat after 4099, and so
    do the results, bit for bit; some of the 4099 are compared with their values."""
    n, hidden, vocab = 1 << 24, 8, 40000
    rng = np.random.default_rng(6)
    t, w = _weight(dev, "bf16", vocab, hidden, 6)
    try:
        stored, values = rr.to_rows(rng.standard_normal((PERIOD, hidden)) * 2, "bf16")
        targets = rng.integers(-1, vocab, PERIOD).astype(np.int32)
        at = np.arange(n) % PERIOD
        x, tg = hipmem.Buffer.from_array(stored[at]), hipmem.Buffer.from_array(targets[at])
        need = t.head_loss_workspace(n, "bf16")
        assert need
        ws, out = hipmem.Buffer(need), [rr.Floats(n) for _ in range(2)]
        t.head_loss("bf16", out[0].ptr, out[1].ptr, dev.kv_rows(x.ptr, n * hidden * 2, hidden), n, tg.ptr, ws.ptr, need)
        hipmem.synchronize()
        few = np.r_[:20, PERIOD - 20:PERIOD]
        want = rr.loss(values[few], w, targets[few], "bf16", "bf16")
        for k, f in zip(("loss", "lse"), out):
            got = f.get()
            rr.check(got[few], *want[k], k)
            np.testing.assert_array_equal(got, got[:PERIOD][at], err_msg=k)
    finally:
        t.free()


def test_gradients_of_the_most_rows(dev):
    """The same over 600 words in pieces of 256, whose d are 8.6 GB each: dx repeats bit for bit, dW is the period's
    taken as often as its rows come (sums of 2^24 / 32 steps)."""
    n, hidden, vocab = 1 << 24, 8, 600
    rng = np.random.default_rng(7)
    t, w = _weight(dev, "bf16", vocab, hidden, 7)
    try:
        stored, values = rr.to_rows(rng.standard_normal((PERIOD, hidden)) * 2, "bf16")
        targets = rng.integers(-1, vocab, PERIOD).astype(np.int32)
        g = rng.standard_normal(PERIOD).astype(np.float32)
        at = np.arange(n) % PERIOD
        lse = rr._lse(values @ w.T).astype(np.float32)
        x, tg = hipmem.Buffer.from_array(stored[at]), hipmem.Buffer.from_array(targets[at])
        d_lse, d_g = rr.Floats(n, lse[at]), rr.Floats(n, g[at])
        dx, dw = rr.Rows(dev, n, hidden, "bf16"), rr.Rows(dev, vocab, hidden, "bf16")
        need = t.head_loss_grad_workspace(n, "bf16")
        ws = hipmem.Buffer(need)
        t.head_loss_grad("bf16", dx.desc, dw.desc, dev.kv_rows(x.ptr, n * hidden * 2, hidden), n, tg.ptr, d_lse.ptr,
                         d_g.ptr, ws.ptr, need)
        hipmem.synchronize()
        few = np.r_[:20, PERIOD - 20:PERIOD]
        got = dx.get()
        rr.check(got[few], *rr.loss_grad(values[few], w, targets[few], g[few].astype(np.float64), "bf16", "bf16")["dx"], "dx")
        np.testing.assert_array_equal(got, got[:PERIOD][at])
        l, off = rr.logits(values, w, "bf16", "bf16")
        _, _, p, p_off = rr._softmax(l, off)
        live = targets >= 0
        one = np.zeros_like(p)
        one[np.arange(PERIOD)[live], targets[live]] = 1
        weight = np.where(live, g.astype(np.float64), 0)[:, None] * np.bincount(at)[:, None]
        v, off = rr._back(((p - one) * weight).T, ((p_off + 2.0 ** -24) * np.abs(weight)).T, values, n, "bf16", 1, 1)
        rr.check(dw.get(), v, off, "dw")
    finally:
        t.free()


def test_hidden_rows_past_a_launch(dev):
    """2^24 + 77 final hidden rows, a workgroup of 256 threads each: the same few rows over and over."""
    spec = mg.dense(hidden=36, inter=64, layers=1, heads=2, kv_heads=1, head_dim=32, vocab=50, seed=3)
    model = Model(dev, spec)
    try:
        hidden, n, many = 36, 11, (1 << 24) + 77
        rng = np.random.default_rng(1)
        tokens = hipmem.Buffer.from_array(rng.integers(0, 50, n).astype(np.uint32))
        rows = hipmem.Buffer.from_array(np.array([(0, p) for p in range(n)], np.uint32))
        want = []
        for count in (n, many):
            at = hipmem.Buffer.from_array((np.arange(count) % n).astype(np.uint64))
            out = hipmem.Buffer.from_array(np.full(count * hidden, np.nan, np.float32))
            model.forward_hidden_device(tokens.ptr, rows.ptr, n, 1, n, at.ptr, count, out.ptr)
            dev.sync()
            want.append(out.download(np.float32, (count, hidden)))
        assert np.isfinite(want[0]).all()
        whole = many // n * n
        assert (want[1][:whole].reshape(-1, n, hidden) == want[0]).all() and (want[1][whole:] == want[0][:many - whole]).all()
    finally:
        model.free()
