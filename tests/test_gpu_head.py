"""Losses of rows against a head, and their gradients, against their
definitions in 64 bits (rows_ref.py: values and bounds)."""
import ctypes

import numpy as np
import pytest
import torch

import rows_ref as rr
from ditch_amd import abi, hipmem, synth
from ditch_amd.hip import DeviceError
from ditch_amd.weights import HostWeight

pytestmark = pytest.mark.gpu


def _weight(dev, fmt, rows, cols, seed):
    """A registered weight and the values it decodes to."""
    gen = torch.Generator().manual_seed(seed)
    w = torch.randn(rows, cols, generator=gen) * 0.05
    host = HostWeight.f16(w.half().numpy()) if fmt == "f16" else synth.QUANTIZERS[fmt](w)
    v = dev.dequant(host)
    return dev.upload(host), rr.from_rows(v, "bf16") if v.dtype == np.uint16 else v.astype(np.float64)


def _targets(rng, n, vocab):
    t = rng.integers(0, vocab, n).astype(np.int32)
    t[::5] = -100
    t[0] = vocab - 1
    return t


def _loss(dev, t, x, targets, stream=None):
    ws = rr.Workspace(t.head_loss_workspace(x.n, x.dtype))
    loss, lse = rr.Floats(x.n), rr.Floats(x.n)
    tg = hipmem.Buffer.from_array(targets)
    t.head_loss(x.dtype, loss.ptr, lse.ptr, x.desc, x.n, tg.ptr, *ws.args, stream=stream)
    hipmem.synchronize()
    ws.check()
    return {"loss": loss.get(), "lse": lse.get()}


def _loss_grad(dev, t, x, targets, lse, g, rows, cols, want=("dx", "dw"), gap=0):
    ws = rr.Workspace(t.head_loss_grad_workspace(x.n, x.dtype, dw="dw" in want))
    dx, dw = rr.Rows(dev, x.n, cols, x.dtype, gap=gap), rr.Rows(dev, rows, cols, x.dtype, gap=gap)
    tg, ls, gr = hipmem.Buffer.from_array(targets), rr.Floats(x.n, lse), rr.Floats(x.n, g)
    t.head_loss_grad(x.dtype, dx.desc if "dx" in want else None, dw.desc if "dw" in want else None, x.desc, x.n,
                     tg.ptr, ls.ptr, gr.ptr, *ws.args)
    hipmem.synchronize()
    ws.check()
    return {k: v.get() for k, v in (("dx", dx), ("dw", dw)) if k in want}


# (rows' type, weights' format, rows, vocabulary, width, elements between rows)
SHAPES = [("f32", "bf16", 1, 1, 1, 0), ("bf16", "bf16", 1, 300, 40, 3), ("f16", "bf16", 3, 17, 100, 1),
          ("f32", "f32", 5, 1000, 65, 0), ("bf16", "f32", 33, 257, 128, 8), ("f16", "f16", 70, 513, 96, 0),
          ("f32", "f16", 130, 255, 31, 5), ("bf16", "fp8", 64, 700, 256, 0), ("f32", "mxfp4", 17, 400, 128, 4),
          ("f16", "int4", 200, 300, 128, 0), ("f32", "q8_0", 9, 129, 64, 0), ("bf16", "bf16", 300, 1025, 200, 0),
          ("f32", "bf16", 129, 515, 897, 0), ("bf16", "bf16", 513, 64, 64, 0), ("f16", "q8_0", 16, 2049, 32, 2),
          ("f32", "fp8", 31, 600, 130, 0), ("bf16", "int4", 8, 4000, 256, 0), ("bf16", "f16", 2, 5000, 33, 0)]
ids = ["-".join(map(str, s)) for s in SHAPES]


@pytest.mark.parametrize("dtype,fmt,n,vocab,hidden,gap", SHAPES, ids=ids)
def test_loss_and_gradient(dev, dtype, fmt, n, vocab, hidden, gap):
    rng = np.random.default_rng(n * 1000 + vocab)
    t, w = _weight(dev, fmt, vocab, hidden, vocab)
    try:
        x = rr.Rows(dev, n, hidden, dtype, rng.standard_normal((n, hidden)) * 2, gap)
        targets = _targets(rng, n, vocab)
        got = _loss(dev, t, x, targets)
        for k, (v, off) in rr.loss(x.values, w, targets, dtype, fmt).items():
            rr.check(got[k], v, off, k)
        g = rng.standard_normal(n).astype(np.float32)
        grads = _loss_grad(dev, t, x, targets, got["lse"], g, vocab, hidden, gap=gap)
        for k, (v, off) in rr.loss_grad(x.values, w, targets, g.astype(np.float64), dtype, fmt).items():
            rr.check(grads[k], v, off, k)
        assert not grads["dx"][targets < 0].any()
        # one of the two alone is the same
        for want in ("dx", "dw"):
            alone = _loss_grad(dev, t, x, targets, got["lse"], g, vocab, hidden, want=(want,), gap=gap)
            np.testing.assert_array_equal(alone[want], grads[want])
    finally:
        t.free()


@pytest.mark.parametrize("dtype,fmt,n,vocab,hidden,gap", SHAPES, ids=ids)
@pytest.mark.parametrize("far", [0.01, 0.5, 4.0])
def test_divergence_and_gradient(dev, dtype, fmt, n, vocab, hidden, gap, far):
    rng = np.random.default_rng(n * 1000 + vocab)
    t, w = _weight(dev, fmt, vocab, hidden, vocab)
    try:
        a = rng.standard_normal((n, hidden)) * 2
        base = rr.Rows(dev, n, hidden, dtype, a, gap)
        trial = rr.Rows(dev, n, hidden, dtype, a + far * rng.standard_normal((n, hidden)), gap)
        got = _kl(dev, t, base, trial)
        for k, (v, off) in rr.kl(base.values, trial.values, w, dtype, fmt).items():
            rr.check(got[k], v, off, k)
        g = rng.standard_normal(n).astype(np.float32)
        dx = _kl_grad(dev, t, base, trial, got, g, gap)
        v, off = rr.kl_grad(base.values, trial.values, w, g.astype(np.float64), dtype, fmt)["dx"]
        rr.check(dx, v, off, "dx")
        # the same rows: no divergence, no gradient
        got = _kl(dev, t, base, base)
        assert not got["kl"].any()
        assert not _kl_grad(dev, t, base, base, got, g).any()
    finally:
        t.free()


def _kl(dev, t, base, trial):
    n = base.n
    ws = rr.Workspace(t.head_kl_workspace(n, base.dtype))
    out = {k: rr.Floats(n) for k in ("kl", "lse_base", "lse_trial")}
    t.head_kl(base.dtype, out["kl"].ptr, out["lse_base"].ptr, out["lse_trial"].ptr, base.desc, trial.desc, n, *ws.args)
    hipmem.synchronize()
    ws.check()
    return {k: v.get() for k, v in out.items()}


def _kl_grad(dev, t, base, trial, got, g, gap=0):
    n = base.n
    ws = rr.Workspace(t.head_kl_grad_workspace(n, base.dtype))
    dx = rr.Rows(dev, n, base.width, base.dtype, gap=gap)
    lb, lt, gr = rr.Floats(n, got["lse_base"]), rr.Floats(n, got["lse_trial"]), rr.Floats(n, g)
    t.head_kl_grad(base.dtype, dx.desc, base.desc, trial.desc, n, lb.ptr, lt.ptr, gr.ptr, *ws.args)
    hipmem.synchronize()
    ws.check()
    return dx.get()


@pytest.mark.parametrize("fmt,dtype,n,vocab,hidden", [("f32", "bf16", 3, 60000, 896), ("bf16", "f32", 700, 130000, 64)])
def test_several_pieces(dev, fmt, dtype, n, vocab, hidden):
    """Vocabularies that are taken in several pieces: decoded weights (60000 x 896 as three planes), and gradients of
    many rows (700 x 130000 as three terms)."""
    rng = np.random.default_rng(5)
    t, w = _weight(dev, fmt, vocab, hidden, 1)
    try:
        x = rr.Rows(dev, n, hidden, dtype, rng.standard_normal((n, hidden)))
        targets = _targets(rng, n, vocab)
        targets[1:3] = [0, vocab // 2]
        got = _loss(dev, t, x, targets)
        few = np.r_[:3, n - 1]  # rows that are compared; the sums over rows need them all
        for k, (v, off) in rr.loss(x.values[few], w, targets[few], dtype, fmt).items():
            rr.check(got[k][few], v, off, k)
        g = np.zeros(n, dtype=np.float32)
        g[few] = rng.standard_normal(len(few))
        few = np.unique(few)
        grads = _loss_grad(dev, t, x, targets, got["lse"], g, vocab, hidden)
        want = rr.loss_grad(x.values[few], w, targets[few], g[few].astype(np.float64), dtype, fmt)
        rr.check(grads["dx"][few], *want["dx"], "dx")
        # the others weigh nothing, but lengthen the sums
        rr.check(grads["dw"], want["dw"][0], want["dw"][1] * (1 + n / 32), "dw")
    finally:
        t.free()


def test_targets_outside_and_rows_that_are_not_finite(dev):
    rng = np.random.default_rng(3)
    n, vocab, hidden = 40, 333, 72
    t, w = _weight(dev, "bf16", vocab, hidden, 2)
    try:
        a = rng.standard_normal((n, hidden))
        targets = rng.integers(0, vocab, n).astype(np.int32)
        targets[[4, 5]] = [vocab, np.iinfo(np.int32).max]
        targets[[6, 7]] = [-1, np.iinfo(np.int32).min]
        bad = a.copy()
        bad[20, 3], bad[21, 7] = np.nan, np.inf
        x = rr.Rows(dev, n, hidden, "f32", bad)
        got = _loss(dev, t, x, targets)
        clean = np.ones(n, dtype=bool)
        clean[[20, 21]] = False
        want = rr.loss(a.astype(np.float32).astype(np.float64), w, targets, "f32", "bf16")
        rr.check(got["loss"][clean], want["loss"][0][clean], want["loss"][1][clean])
        assert np.isnan(got["loss"][[4, 5, 20]]).all() and not np.isfinite(got["loss"][21])
        assert (got["loss"][[6, 7]] == 0).all()
        grads = _loss_grad(dev, t, x, targets, np.where(clean, got["lse"], 0), np.ones(n), vocab, hidden, want=("dx",))
        v, off = rr.loss_grad(a.astype(np.float32).astype(np.float64), w, targets, np.ones(n), "f32", "bf16")["dx"]
        clean[[4, 5]] = False
        rr.check(grads["dx"][clean], v[clean], off[clean])
        assert np.isnan(grads["dx"][[4, 5, 20]]).all()
    finally:
        t.free()


def test_large_logits(dev):
    """Logits of some thousands: the sums are relative to the maximum; a divergence of rows far apart."""
    rng = np.random.default_rng(4)
    n, vocab, hidden = 20, 700, 64
    t, w = _weight(dev, "bf16", vocab, hidden, 9)
    try:
        a = rng.standard_normal((n, hidden)) * 5000
        x = rr.Rows(dev, n, hidden, "f32", a)
        y = rr.Rows(dev, n, hidden, "f32", -a)
        targets = _targets(rng, n, vocab)
        got = _loss(dev, t, x, targets)
        for k, (v, off) in rr.loss(x.values, w, targets, "f32", "bf16").items():
            rr.check(got[k], v, off, k)
        got = _kl(dev, t, x, y)
        for k, (v, off) in rr.kl(x.values, y.values, w, "f32", "bf16").items():
            rr.check(got[k], v, off, k)
    finally:
        t.free()


def test_gradient_against_differences(dev):
    """The gradients as slopes of the kernels' own losses: central differences of step h are off by h^2 / 6 times the
    third derivative (below 8 |w|^3 of the loss by a logit, |w| the change of the logits along the step) and by the
    losses' own error over h."""
    rng = np.random.default_rng(8)
    n, vocab, hidden, h = 6, 500, 48, 2.0 ** -6
    t, w = _weight(dev, "bf16", vocab, hidden, 4)
    try:
        a = (rng.integers(-200, 200, (n, hidden)) / 64.0)
        b = (rng.integers(-200, 200, (n, hidden)) / 64.0)
        targets = rng.integers(0, vocab, n).astype(np.int32)
        step = rng.integers(-1, 2, (n, hidden)).astype(np.float64)
        up, down, mid, base = (rr.Rows(dev, n, hidden, "f32", v) for v in (a + h * step, a - h * step, a, b))
        l = [_loss(dev, t, r, targets) for r in (up, down, mid)]
        grads = _loss_grad(dev, t, mid, targets, l[2]["lse"], np.ones(n), vocab, hidden, want=("dx",))["dx"]
        off = [rr.loss(r.values, w, targets, "f32", "bf16")["loss"][1] for r in (up, down)]
        bend = 8 * np.abs(step @ w.T).max(1) ** 3 * h * h / 6
        slack = (off[0] + off[1]) / (2 * h) + bend
        assert (np.abs((l[0]["loss"] - l[1]["loss"]) / (2 * h) - (grads * step).sum(1)) <= slack).all()
        k = [_kl(dev, t, base, r) for r in (up, down, mid)]
        grads = _kl_grad(dev, t, base, mid, k[2], np.ones(n))
        off = [rr.kl(base.values, r.values, w, "f32", "bf16")["kl"][1] for r in (up, down)]
        slack = (off[0] + off[1]) / (2 * h) + bend
        assert (np.abs((k[0]["kl"] - k[1]["kl"]) / (2 * h) - (grads * step).sum(1)) <= slack).all()
    finally:
        t.free()


def test_refusals(dev):
    n, vocab, hidden = 8, 100, 32
    t, _ = _weight(dev, "bf16", vocab, hidden, 1)
    lib = dev.lib
    try:
        x, dx, dw = (rr.Rows(dev, r, hidden, "f32", np.zeros((r, hidden))) for r in (n, n, vocab))
        f = rr.Floats(n, np.zeros(n))
        tg = hipmem.Buffer.from_array(np.zeros(n, dtype=np.int32))
        need = {k: getattr(t, k + "_workspace")(n, "f32") for k in ("head_loss", "head_loss_grad", "head_kl",
                                                                    "head_kl_grad")}
        ws = rr.Workspace(max(need.values()))
        p = ws.buf.ptr.value
        assert lib.ditch_hip_head_loss_workspace(t.handle, 0, abi.F32) == 0
        assert lib.ditch_hip_head_loss_workspace(t.handle, n, 4) == 0
        assert lib.ditch_hip_head_loss_workspace(None, n, abi.F32) == 0
        assert lib.ditch_hip_head_loss_workspace(t.handle, (1 << 24) + 1, abi.F32) == 0
        short = dev.kv_rows(x.buf.ptr, n * hidden * 4 - 1, hidden)
        narrow = dev.kv_rows(x.buf.ptr, n * hidden * 4, hidden - 1)
        crooked = dev.kv_rows(x.buf.ptr.value + 2, n * hidden * 4, hidden)
        null = dev.kv_rows(None, n * hidden * 4, hidden)

        def loss(loss=f.ptr, lse=f.ptr, rows=x.desc, targets=tg.ptr, at=p, size=need["head_loss"], count=n):
            t.head_loss("f32", loss, lse, rows, count, targets, at, size)

        def loss_grad(a=dx.desc, b=dw.desc, rows=x.desc, targets=tg.ptr, lse=f.ptr, g=f.ptr, at=p,
                      size=need["head_loss_grad"]):
            t.head_loss_grad("f32", a, b, rows, n, targets, lse, g, at, size)

        def kl(out=f.ptr, lse=f.ptr, base=x.desc, trial=x.desc, at=p, size=need["head_kl"]):
            t.head_kl("f32", out, lse, lse, base, trial, n, at, size)

        def kl_grad(a=dx.desc, base=x.desc, trial=x.desc, lse=f.ptr, g=f.ptr, at=p, size=need["head_kl_grad"]):
            t.head_kl_grad("f32", a, base, trial, n, lse, lse, g, at, size)

        bad = [lambda v=v: loss(rows=v) for v in (short, narrow, crooked, null, None)]
        bad += [lambda: loss(loss=None), lambda: loss(lse=None), lambda: loss(targets=None), lambda: loss(at=None),
                lambda: loss(at=p + 8), lambda: loss(size=need["head_loss"] - 1), lambda: loss(count=(1 << 24) + 1)]
        bad += [lambda v=v: loss_grad(a=v) for v in (short, narrow, crooked, null)]
        bad += [lambda: loss_grad(b=short), lambda: loss_grad(a=None, b=None), lambda: loss_grad(rows=None),
                lambda: loss_grad(targets=None), lambda: loss_grad(lse=None), lambda: loss_grad(g=None),
                lambda: loss_grad(size=need["head_loss_grad"] - 1)]
        bad += [lambda: kl(out=None), lambda: kl(lse=None), lambda: kl(base=short), lambda: kl(trial=narrow),
                lambda: kl(size=need["head_kl"] - 1)]
        bad += [lambda: kl_grad(a=None), lambda: kl_grad(a=short), lambda: kl_grad(base=null), lambda: kl_grad(trial=None),
                lambda: kl_grad(lse=None), lambda: kl_grad(g=None), lambda: kl_grad(size=need["head_kl_grad"] - 1)]
        for f_ in bad:
            with pytest.raises(DeviceError) as e:
                f_()
            assert e.value.status == abi.INVALID_ARGUMENT
        loss(count=0, rows=null, at=None, size=0)
        rc = lib.ditch_hip_head_loss_device(dev.h, f.ptr, f.ptr, 4, ctypes.byref(x.desc), n, t.handle, tg.ptr, p, ws.need, None)
        assert rc == abi.INVALID_ARGUMENT
    finally:
        t.free()
