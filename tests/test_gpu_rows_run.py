"""The head's losses, the gated block and their gradients as a program runs
them: on a model's own hidden rows, on other streams, in graphs, with offsets
past 32 bits."""
import ctypes

import numpy as np
import pytest

import model_gen as mg
import rows_ref as rr
from ditch_amd import abi, hipmem
from ditch_amd.hip import DeviceError, Model
from ditch_amd.weights import HostWeight
from test_gpu_glu import _glu, _glu_grad
from test_gpu_head import _kl, _kl_grad, _loss, _loss_grad, _weight

pytestmark = pytest.mark.gpu


def _hidden(model, tokens, rows, want, prompts, max_len, width):
    """The final hidden rows `want` of a batch, in device memory."""
    bt, br = hipmem.Buffer.from_array(np.asarray(tokens, np.uint32)), hipmem.Buffer.from_array(np.asarray(rows, np.uint32))
    bw, out = hipmem.Buffer.from_array(np.asarray(want, np.uint64)), hipmem.Buffer(len(want) * width * 4)
    model.forward_hidden_device(bt.ptr, br.ptr, len(tokens), prompts, max_len, bw.ptr, len(want), out.ptr)
    model.dev.sync()
    return out


@pytest.mark.parametrize("tie", [True, False])
def test_a_trial_scored_and_its_gradient(dev, tie):
    """A search's trial: the unedited model's final rows, an edit, the edited
    model's; their divergence over the head against the one from kept logits,
    the loss of the next tokens against their log-softmax, and gradients.

    The forward's own logits come from two-term products, off by 2^-18 of their
    absolute terms (four times that allowed); through a row's divergence that
    goes by p |u - kl| and |q - p|, and by its square."""
    spec = mg.dense(tie=tie, seed=5)
    c = spec.config
    model = Model(dev, spec)
    try:
        rng = np.random.default_rng(2)
        lens = [9, 1, 14]
        tokens = rng.integers(0, c["vocab"], sum(lens)).astype(np.uint32)
        rows = [(b, p) for b, n in enumerate(lens) for p in range(n)]
        n = len(rows)
        head = model.head()
        assert (head.rows, head.cols) == (c["vocab"], c["hidden"])
        w = rr.from_rows(dev.dequant(spec.tensors[(-1, abi.SLOT["EMBED" if tie else "LM_HEAD"], -1)]), "f32")

        def run():
            out = _hidden(model, tokens, rows, range(n), len(lens), max(lens), c["hidden"])
            x = rr.Rows(dev, n, c["hidden"], "f32", out.download(np.float32, (n, c["hidden"])))
            return x, model.forward(tokens, rows, logit_rows=range(n))[1]

        base, base_logits = run()
        v = rng.standard_normal((1, c["hidden"]))
        for layer in range(c["layers"]):
            for slot in ("O", "DOWN"):
                model.edit(layer, abi.SLOT[slot], -1, (v / np.linalg.norm(v)).astype(np.float32), 1.0)
        trial, trial_logits = run()
        got = _kl(dev, head, base, trial)
        for k, (value, off) in rr.kl(base.values, trial.values, w, "f32", "bf16").items():
            rr.check(got[k], value, off, k)
        assert (got["kl"] > 1e-6).all()
        kept = dev.klRows(dev.logSoftmaxRows(base_logits), trial_logits)
        lb, lt = base.values @ w.T, trial.values @ w.T
        p, q = (np.exp(l - rr._lse(l)[:, None]) for l in (lb, lt))
        u = np.log(p) - np.log(q)
        ob, ot = (2.0 ** -16 * np.abs(r.values) @ np.abs(w).T for r in (base, trial))
        off = (p * np.abs(u - got["kl"][:, None]) * ob + np.abs(q - p) * ot + (p + q) * (ob + ot) ** 2).sum(1)
        # (the f32 log-probabilities of the kept form: 2^-24 of each, p times)
        off += (p * np.abs(np.log(p))).sum(1) * 2.0 ** -23 + rr.kl(base.values, trial.values, w, "f32", "bf16")["kl"][1]
        assert (np.abs(kept - got["kl"]) <= off).all()
        # the loss of each prompt's next token; the last rows have none
        targets = np.array([tokens[i + 1] if i + 1 < n and rows[i + 1][0] == rows[i][0] else -100 for i in range(n)], np.int32)
        loss = _loss(dev, head, trial, targets)
        for k, (value, off) in rr.loss(trial.values, w, targets, "f32", "bf16").items():
            rr.check(loss[k], value, off, k)
        live = targets >= 0
        kept = -dev.logSoftmaxRows(trial_logits)[np.arange(n)[live], targets[live]]
        assert (np.abs(kept - loss["loss"][live]) <= 2 * ot.max(1)[live] + 2.0 ** -20 * np.abs(kept)).all()
        g = np.full(n, 1 / live.sum(), np.float32)
        grads = _loss_grad(dev, head, trial, targets, loss["lse"], g, c["vocab"], c["hidden"])
        for k, (value, off) in rr.loss_grad(trial.values, w, targets, g.astype(np.float64), "f32", "bf16").items():
            rr.check(grads[k], value, off, k)
        value, off = rr.kl_grad(base.values, trial.values, w, g.astype(np.float64), "f32", "bf16")["dx"]
        rr.check(_kl_grad(dev, head, base, trial, got, g), value, off, "dx")
    finally:
        model.free()


def test_an_edited_head_is_refused(dev):
    spec = mg.dense(tie=False, layers=1, seed=1)
    c = spec.config
    model = Model(dev, spec)
    try:
        model.head()
        model.set_delta(-1, abi.SLOT["LM_HEAD"], -1, np.ones((1, c["hidden"])), np.ones((c["vocab"], 1)))
        with pytest.raises(DeviceError, match="delta"):
            model.head()
        buf = hipmem.Buffer(4096)
        with pytest.raises(DeviceError):
            model.forward_hidden_device(buf.ptr, buf.ptr, 4, 1, 4, buf.ptr, 2, buf.ptr, hidden_bytes=2 * c["hidden"] * 4 - 1)
        with pytest.raises(DeviceError):
            model.forward_hidden_device(buf.ptr, buf.ptr, 4, 1, 4, None, 2, buf.ptr)
    finally:
        model.free()


class Step:
    """Everything of a training step of a head and a block on fixed buffers: loss and gradient, divergence and
    gradient, block and gradient, on one stream."""

    def __init__(self, dev, head, gate, up, dtype, n, hidden, seed, share=None):
        rng = np.random.default_rng(seed)
        self.dev, self.head, self.gate, self.up, self.dtype, self.n = dev, head, gate, up, dtype, n
        inter, vocab = gate.rows, head.rows
        self.x, self.y, self.dout = (rr.Rows(dev, n, k, dtype, rng.standard_normal((n, k))) for k in (hidden, hidden, inter))
        self.targets = hipmem.Buffer.from_array(rng.integers(-1, vocab, n).astype(np.int32))
        self.g = rr.Floats(n, rng.standard_normal(n).astype(np.float32))
        self.f = {k: rr.Floats(n) for k in ("loss", "lse", "kl", "lse_base", "lse_trial")}
        self.r = {"dx": rr.Rows(dev, n, hidden, dtype), "dw": rr.Rows(dev, vocab, hidden, dtype),
                  "dt": rr.Rows(dev, n, hidden, dtype), "out": rr.Rows(dev, n, inter, dtype),
                  "dh": rr.Rows(dev, n, hidden, dtype), "dgate": rr.Rows(dev, inter, hidden, dtype),
                  "dup": rr.Rows(dev, inter, hidden, dtype)}
        # one scratch for all of them: they follow each other
        self.ws = share or rr.Workspace(max(
            head.head_loss_workspace(n, dtype), head.head_loss_grad_workspace(n, dtype), head.head_kl_workspace(n, dtype),
            head.head_kl_grad_workspace(n, dtype), gate.glu_rows_workspace(up, n, dtype),
            gate.glu_rows_grad_workspace(up, n, dtype)))

    def renew(self, rng):
        for r in (self.x, self.y, self.dout):
            raw = r.buf.download(rr.STORE[self.dtype], (r.size,))
            raw[:r.n * r.stride] = rr.to_rows(rng.standard_normal((r.n, r.stride)), self.dtype)[0].reshape(-1)
            r.buf.upload(raw)
        self.targets.upload(rng.integers(-1, self.head.rows, self.n).astype(np.int32))

    def run(self, stream=None):
        h, f, r, n, ws, t = self.head, self.f, self.r, self.n, self.ws.args, self.dtype
        h.head_loss(t, f["loss"].ptr, f["lse"].ptr, self.x.desc, n, self.targets.ptr, *ws, stream=stream)
        h.head_loss_grad(t, r["dx"].desc, r["dw"].desc, self.x.desc, n, self.targets.ptr, f["lse"].ptr, self.g.ptr, *ws,
                         stream=stream)
        h.head_kl(t, f["kl"].ptr, f["lse_base"].ptr, f["lse_trial"].ptr, self.x.desc, self.y.desc, n, *ws, stream=stream)
        h.head_kl_grad(t, r["dt"].desc, self.x.desc, self.y.desc, n, f["lse_base"].ptr, f["lse_trial"].ptr, self.g.ptr,
                       *ws, stream=stream)
        self.gate.glu_rows(self.up, t, r["out"].desc, self.x.desc, n, *ws, stream=stream)
        self.gate.glu_rows_grad(self.up, t, r["dh"].desc, r["dgate"].desc, r["dup"].desc, self.dout.desc, self.x.desc, n,
                                *ws, stream=stream)

    def get(self):
        return {k: v.get() for k, v in {**self.f, **self.r}.items()}


def _same(a, b):
    for k in a:
        np.testing.assert_array_equal(a[k], b[k], err_msg=k)


@pytest.mark.parametrize("dtype,fmt,n", [("bf16", "bf16", 70), ("f32", "fp8", 20), ("f16", "f32", 300)])
def test_steps_on_two_streams_at_once(dev, dtype, fmt, n):
    """Two steps queued on two streams, each with its own scratch, give what they give one after the other."""
    lib = hipmem.hip()
    (head, _), (gate, _), (up, _) = (_weight(dev, fmt, r, 256, i) for i, r in enumerate((1100, 300, 300)))
    streams = [ctypes.c_void_p() for _ in range(2)]
    for s in streams:
        assert lib.hipStreamCreateWithFlags(ctypes.byref(s), 1) == 0
    try:
        steps = [Step(dev, head, gate, up, dtype, n + i, 256, i) for i in range(2)]
        want = []
        for s in steps:
            s.run()
            dev.sync()
            want.append(s.get())
        for _ in range(3):
            for s, st in zip(steps, streams):
                s.run(st.value)
            for st in streams:
                assert lib.hipStreamSynchronize(st) == 0
            for s, w in zip(steps, want):
                _same(s.get(), w)
                s.ws.check()
    finally:
        for st in streams:
            lib.hipStreamDestroy(st)
        for t in (head, gate, up):
            t.free()


@pytest.mark.parametrize("dtype,fmt,n", [("bf16", "bf16", 5), ("f32", "bf16", 150), ("f16", "fp8", 40)])
def test_steps_replayed_from_graphs(dev, dtype, fmt, n):
    """Two steps captured into two graphs that share one scratch, replayed in turn on one stream with new rows and
    eager calls between the replays: every replay is the eager step on the same rows."""
    lib = hipmem.hip()
    P = ctypes.c_void_p
    for name, args in {"hipStreamBeginCapture": [P, ctypes.c_int], "hipStreamEndCapture": [P, ctypes.POINTER(P)],
                       "hipGraphInstantiate": [ctypes.POINTER(P), P, P, P, ctypes.c_size_t],
                       "hipGraphLaunch": [P, P], "hipGraphExecDestroy": [P], "hipGraphDestroy": [P]}.items():
        getattr(lib, name).argtypes = args
        getattr(lib, name).restype = ctypes.c_int
    (head, _), (gate, _), (up, _) = (_weight(dev, fmt, r, 192, i) for i, r in enumerate((900, 260, 260)))
    stream, graphs, exes = P(), [P(), P()], [P(), P()]
    assert lib.hipStreamCreateWithFlags(ctypes.byref(stream), 1) == 0
    try:
        first = Step(dev, head, gate, up, dtype, n + 3, 192, 1)
        steps = [first, Step(dev, head, gate, up, dtype, n, 192, 2, share=first.ws)]
        hipmem.synchronize()
        for s, g, e in zip(steps, graphs, exes):
            assert lib.hipStreamBeginCapture(stream, 0) == 0
            s.run(stream.value)
            assert lib.hipStreamEndCapture(stream, ctypes.byref(g)) == 0
            assert lib.hipGraphInstantiate(ctypes.byref(e), g, None, None, 0) == 0
        rng = np.random.default_rng(3)
        for _ in range(4):
            for s in steps:
                s.renew(rng)
            hipmem.synchronize()
            for e in exes:
                assert lib.hipGraphLaunch(e, stream) == 0
            assert lib.hipStreamSynchronize(stream) == 0
            got = [s.get() for s in steps]
            for s, g in zip(steps, got):
                s.run()
                dev.sync()
                _same(g, s.get())
    finally:
        for e in exes:
            if e.value:
                lib.hipGraphExecDestroy(e)
        for g in graphs:
            if g.value:
                lib.hipGraphDestroy(g)
        lib.hipStreamDestroy(stream)
        for t in (head, gate, up):
            t.free()


def test_rows_far_apart(dev):
    """Two bf16 rows 2^31 + 64 elements apart."""
    hidden, vocab, stride = 48, 300, 2 ** 31 + 64
    t, w = _weight(dev, "bf16", vocab, hidden, 3)
    lib = hipmem.hip()
    try:
        rng = np.random.default_rng(1)
        stored, values = rr.to_rows(rng.standard_normal((2, hidden)), "bf16")
        buf = hipmem.Buffer((stride + hidden) * 2)
        for i in range(2):
            hipmem.check(lib.hipMemcpy(ctypes.c_void_p(buf.ptr.value + i * stride * 2), stored[i].ctypes.data_as(ctypes.c_void_p),
                                       hidden * 2, hipmem.H2D), "hipMemcpy")
        x = rr.Rows(dev, 2, hidden, "bf16")
        x.desc = dev.kv_rows(buf.ptr, (stride + hidden) * 2, stride)
        targets = np.array([7, 299], np.int32)
        got = _loss(dev, t, x, targets)
        for k, (v, off) in rr.loss(values, w, targets, "bf16", "bf16").items():
            rr.check(got[k], v, off, k)
    finally:
        t.free()


def test_direct_rows_far_apart(dev):
    """Sixteen bf16 rows as far apart as rows are read where they are: the last begins 1.9 GiB on."""
    n, hidden, vocab, stride = 16, 128, 300, 2 ** 26 - 8
    (t, w), (up, wu) = (_weight(dev, "bf16", vocab, hidden, i) for i in range(2))
    lib = hipmem.hip()
    try:
        stored, values = rr.to_rows(np.random.default_rng(1).standard_normal((n, hidden)), "bf16")
        size = ((n - 1) * stride + hidden) * 2
        buf = hipmem.Buffer(size)
        for i in range(n):
            hipmem.check(lib.hipMemcpy(ctypes.c_void_p(buf.ptr.value + i * stride * 2), stored[i].ctypes.data_as(ctypes.c_void_p),
                                       hidden * 2, hipmem.H2D), "hipMemcpy")
        x = rr.Rows(dev, n, hidden, "bf16")
        x.desc = dev.kv_rows(buf.ptr, size, stride)
        targets = np.arange(n, dtype=np.int32) * 9
        got = _loss(dev, t, x, targets)
        for k, (v, off) in rr.loss(values, w, targets, "bf16", "bf16").items():
            rr.check(got[k], v, off, k)
        v, off = rr.glu(values, w, wu, 0, "bf16", "bf16")
        rr.check(_glu(dev, t, up, x, vocab, 0), v, off, "out")
    finally:
        t.free()
        up.free()


def test_a_weight_gradient_past_32_bits(dev):
    """dW of 262400 x 4096 f32: 4.3 GB, its last rows past 2^32 bytes (MXFP4 weights, in many pieces). lse is an input
    here: any number."""
    vocab, hidden, n, lse = 262400, 4096, 3, 9.0
    rng = np.random.default_rng(7)
    host = HostWeight.mxfp4(rng.integers(0, 256, (vocab, hidden // 2), dtype=np.uint8),
                            rng.integers(118, 121, (vocab, hidden // 32), dtype=np.uint8))
    t = dev.upload(host)
    try:
        x = rr.Rows(dev, n, hidden, "f32", rng.standard_normal((n, hidden)) * 0.3)
        targets = hipmem.Buffer.from_array(np.array([vocab - 1, 5, -1], np.int32))
        g = np.array([1.0, -2.0, 1.0], np.float32)
        dw = hipmem.Buffer(vocab * hidden * 4)
        ws = rr.Workspace(t.head_loss_grad_workspace(n, "f32"))
        d_lse, d_g = rr.Floats(n, np.full(n, lse, np.float32)), rr.Floats(n, g)
        t.head_loss_grad("f32", None, dev.kv_rows(dw.ptr, vocab * hidden * 4, hidden), x.desc, n, targets.ptr, d_lse.ptr,
                         d_g.ptr, *ws.args)
        hipmem.synchronize()
        ws.check()
        for first in (0, 131072, 262144 - 8, vocab - 16):
            w = rr.from_rows(dev.dequant(host, first, 16), "bf16")
            l, off = rr.logits(x.values, w, "f32", "mxfp4")
            p = np.exp(l - lse)
            one = np.zeros_like(p)
            for i, v in enumerate((vocab - 1, 5)):
                if first <= v < first + 16:
                    one[i, v - first] = 1
            weight = np.array([1.0, -2.0, 0.0])
            d = (p - one) * weight[:, None]
            d_off = p * (off + 2.0 ** -21 + np.abs(l - lse) * 2.0 ** -22) * np.abs(weight)[:, None] + np.abs(d) * 2.0 ** -21
            got = np.empty((16, hidden), np.float32)
            hipmem.check(hipmem.hip().hipMemcpy(got.ctypes.data_as(ctypes.c_void_p),
                                                ctypes.c_void_p(dw.ptr.value + first * hidden * 4), got.nbytes,
                                                hipmem.D2H), "hipMemcpy")
            want = d.T @ x.values
            size = np.abs(d).T @ np.abs(x.values)
            rr.check(got, want, d_off.T @ np.abs(x.values) + size * 2.0 ** -18, f"rows from {first}")
    finally:
        t.free()


# a gradient's few rows on weights that are not planes, around the blocks of rows and of words that it counts in:
# (weights' format, rows' type, rows, vocabulary or block's width, hidden)
CODED = [("f16", "bf16", 16, 16, 32), ("f16", "f32", 17, 47, 64), ("f16", "f16", 256, 2100, 96), ("f32", "bf16", 65, 1045, 40),
         ("f32", "f32", 128, 3333, 72), ("f32", "f16", 129, 600, 320), ("q8_0", "bf16", 64, 335, 96), ("q8_0", "f32", 100, 31, 64),
         ("fp8", "bf16", 128, 4111, 200), ("fp8", "f16", 129, 300, 128), ("mxfp4", "bf16", 65, 2333, 160),
         ("mxfp4", "f32", 16, 1040, 288), ("int4", "f32", 100, 777, 256), ("int4", "bf16", 1, 1500, 128),
         ("f32", "f32", 500, 333, 64), ("f16", "bf16", 380, 700, 96), ("int4", "f16", 250, 130, 128)]


@pytest.mark.parametrize("fmt,dtype,n,rows,hidden", CODED, ids=["-".join(map(str, c)) for c in CODED])
def test_gradients_of_few_rows_on_coded_weights(dev, fmt, dtype, n, rows, hidden):
    rng = np.random.default_rng(rows + n)
    (t, w), (up, wu) = (_weight(dev, fmt, rows, hidden, i) for i in range(2))
    try:
        x = rr.Rows(dev, n, hidden, dtype, rng.standard_normal((n, hidden)))
        y = rr.Rows(dev, n, hidden, dtype, x.values + rng.standard_normal((n, hidden)))
        targets = rng.integers(-1, rows, n).astype(np.int32)
        g = rng.standard_normal(n).astype(np.float32)
        lse = rr.loss(x.values, w, targets, dtype, fmt)["lse"][0].astype(np.float32)
        got = _loss_grad(dev, t, x, targets, lse, g, rows, hidden)
        for k, (v, off) in rr.loss_grad(x.values, w, targets, g.astype(np.float64), dtype, fmt).items():
            rr.check(got[k], v, off, k)
        v, off = rr.kl_grad(x.values, y.values, w, g.astype(np.float64), dtype, fmt)["dx"]
        rr.check(_kl_grad(dev, t, x, y, _kl(dev, t, x, y), g), v, off, "dx")
        dout = rr.Rows(dev, n, rows, dtype, rng.standard_normal((n, rows)))
        got = _glu_grad(dev, t, up, x, dout, rows, 1)
        for k, (v, off) in rr.glu_grad(x.values, w, wu, dout.values, 1, dtype, fmt).items():
            rr.check(got[k], v, off, k)
    finally:
        t.free()
        up.free()


def test_a_coded_gradient_in_several_pieces(dev):
    """200 x 240000 values of d as three terms: 288 MB, two pieces of a weight that is read as it stands."""
    n, vocab, hidden = 200, 240000, 32
    rng = np.random.default_rng(9)
    t, w = _weight(dev, "f16", vocab, hidden, 1)
    try:
        x = rr.Rows(dev, n, hidden, "f32", rng.standard_normal((n, hidden)))
        targets = rng.integers(0, vocab, n).astype(np.int32)
        few = np.array([0, 77, 199])
        targets[few] = [vocab - 1, vocab // 2, 3]
        lse = np.full(n, 14.0, np.float32)
        want = rr.loss(x.values[few], w, targets[few], "f32", "f16")
        lse[few] = want["lse"][0]
        g = np.zeros(n, np.float32)
        g[few] = [1.0, -0.5, 2.0]
        got = _loss_grad(dev, t, x, targets, lse, g, vocab, hidden)
        want = rr.loss_grad(x.values[few], w, targets[few], g[few].astype(np.float64), "f32", "f16")
        rr.check(got["dx"][few], *want["dx"], "dx")
        # the others weigh nothing, but lengthen the sums
        rr.check(got["dw"], want["dw"][0], want["dw"][1] * (1 + n / 32), "dw")
    finally:
        t.free()


@pytest.mark.parametrize("dtype,n", [("bf16", 20), ("f32", 150)])
@pytest.mark.parametrize("kind", ["e5m2", "odd blocks", "special"])
def test_fp8_that_the_conversions_do_not_decode(dev, kind, dtype, n):
    """E5M2 codes, scale blocks of 32 columns, and a NaN code (whose word has no logit)."""
    rows, hidden = 203, 160
    rng = np.random.default_rng(n)
    codes = rng.integers(0, 256, (rows, hidden), dtype=np.uint8) & 0xbb  # finite in either form
    if kind == "special":
        codes[0, 0] = 0x7f
    block = 32 if kind == "odd blocks" else 64
    scale = (rng.random((-(-rows // 64), -(-hidden // block))) * 0.01 + 0.001).astype(np.float32)
    host = HostWeight.fp8(codes, scale, 64, block, e5m2=kind == "e5m2")
    t, w = dev.upload(host), rr.from_rows(dev.dequant(host), "bf16")
    try:
        x = rr.Rows(dev, n, hidden, dtype, rng.standard_normal((n, hidden)) * 0.1)
        targets = rng.integers(0, rows, n).astype(np.int32)
        if kind == "special":
            got = _loss(dev, t, x, targets)
            assert np.isnan(got["lse"]).all() and np.isnan(got["loss"]).all()
            return
        got = _loss(dev, t, x, targets)
        for k, (v, off) in rr.loss(x.values, w, targets, dtype, "fp8").items():
            rr.check(got[k], v, off, k)
        g = rng.standard_normal(n).astype(np.float32)
        grads = _loss_grad(dev, t, x, targets, got["lse"], g, rows, hidden)
        for k, (v, off) in rr.loss_grad(x.values, w, targets, g.astype(np.float64), dtype, "fp8").items():
            rr.check(grads[k], v, off, k)
    finally:
        t.free()


# up to 16 bf16 rows, read where they are if aligned; around the blocks of 16 and 32 rows:
# (weights' format, rows, vocabulary or block's width, hidden, elements between rows)
FEW = [("bf16", 1, 300, 128, 0), ("bf16", 16, 515, 256, 8), ("bf16", 7, 700, 384, 3), ("bf16", 15, 70, 128, 64),
       ("bf16", 32, 300, 64, 0), ("bf16", 33, 300, 128, 8), ("bf16", 96, 333, 40, 1), ("fp8", 16, 400, 256, 8),
       ("mxfp4", 5, 333, 128, 0), ("int4", 2, 90, 384, 24), ("q8_0", 3, 129, 128, 16), ("f16", 9, 100, 640, 0),
       ("f32", 16, 65, 256, 8), ("f16", 80, 100, 128, 0), ("bf16", 64, 8190, 32, 0), ("bf16", 40, 8210, 160, 0),
       ("bf16", 1, 16384, 64, 0), ("bf16", 3, 16385, 128, 0), ("bf16", 17, 31, 2049, 5)]


@pytest.mark.parametrize("fmt,n,rows,hidden,gap", FEW, ids=["-".join(map(str, c)) for c in FEW])
def test_few_bf16_rows(dev, fmt, n, rows, hidden, gap):
    rng = np.random.default_rng(rows * 7 + n)
    (t, w), (up, wu) = (_weight(dev, fmt, rows, hidden, i) for i in range(2))
    try:
        a = rng.standard_normal((n, hidden))
        x, y, far = (rr.Rows(dev, n, hidden, "bf16", v, g) for v, g in
                     ((a, gap), (a + rng.standard_normal((n, hidden)), gap), (a * 0.5, gap + 8)))
        targets = rng.integers(-1, rows, n).astype(np.int32)
        g = rng.standard_normal(n).astype(np.float32)
        got = _loss(dev, t, x, targets)
        for k, (v, off) in rr.loss(x.values, w, targets, "bf16", fmt).items():
            rr.check(got[k], v, off, k)
        got = _loss_grad(dev, t, x, targets, got["lse"], g, rows, hidden)
        for k, (v, off) in rr.loss_grad(x.values, w, targets, g.astype(np.float64), "bf16", fmt).items():
            rr.check(got[k], v, off, k)
        for trial in (y, far):  # (of the base's stride, and of another)
            got = _kl(dev, t, x, trial)
            for k, (v, off) in rr.kl(x.values, trial.values, w, "bf16", fmt).items():
                rr.check(got[k], v, off, k)
            v, off = rr.kl_grad(x.values, trial.values, w, g.astype(np.float64), "bf16", fmt)["dx"]
            rr.check(_kl_grad(dev, t, x, trial, got, g), v, off, "dx")
        v, off = rr.glu(x.values, w, wu, 2, "bf16", fmt)
        rr.check(_glu(dev, t, up, x, rows, 2), v, off, "out")
        dout = rr.Rows(dev, n, rows, "bf16", rng.standard_normal((n, rows)))
        got = _glu_grad(dev, t, up, x, dout, rows, 2)
        for k, (v, off) in rr.glu_grad(x.values, w, wu, dout.values, 2, "bf16", fmt).items():
            rr.check(got[k], v, off, k)
    finally:
        t.free()
        up.free()


@pytest.mark.parametrize("fmt,dtype,n,rows,hidden", [("f32", "f32", 890, 200, 72), ("f16", "bf16", 600, 450, 96),
                                                     ("mxfp4", "f32", 450, 333, 160), ("q8_0", "f16", 700, 129, 64),
                                                     ("int4", "bf16", 800, 90, 128), ("fp8", "f16", 250, 515, 200)])
def test_losses_of_many_rows_on_coded_weights(dev, fmt, dtype, n, rows, hidden):
    rng = np.random.default_rng(n)
    (t, w), (up, wu) = (_weight(dev, fmt, rows, hidden, i) for i in range(2))
    try:
        x = rr.Rows(dev, n, hidden, dtype, rng.standard_normal((n, hidden)))
        targets = rng.integers(-1, rows, n).astype(np.int32)
        got = _loss(dev, t, x, targets)
        for k, (v, off) in rr.loss(x.values, w, targets, dtype, fmt).items():
            rr.check(got[k], v, off, k)
        half = rr.Rows(dev, n // 2, hidden, dtype, x.values[: n // 2])
        other = rr.Rows(dev, n // 2, hidden, dtype, x.values[n // 2: n // 2 * 2])
        got = _kl(dev, t, half, other)
        for k, (v, off) in rr.kl(half.values, other.values, w, dtype, fmt).items():
            rr.check(got[k], v, off, k)
        v, off = rr.glu(x.values, w, wu, 0, dtype, fmt)
        rr.check(_glu(dev, t, up, x, rows, 0), v, off, "out")
    finally:
        t.free()
        up.free()


@pytest.mark.parametrize("dtype,fmt,n,vocab,hidden", [("f16", "f16", 4, 40000, 40), ("bf16", "f32", 3, 30000, 64),
                                                      ("f16", "f32", 70, 2000, 96), ("bf16", "q8_0", 40, 3000, 128),
                                                      ("f16", "q8_0", 1000, 300, 64), ("f16", "f16", 700, 515, 72)])
def test_losses_of_16_bit_rows_are_as_exact_as_f32_ones(dev, dtype, fmt, n, vocab, hidden):
    """Losses, log sums and divergences are f32, so 16-bit rows' products with any weights are held to the bounds of
    f32 rows (near ones: a divergence of 2^-8 of the logits would show what a 16-bit product leaves out)."""
    rng = np.random.default_rng(vocab)
    t, w = _weight(dev, fmt, vocab, hidden, 4)
    try:
        a = rng.standard_normal((n, hidden))
        x, y = (rr.Rows(dev, n, hidden, dtype, v) for v in (a, a + 0.02 * rng.standard_normal((n, hidden))))
        targets = rng.integers(0, vocab, n).astype(np.int32)
        got = _loss(dev, t, x, targets)
        for k, (v, off) in rr.loss(x.values, w, targets, "f32", fmt).items():
            rr.check(got[k], v, off, k)
        got = _kl(dev, t, x, y)
        for k, (v, off) in rr.kl(x.values, y.values, w, "f32", fmt).items():
            rr.check(got[k], v, off, k)
        # and, those bounds being far wider than what f32 sums lose: no worse than the same values as f32 rows, whose
        # terms are all multiplied (16 times, for sums in another order)
        full = _kl(dev, t, *(rr.Rows(dev, n, hidden, "f32", v.values) for v in (x, y)))["kl"]
        want = rr.kl(x.values, y.values, w, "f32", fmt)["kl"][0]
        worst = lambda v: (np.abs(v - want) / want).max()
        assert worst(got["kl"]) <= 16 * max(worst(full), 2.0 ** -23)
        if dtype == "f16":  # its gradient: d is held in 16 bits and the result rounded to 11
            g = rng.standard_normal(n).astype(np.float32)
            want = rr.kl_grad(x.values, y.values, w, g.astype(np.float64), "f32", fmt)["dx"][0]
            off = np.linalg.norm(_kl_grad(dev, t, x, y, got, g) - want, axis=1)
            assert (off <= 2.0 ** -11 * np.linalg.norm(want, axis=1) + 2.0 ** -24 * hidden ** 0.5).all()
    finally:
        t.free()


@pytest.mark.parametrize("dtype,fmt,n,hidden", [("bf16", "bf16", 12, 128), ("bf16", "bf16", 90, 200), ("f32", "bf16", 40, 72),
                                                ("f16", "fp8", 20, 128), ("bf16", "f16", 9, 256)])
def test_padding_holds_anything(dev, dtype, fmt, n, hidden):
    """A padded batch: rows without a target hold infinities, NaN and what their memory held, and change nothing."""
    vocab = 300
    rng = np.random.default_rng(n)
    t, w = _weight(dev, fmt, vocab, hidden, 2)
    try:
        a = rng.standard_normal((n, hidden))
        targets = rng.integers(0, vocab, n).astype(np.int32)
        pad = np.arange(n) % 3 == 1
        targets[pad] = np.where(np.arange(pad.sum()) % 2, -100, -1)
        a[pad] = 0
        x = rr.Rows(dev, n, hidden, dtype, a)
        a[pad] = rng.choice([np.nan, np.inf, -np.inf, 3.0], (pad.sum(), hidden))
        dirty = rr.Rows(dev, n, hidden, dtype, a)
        g = rng.standard_normal(n).astype(np.float32)
        g[pad] = np.nan
        want, got = _loss(dev, t, x, targets), _loss(dev, t, dirty, targets)
        np.testing.assert_array_equal(got["loss"], want["loss"])
        assert not got["loss"][pad].any()
        grads = _loss_grad(dev, t, dirty, targets, got["lse"], g, vocab, hidden)
        g[pad] = 0
        for k, (v, off) in rr.loss_grad(x.values, w, targets, g.astype(np.float64), dtype, fmt).items():
            rr.check(grads[k], v, off, k)
        assert not grads["dx"][pad].any()
    finally:
        t.free()
