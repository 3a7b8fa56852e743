"""The gated block over rows and its gradient against their definitions in 64
bits (rows_ref.py: values and bounds)."""
import numpy as np
import pytest

import rows_ref as rr
from ditch_amd import abi, hipmem
from ditch_amd.hip import DeviceError
from test_gpu_head import _weight

pytestmark = pytest.mark.gpu


def _glu(dev, gate, up, x, rows, act, gap=0):
    ws = rr.Workspace(gate.glu_rows_workspace(up, x.n, x.dtype))
    out = rr.Rows(dev, x.n, rows, x.dtype, gap=gap)
    gate.glu_rows(up, x.dtype, out.desc, x.desc, x.n, *ws.args, act=act)
    hipmem.synchronize()
    ws.check()
    return out.get()


def _glu_grad(dev, gate, up, x, dout, rows, act, want=("dx", "dgate", "dup"), gap=0):
    ws = rr.Workspace(gate.glu_rows_grad_workspace(up, x.n, x.dtype, dw=want != ("dx",)))
    out = {k: rr.Rows(dev, x.n if k == "dx" else rows, x.width, x.dtype, gap=gap) for k in want}
    gate.glu_rows_grad(up, x.dtype, *(out[k].desc if k in out else None for k in ("dx", "dgate", "dup")), dout.desc,
                       x.desc, x.n, *ws.args, act=act)
    hipmem.synchronize()
    ws.check()
    return {k: v.get() for k, v in out.items()}


# (rows' type, weights' format, rows, block's width, hidden width, activation, elements between rows)
SHAPES = [("f32", "bf16", 1, 1, 1, 0, 0), ("bf16", "bf16", 1, 300, 40, 0, 3), ("f16", "bf16", 3, 17, 100, 1, 1),
          ("f32", "f32", 5, 200, 65, 2, 0), ("bf16", "f32", 33, 129, 128, 5, 8), ("f16", "f16", 70, 257, 96, 4, 0),
          ("f32", "f16", 130, 127, 31, 3, 5), ("bf16", "fp8", 64, 300, 256, 0, 0), ("f32", "mxfp4", 17, 100, 128, 0, 4),
          ("f16", "int4", 200, 150, 128, 0, 0), ("f32", "q8_0", 9, 65, 64, 1, 0), ("bf16", "bf16", 300, 515, 200, 0, 0),
          ("f32", "bf16", 129, 260, 897, 2, 0), ("bf16", "bf16", 513, 64, 64, 5, 0), ("f32", "fp8", 31, 150, 130, 0, 0),
          ("bf16", "bf16", 16, 640, 72, 1, 2)]


@pytest.mark.parametrize("dtype,fmt,n,inter,hidden,act,gap", SHAPES, ids=["-".join(map(str, s)) for s in SHAPES])
def test_block_and_gradient(dev, dtype, fmt, n, inter, hidden, act, gap):
    rng = np.random.default_rng(n * 1000 + inter)
    (gate, wg), (up, wu) = (_weight(dev, fmt, inter, hidden, inter + i) for i in range(2))
    try:
        x = rr.Rows(dev, n, hidden, dtype, rng.standard_normal((n, hidden)) * 3, gap)
        dout = rr.Rows(dev, n, inter, dtype, rng.standard_normal((n, inter)), gap)
        v, off = rr.glu(x.values, wg, wu, act, dtype, fmt)
        rr.check(_glu(dev, gate, up, x, inter, act, gap), v, off, "out")
        grads = _glu_grad(dev, gate, up, x, dout, inter, act, gap=gap)
        for k, (v, off) in rr.glu_grad(x.values, wg, wu, dout.values, act, dtype, fmt).items():
            rr.check(grads[k], v, off, k)
        for want in ("dx", "dgate", "dup"):
            alone = _glu_grad(dev, gate, up, x, dout, inter, act, want=(want,), gap=gap)
            np.testing.assert_array_equal(alone[want], grads[want])
    finally:
        gate.free()
        up.free()


def test_refusals(dev):
    n, inter, hidden = 4, 64, 32
    (gate, _), (up, _), (odd, _), (other, _) = (_weight(dev, f, r, hidden, 1) for f, r in
                                                 (("bf16", inter), ("bf16", inter), ("bf16", inter + 16), ("f32", inter)))
    try:
        x, out, dw = (rr.Rows(dev, r, c, "f32", np.zeros((r, c))) for r, c in ((n, hidden), (n, inter), (inter, hidden)))
        need, need_grad = gate.glu_rows_workspace(up, n, "f32"), gate.glu_rows_grad_workspace(up, n, "f32")
        ws = rr.Workspace(max(need, need_grad))
        p = ws.buf.ptr.value
        short = dev.kv_rows(x.buf.ptr, n * hidden * 4 - 1, hidden)
        for pair in ((gate, odd), (gate, other)):
            assert pair[0].glu_rows_workspace(pair[1], n, "f32") == 0
            with pytest.raises(DeviceError) as e:
                pair[0].glu_rows(pair[1], "f32", out.desc, x.desc, n, p, need)
            assert e.value.status == abi.UNSUPPORTED
        bad = [lambda: gate.glu_rows(up, "f32", out.desc, x.desc, n, p, need, act=6),
               lambda: gate.glu_rows(up, "f32", None, x.desc, n, p, need),
               lambda: gate.glu_rows(up, "f32", out.desc, short, n, p, need),
               lambda: gate.glu_rows(up, "f32", out.desc, x.desc, n, p, need - 1),
               lambda: gate.glu_rows(up, "f32", out.desc, x.desc, n, None, need),
               lambda: gate.glu_rows_grad(up, "f32", None, None, None, out.desc, x.desc, n, p, need_grad),
               lambda: gate.glu_rows_grad(up, "f32", x.desc, None, None, None, x.desc, n, p, need_grad),
               lambda: gate.glu_rows_grad(up, "f32", x.desc, short, None, out.desc, x.desc, n, p, need_grad),
               lambda: gate.glu_rows_grad(up, "f32", x.desc, dw.desc, None, out.desc, x.desc, n, p, need_grad - 1)]
        for f in bad:
            with pytest.raises(DeviceError) as e:
                f()
            assert e.value.status == abi.INVALID_ARGUMENT
        gate.glu_rows(up, "f32", out.desc, x.desc, 0, None, 0)
    finally:
        for t in (gate, up, odd, other):
            t.free()
