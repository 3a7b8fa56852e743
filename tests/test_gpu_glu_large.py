"""The gated block and its gradient where the gate's values are as large as f32 holds."""
import numpy as np
import pytest

import rows_ref as rr
from ditch_amd.weights import HostWeight
from test_gpu_glu import _glu, _glu_grad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", range(6))
@pytest.mark.parametrize("size", [1e3, 1e10, 1e20, 2.5e38])
def test_gates_of_any_size(dev, act, size):
    """Gates of +-size and 0, ups of +-1 and 2: every activation is flat or straight there (relu's square is left out
    where it overflows), so values and gradients are products of a few numbers, and f32's own rounding, half a step for
    each of at most eight operations, is all that they are off by."""
    if act == 4 and size > 1e10:
        pytest.skip("the square overflows")
    # three columns: the gate's, the up's, one that the weights do not read
    gate, up = np.zeros((3, 3), np.float32), np.zeros((3, 3), np.float32)
    gate[:, 0], up[:, 1] = [1, -1, 0], [1, -1, 2]
    tensors = [dev.upload(HostWeight.f32(w)) for w in (gate, up)]
    try:
        x = rr.Rows(dev, 2, 3, "f32", np.array([[size, 1, 3], [-size, 1, 5]]))
        dout = rr.Rows(dev, 2, 3, "f32", np.array([[0.5, 0.25, 1], [-0.5, 1, 2]]))
        g, u = x.values @ gate.astype(np.float64).T, x.values @ up.astype(np.float64).T
        y, dy, _ = rr.act(act, g)
        if act == 1:  # (rr.act's tanh form has infinity times 0 there, too)
            y, dy = np.where(g > 0, g, 0.0), np.where(g > 0, 1.0, np.where(g < 0, 0.0, 0.5))
        v = y * u
        rr.check(_glu(dev, *tensors, x, 3, act), v, np.abs(v) * 2.0 ** -21)
        got = _glu_grad(dev, *tensors, x, dout, 3, act)
        dg, du = dout.values * u * dy, dout.values * y
        want = {"dx": dg @ gate.astype(np.float64) + du @ up.astype(np.float64)}
        size = {"dx": np.abs(dg) @ np.abs(gate) + np.abs(du) @ np.abs(up)}
        rr.check(got["dx"], want["dx"], size["dx"] * 2.0 ** -20, "dx")
        for k, d in (("dgate", dg), ("dup", du)):
            with np.errstate(over="ignore"):
                want = d.T @ x.values
            fits = np.abs(d).T @ np.abs(x.values) < 3e38  # (a product past f32's range is what it is)
            rr.check(got[k][fits], want[fits], (np.abs(d).T @ np.abs(x.values))[fits] * 2.0 ** -20, k)
    finally:
        for t in tensors:
            t.free()
