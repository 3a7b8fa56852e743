"""The loss' gradient of 16-bit rows where logits are large: it takes the log sums of
the loss call, so its own logits have to be those that the loss summed."""
import numpy as np
import pytest

import rows_ref as rr
from test_gpu_head import _loss, _loss_grad
from test_gpu_rows_near import _head

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [3, 40, 700])
@pytest.mark.parametrize("dtype,fmt", [("f16", "f16"), ("f16", "f32"), ("f16", "q8_0"), ("bf16", "f16"), ("bf16", "f32"),
                                       ("f16", "bf16"), ("f32", "f32")])
def test_large_logits_of_a_common_direction(dev, dtype, fmt, n):
    """A head with a mean direction eight times the words' own part, rows along it: logits about 40. What all logits are
    off by alike moves dx along the mean direction. That is the log sum's rounding, half a step of f32, an
    exponential's 2^-21, nothing else: products leave no terms out, so logits are off by their roundings, independent
    of each other (four times the root of their squares' sum), by 2^-23 sqrt(4 k / 32 + 2) of their size, and by
    2^-17 of the root of the squared products' sum where a weight is taken at 16 bits. Then d held as the row type's
    terms and the result's half step."""
    vocab, hidden = 3000, 256
    rng = np.random.default_rng(n)
    mean = 8 * rng.standard_normal(hidden)
    t, w = _head(dev, fmt, vocab, hidden, 11, mean)
    try:
        x = rr.Rows(dev, n, hidden, dtype, 40 * mean / (0.05 * mean @ mean) + 0.5 * rng.standard_normal((n, hidden)))
        targets = rng.integers(0, vocab, n).astype(np.int32)
        got = _loss(dev, t, x, targets)
        g = rng.choice([-1.0, 0.5, 2.0], n).astype(np.float32)
        dx = _loss_grad(dev, t, x, targets, got["lse"], g, vocab, hidden, want=("dx",))["dx"]
        few = np.unique(np.r_[:min(n, 20), n - 1])
        v = x.values[few]
        l = v @ w.T
        p = np.exp(l - rr._lse(l)[:, None])
        sums = p @ w
        want = (sums - w[targets[few]]) * g[few, None]
        root = np.sqrt((v ** 2) @ (w ** 2).T).max(1)
        off = 2.0 ** -23 * np.sqrt(4 * hidden / 32 + 2) * (np.abs(l).max(1) + root)
        if fmt in ("f32", "q8_0") and dtype != "f32":
            off += 2.0 ** -17 * root
        each = off * np.sqrt(((p ** 2) @ (w ** 2)).sum(1))
        alike = (2.0 ** -24 * np.abs(l).max(1) + 2.0 ** -20) * np.linalg.norm(sums, axis=1)
        size = np.linalg.norm(want, axis=1)
        held = rr.HELD[rr.TERMS[dtype]] * np.sqrt((p ** 2 @ w ** 2).sum(1) + (w[targets[few]] ** 2).sum(1))
        bound = np.abs(g[few]) * (4 * each + alike + held) + (rr.HALF[dtype] + 2.0 ** -18) * size + rr.LEAST[dtype] * hidden ** 0.5
        err = np.linalg.norm(dx[few] - want, axis=1)
        assert (err <= bound).all(), f"{(err / size).max():.3g} of the gradient, allowed {(bound / size)[np.argmax(err / bound)]:.3g}"
    finally:
        t.free()
