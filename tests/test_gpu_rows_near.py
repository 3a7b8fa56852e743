"""Divergences of rows near each other, and their gradients, held to a share of
themselves.

The heads here have a mean direction: every word's row is a common one plus its
own. What moves along it moves all logits alike, and what is lost there is lost
for all words alike, while the roundings of the words' logits are independent of
each other, so that their sum over the words is taken as the root of the sum of
squares (six times that for one number, four times for the norm of a row's many).

A logit's own error: a product of k columns adds `pairs` matrix instructions for
each 32, each of which rounds the running sum by 2^-23 of it at most; as
independent roundings that is 2^-23 sqrt(pairs k / 32 + 2) of the largest logit
(running sums stay within it and the root of the sum of the squared products)."""
import numpy as np
import pytest
import torch

import rows_ref as rr
from ditch_amd import synth
from ditch_amd.weights import HostWeight
from test_gpu_head import _kl, _kl_grad

pytestmark = pytest.mark.gpu


def _head(dev, fmt, rows, cols, seed, mean, alike=None):
    """A registered head with a mean direction (`mean`: [cols], in units of the words' own part; the column `alike` has
    no part of their own) and its values."""
    gen = torch.Generator().manual_seed(seed)
    own = torch.randn(rows, cols, generator=gen)
    if alike is not None:
        own[:, alike] = 0
    w = (own + torch.as_tensor(mean, dtype=torch.float32)) * 0.05
    host = HostWeight.f16(w.half().numpy()) if fmt == "f16" else synth.QUANTIZERS[fmt](w)
    v = dev.dequant(host)
    return dev.upload(host), rr.from_rows(v, "bf16") if v.dtype == np.uint16 else v.astype(np.float64)


def _distributions(base, trial, w, dtype, fmt):
    """Logits, log sums and probabilities of both, and a logit's error."""
    lb, lt = base @ w.T, trial @ w.T
    sb, st = rr._lse(lb), rr._lse(lt)
    pairs = rr._pairs(3, rr.TERMS[dtype], rr.W_TERMS[fmt])
    size = np.abs(lb).max(1) + np.sqrt((base ** 2) @ (w ** 2).T).max(1)
    off = 2.0 ** -23 * np.sqrt(pairs * (w.shape[1] / 32) + 2) * size
    return lb, lt, sb, st, np.exp(lb - sb[:, None]), np.exp(lt - st[:, None]), off


def _kl_exact(base, trial, w, dtype, fmt):
    """The divergence and its bound: its derivatives by the logits are p (u - kl) and q - p, the second ones at most p;
    what is summed is of the size of p times the square of the differences' range, each to 2^-20 of itself."""
    lb, lt, sb, st, p, q, off = _distributions(base, trial, w, dtype, fmt)
    u = (lb - sb[:, None]) - (lt - st[:, None])
    small = np.abs(u) < 1e-3
    phi = np.where(small, u * u / 2 - u ** 3 / 6 + u ** 4 / 24, u + np.expm1(-np.where(small, 1, u)))
    v = (p * phi).sum(1)  # (sum p u, with the terms that sum p e^-u = 1 takes off)
    spread = u.max(1) - u.min(1)
    one = np.sqrt(((p * (u - v[:, None])) ** 2 + (q - p) ** 2).sum(1)) * off
    return v, 6 * one + 2 * off ** 2 + 2.0 ** -20 * (v + np.minimum(spread ** 2, spread)) + 2.0 ** -24 * v


# what the two rows' logits differ by alike for all words: nothing, less than 1 and more
@pytest.mark.parametrize("shift", [0.0, 0.5, -0.5, 4.0, -20.0])
@pytest.mark.parametrize("dtype,fmt,n,vocab,hidden", [("f32", "bf16", 7, 30000, 96), ("bf16", "bf16", 40, 9000, 128),
                                                      ("f16", "f16", 3, 5000, 65), ("f32", "fp8", 20, 4000, 128),
                                                      ("f32", "bf16", 300, 1500, 64)])
def test_near_divergences_under_a_common_shift(dev, dtype, fmt, n, vocab, hidden, shift):
    """Rows that differ by little but what moves all words' logits alike: no less exact than without that."""
    rng = np.random.default_rng(vocab)
    mean = np.zeros(hidden)
    mean[1] = 20.0  # column 1 of every word: 1
    t, w = _head(dev, fmt, vocab, hidden, 3, mean, alike=1)
    try:
        a = rng.standard_normal((n, hidden)) * 0.5
        a[:, 1] = 0.25
        b = a + 2.0 ** -6 * rng.standard_normal((n, hidden))
        b[:, 1] = 0.25 + shift
        base, trial = rr.Rows(dev, n, hidden, dtype, a), rr.Rows(dev, n, hidden, dtype, b)
        got = _kl(dev, t, base, trial)["kl"]
        v, off = _kl_exact(base.values, trial.values, w, dtype, fmt)
        rr.check(got, v, off, "kl")
    finally:
        t.free()


@pytest.mark.parametrize("far", [2.0 ** -1, 2.0 ** -4, 2.0 ** -7, 2.0 ** -10])
@pytest.mark.parametrize("dtype,fmt,n,vocab,hidden", [("f32", "bf16", 12, 40000, 256), ("f32", "fp8", 30, 20000, 256),
                                                      ("f32", "f32", 5, 30000, 200), ("f32", "mxfp4", 70, 9000, 128),
                                                      ("f32", "bf16", 700, 130000, 64), ("f32", "q8_0", 600, 5000, 64),
                                                      ("f16", "bf16", 20, 40000, 256), ("f16", "f16", 100, 20000, 128)])
def test_gradients_of_near_divergences(dev, dtype, fmt, n, vocab, hidden, far):
    """The gradient's error against its norm, where the log sums' own rounding (2^-21 of what they are taken from, along
    the head's mean direction) would be many times what the logits' roundings leave.

    d = p (e^(t - b - c) - 1): the logits' errors enter as p times theirs, independent for each word; p, its
    exponentials, the terms of d and the sums of the product by 2^-18 of the whole; a 16-bit result by half a step."""
    rng = np.random.default_rng(n)
    t, w = _head(dev, fmt, vocab, hidden, 5, rng.standard_normal(hidden))
    try:
        a = rng.standard_normal((n, hidden)) * 0.5
        base = rr.Rows(dev, n, hidden, dtype, a)
        trial = rr.Rows(dev, n, hidden, dtype, a + far * rng.standard_normal((n, hidden)))
        g = rng.standard_normal(n).astype(np.float32)
        dx = _kl_grad(dev, t, base, trial, _kl(dev, t, base, trial), g)
        few = np.unique(np.r_[:min(n, 12), n - 1])
        _, _, _, _, p, q, off = _distributions(base.values[few], trial.values[few], w, dtype, fmt)
        want = ((q - p) * g[few, None]) @ w
        size = np.linalg.norm(want, axis=1)
        each = np.abs(g[few]) * off * np.sqrt(((p ** 2 + q ** 2) @ (w ** 2)).sum(1))
        bound = 4 * each + 2.0 ** -18 * size
        if dtype == "f16":
            bound += 2.0 ** -11 * size + 2.0 ** -25 * hidden ** 0.5
        err = np.linalg.norm(dx[few] - want, axis=1)
        assert (err <= bound).all(), f"{(err / size).max():.3g} of the gradient, allowed {(bound / size)[np.argmax(err / bound)]:.3g}"
    finally:
        t.free()
