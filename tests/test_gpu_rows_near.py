"""Divergences of rows near each other, held to a share of themselves.

The heads here have a mean direction: every word's row is a common one plus its
own. What moves along it moves all logits alike, while the roundings of the words' logits are independent of each other, so that
their sum over the words is taken as the root of the sum of squares (six times
that).

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
from test_gpu_head import _kl

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
