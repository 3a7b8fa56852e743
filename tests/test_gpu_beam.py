"""The beam step against its definition in 64 bits.

The kernel forms d = logit - maximum in f32 (off by 2^-24 |d| at most) and
e^d within 2^-22, adds four in f32 (2 * 2^-24) and the rest in 64 bits: the log
sum exp is off by the mean of (2^-24 |d| + 2^-21) weighted with e^d. A score
adds its rounding to f32, 2^-24 of it. The choice is compared for equality,
with inputs whose scores are further apart than that, or tie exactly."""
import numpy as np
import pytest

from ditch_amd import abi, hipmem
from ditch_amd.hip import DeviceError

pytestmark = pytest.mark.gpu


def _plain(logits, prev, k):
    """logits [prompts][beams][vocab], prev [prompts][beams]: scores, parents, tokens, bounds [prompts][k]."""
    x = logits.astype(np.float64)
    with np.errstate(all="ignore"):
        m = x.max(-1, keepdims=True)
        e = np.exp(x - m)
        total = prev.astype(np.float64)[..., None] + (x - (m + np.log(e.sum(-1, keepdims=True))))
        off = np.where(e > 0, np.abs(x - m), 0) * 2.0 ** -24 + 2.0 ** -21
        off = ((off * e).sum(-1) / e.sum(-1)).reshape(len(x), -1)
    out = []
    for p, t in enumerate(total.reshape(len(x), -1)):
        beam, token, logit = np.arange(t.size) // x.shape[2], np.arange(t.size) % x.shape[2], x[p].reshape(-1)
        order = np.lexsort((token, -np.where(np.isnan(logit), -np.inf, logit), np.isnan(logit), beam,
                            -np.where(np.isnan(t), -np.inf, t), np.isnan(t)))[:k]
        out.append((t[order], beam[order], token[order], off[p][beam[order]]))
    return tuple(np.stack(a) for a in zip(*out))


def _select(dev, logits, prev, k, stream=None):
    n, beams, vocab = logits.shape
    need = dev.beam_select_workspace(n, beams, vocab, k)
    ws = hipmem.Buffer(need + 64)
    ws.upload(np.full(need + 64, 0xFF, dtype=np.uint8))
    x, p = hipmem.Buffer.from_array(logits.astype(np.float32)), hipmem.Buffer.from_array(prev.astype(np.float32))
    outs = [hipmem.Buffer(n * k * 4 + 64) for _ in range(3)]
    for o in outs:
        o.upload(np.full(n * k + 16, -77, dtype=np.int32))
    dev.beam_select(outs[0].ptr, outs[1].ptr, outs[2].ptr, x.ptr, p.ptr, n, beams, vocab, k, ws.ptr.value, need,
                    stream=stream)
    hipmem.synchronize()
    raw = [o.download(np.int32, (n * k + 16,)) for o in outs]
    assert all((r[n * k:] == -77).all() for r in raw)
    assert (ws.download(np.uint8, (need + 64,))[need:] == 0xFF).all()
    return raw[0][:n * k].view(np.float32).reshape(n, k), raw[1][:n * k].reshape(n, k), raw[2][:n * k].reshape(n, k)


def _check(dev, logits, prev, k):
    s, p, t = _select(dev, logits, prev, k)
    ws, wp, wt, off = _plain(logits, prev, k)
    np.testing.assert_array_equal(p, wp)
    np.testing.assert_array_equal(t, wt)
    np.testing.assert_array_equal(np.isnan(s), np.isnan(ws))
    fine = np.isfinite(ws)
    np.testing.assert_array_equal(s[~fine & ~np.isnan(ws)], ws[~fine & ~np.isnan(ws)])
    assert (np.abs(s[fine] - ws[fine]) <= off[fine] + 2.0 ** -24 * np.abs(ws[fine])).all()


SHAPES = [(1, 1, 1, 1), (1, 4, 151936, 8), (3, 8, 1000, 16), (2, 1, 4097, 1), (5, 3, 17, 51), (2, 64, 300, 128),
          (1, 2, 100, 128), (2, 5, 8192, 10), (40, 2, 2048, 4), (1, 16, 32768, 32), (7, 4, 33, 4)]


@pytest.mark.parametrize("prompts,beams,vocab,k", SHAPES)
def test_select(dev, prompts, beams, vocab, k):
    rng = np.random.default_rng(vocab + k)
    _check(dev, rng.standard_normal((prompts, beams, vocab)).astype(np.float32) * 3,
           -rng.uniform(0, 5, (prompts, beams)).astype(np.float32), k)


@pytest.mark.parametrize("prompts,beams,vocab,k", [(2, 4, 5000, 8), (1, 8, 70000, 128), (3, 3, 64, 20)])
def test_ties_go_to_the_lowest_index(dev, prompts, beams, vocab, k):
    """Logits of a few values, the same in every beam, and the same previous scores: nearly everything ties."""
    rng = np.random.default_rng(k)
    row = rng.integers(0, 3, (prompts, 1, vocab)).astype(np.float32)
    _check(dev, np.repeat(row, beams, 1), np.full((prompts, beams), -2.5, dtype=np.float32), k)
    _check(dev, np.zeros((prompts, beams, vocab), dtype=np.float32), np.zeros((prompts, beams), dtype=np.float32), k)


def test_the_best_in_one_place(dev):
    """The best continuations next to each other, at the ends, and all in one beam."""
    rng = np.random.default_rng(5)
    for vocab in (4096, 50001):
        x = rng.standard_normal((3, 4, vocab)).astype(np.float32)
        x[0, 2, :16] += 20 + np.arange(16)
        x[1, 1, -16:] += 20 + np.arange(16)
        x[2, 3, vocab // 2:vocab // 2 + 130] += 10 + np.arange(130)
        for k in (1, 16, 128):
            _check(dev, x, np.zeros((3, 4), dtype=np.float32), k)


def test_beams_that_have_not_begun_and_masked_tokens(dev):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((4, 3, 700)).astype(np.float32)
    prev = np.array([[0, -np.inf, -np.inf], [-1, -2, -3], [-np.inf] * 3, [0, -np.inf, -1]], dtype=np.float32)
    x[1, :, 5:] = -np.inf  # 15 continuations left, then those of probability zero, lowest index first
    x[3, 0, :] = -np.inf   # no probabilities
    for k in (1, 4, 20, 128):
        _check(dev, x, prev, k)


def test_logits_that_are_not_finite(dev):
    rng = np.random.default_rng(7)
    x = rng.standard_normal((4, 3, 900)).astype(np.float32)
    x[0, 1, 3] = np.nan
    x[1, 0, 899] = np.inf
    x[2, :, 0] = np.nan
    prev = np.zeros((4, 3), dtype=np.float32)
    prev[3, 1] = np.nan
    for k in (1, 5, 128):
        _check(dev, x, prev, k)


def test_logits_of_every_size(dev):
    rng = np.random.default_rng(8)
    for size in (1e-30, 1e4, 1e30):
        _check(dev, (rng.standard_normal((2, 3, 3000)) * size).astype(np.float32), np.zeros((2, 3), np.float32), 12)


def test_on_another_stream(dev):
    import ctypes
    lib = hipmem.hip()
    stream = ctypes.c_void_p()
    assert lib.hipStreamCreateWithFlags(ctypes.byref(stream), 1) == 0
    try:
        x = np.random.default_rng(9).standard_normal((2, 4, 20000)).astype(np.float32)
        a = _select(dev, x, np.zeros((2, 4), np.float32), 8, stream=stream.value)
        b = _select(dev, x, np.zeros((2, 4), np.float32), 8)
        for u, v in zip(a, b):
            np.testing.assert_array_equal(u, v)
    finally:
        lib.hipStreamDestroy(stream)


def test_refusals(dev):
    for shape in ((1, 0, 10, 1), (1, 65, 10, 1), (1, 2, 0, 1), (1, 2, 10, 0), (1, 2, 10, 21), (1, 4, 100, 129),
                  ((1 << 16) + 1, 1, 10, 1)):
        with pytest.raises(DeviceError) as e:
            dev.beam_select(16, 16, 16, 16, 16, *shape, 16, 1 << 40)
        assert e.value.status == abi.INVALID_ARGUMENT
    need = dev.beam_select_workspace(1, 2, 100, 4)
    for args in ((16, need - 1), (0, need), (8, need)):
        with pytest.raises(DeviceError, match="workspace"):
            dev.beam_select(16, 16, 16, 16, 16, 1, 2, 100, 4, *args)
    with pytest.raises(DeviceError):
        dev.beam_select(16, 16, None, 16, 16, 1, 2, 100, 4, 16, need)
    dev.beam_select(16, 16, 16, 16, 16, 0, 2, 100, 4, 16, need)  # no prompts: nothing to do


@pytest.mark.parametrize("prompts,beams,vocab,k", [(3, 4, 4097, 8), (2, 8, 50257, 16), (1, 6, 1001, 128),
                                                   (90, 4, 50257, 5), (1, 64, 30, 60)])
def test_equal_beams_tie(dev, prompts, beams, vocab, k):
    """Beams with the same random logits and the same previous scores, their rows at every alignment: the lower first."""
    rng = np.random.default_rng(vocab)
    row = rng.standard_normal((prompts, 1, vocab)).astype(np.float32) * 3
    _check(dev, np.repeat(row, beams, 1), np.full((prompts, beams), -1.25, dtype=np.float32), k)


def test_a_prompt_alone_and_in_a_batch(dev):
    """The same bits for a prompt by itself, in a batch of the larger chunks, and at every address."""
    rng = np.random.default_rng(10)
    n, beams, vocab, k = 84, 4, 50257, 6
    x = rng.standard_normal((n, beams, vocab)).astype(np.float32) * 2
    prev = -rng.uniform(0, 5, (n, beams)).astype(np.float32)
    whole = _select(dev, x, prev, k)
    for p in (0, 1, 2, 41, 83):
        for got, want in zip(_select(dev, x[p:p + 1], prev[p:p + 1], k), whole):
            np.testing.assert_array_equal(got[0], want[p])
    need = dev.beam_select_workspace(1, beams, vocab, k)
    ws, pb = hipmem.Buffer(need), hipmem.Buffer.from_array(prev[5])
    for shift in range(4):
        b = hipmem.Buffer.from_array(np.concatenate([np.zeros(shift, np.float32), x[5].ravel()]))
        outs = [hipmem.Buffer(k * 4) for _ in range(3)]
        dev.beam_select(outs[0].ptr, outs[1].ptr, outs[2].ptr, b.ptr.value + 4 * shift, pb.ptr, 1, beams, vocab, k,
                        ws.ptr.value, need)
        hipmem.synchronize()
        for got, want in zip(outs, whole):
            np.testing.assert_array_equal(got.download(np.int32, (k,)), want[5].view(np.int32))
