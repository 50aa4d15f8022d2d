"""opure_logprobs on rows whose masked logits are finite and very low: the type's
lowest value, -1e38 and others that a program fills in, mixed with ordinary ones."""
import numpy as np
import pytest

import opure_hip as H
import test_gpu_logprobs as P
from gpu_util import say

pytestmark = pytest.mark.gpu

LOWEST = np.finfo(np.float32).min
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    d = H.Dev(0)
    yield d
    d.close()


def reference(x, tokens, top, temperature):
    """(log p of tokens, entropy, top tokens, theirs) in 64 bits, and bounds of the errors.  With d = (x - m) /
    temperature, off by 2 u |d|, each e^d is relatively off by that, by u |d| for its argument's product and by 2^-21 (the
    hardware's exponential); a term below 2^-126 may be lost.  Sums of
    positive terms are off by 2^-24 times the longest chain: a lane's share of the vocabulary and 64 joins."""
    x = x.astype(np.float64)
    d = (x - x.max(1, keepdims=True)) / temperature
    e = np.exp(d)
    s = e.sum(1)
    chain = (-(-x.shape[1] // 256) + 16 + 64) * U
    off = 2 * U * np.abs(d)
    de = off + U * np.abs(d) + 2.0 ** -21
    count = e > 0
    rel = np.where(count, e * de, 0).sum(1) / s + chain
    log_s = np.log(s)
    tol_norm = rel + 4 * U * (log_s + 1)
    ent = log_s - np.where(count, e * d, 0).sum(1) / s
    ed = np.where(count, e * np.abs(d), 0)
    ent_tol = tol_norm + (ed * de + np.where(count, e * off, 0)).sum(1) / s + 2 * (chain + rel) * ed.sum(1) / s + 4 * U * np.abs(ent) + 2.0 ** -120 * x.shape[1]
    lp = d - log_s[:, None]
    lp_tol = tol_norm[:, None] + off + 2 * U * (np.abs(d) + log_s[:, None] + 1)
    # past fp32's numbers: -inf
    lp = np.where(lp < float(LOWEST), -np.inf, lp)
    tops = np.stack([P.order(r)[:top] for r in x]) if top else np.zeros((len(x), 0), int)
    pick = lambda a, i: np.take_along_axis(a, i, 1)  # noqa: E731
    at = np.asarray(tokens)[:, None]
    return (pick(lp, at)[:, 0], ent, tops, pick(lp, tops)), (pick(lp_tol, at)[:, 0], ent_tol, None, pick(lp_tol, tops))


def check(dev, x, top, temperature=1.0, tokens=None):
    x = np.asarray(x, np.float32)
    temperature = float(np.float32(temperature))
    tokens = np.random.default_rng(0).integers(0, x.shape[1], len(x)) if tokens is None else tokens
    c = P.Call(dev, x, tokens, top, temperature)
    got = c.run().result()
    want, tol = reference(x, tokens, top, temperature)
    assert np.array_equal(got[2], want[2])
    for i in (0, 1, 3):
        P.compare(got[i], want[i], tol[i])
    c.free()
    return got


def masked(rng, rows, vocab, fill, left):
    """Rows of which `left` of the tokens keep their logits, the first chunk none in every second row."""
    x = P.logits(rng, rows, vocab)
    hidden = rng.random(x.shape) >= left
    hidden[::2, :min(vocab // 2, 2000)] = True
    hidden[np.arange(rows), rng.integers(vocab // 2, vocab, rows)] = False
    x[hidden] = fill
    return x


FILLS = [LOWEST, -3e38, -1e38, -1e37, -1e36, -1e30, -1e20, -1e4]


@pytest.mark.parametrize("fill", FILLS)
@pytest.mark.parametrize("rows,vocab", [(12, 700), (5, 9000), (1, 128256), (530, 6001)])
def test_low_fills(dev, rows, vocab, fill):
    """In one slice a row and in several, a few chunks and many."""
    say("fill", rows, vocab, fill)
    rng = np.random.default_rng(vocab)
    for top, left in ((0, 0.05), (20, 0.3), (5, 0.001)):
        got = check(dev, masked(rng, rows, vocab, np.float32(fill), left), top)
        assert np.isfinite(got[1]).all()


def test_fills_mixed(dev):
    """Each of them in one row, ordinary logits first, last and between."""
    say("mixed")
    rng = np.random.default_rng(8)
    for vocab in (900, 9000, 40000):
        x = rng.choice(np.array(FILLS, np.float32), (6, vocab))
        x[0, :20], x[1, -20:], x[2, ::97] = 1.0, 2.0, 3.0
        x[3, vocab // 2] = 3e38
        x[4] = np.sort(x[4])                                # rising: a new maximum in many chunks
        x[5] = np.sort(x[5])[::-1]
        got = check(dev, x, 20)
        assert np.isfinite(got[1]).all()


@pytest.mark.parametrize("temperature", [0.05, 0.7, 0.999, 1.9, 60.0])
@pytest.mark.parametrize("rows,vocab", [(9, 700), (4, 9000), (1, 128256), (530, 6001)])
def test_low_fills_over_a_temperature(dev, rows, vocab, temperature):
    """A logit's quotient by the temperature may pass fp32's numbers where the differences that count do not."""
    say("temperature", rows, vocab, temperature)
    rng = np.random.default_rng(vocab)
    for fill, left in ((LOWEST, 0.05), (-3e38, 0.3), (-1e38, 0.001), (-1e30, 0.01)):
        got = check(dev, masked(rng, rows, vocab, np.float32(fill), left), 20, temperature)
        assert np.isfinite(got[1]).all()


@pytest.mark.parametrize("temperature", [0.05, 0.7, 1.0, 1.9, 60.0])
def test_rows_of_one_size(dev, temperature):
    """Nothing but masked logits: as likely as each other; and logits near fp32's largest."""
    say("rows", temperature)
    for vocab in (1, 700, 9000, 128256):
        x = np.full((3, vocab), LOWEST, np.float32)
        x[1], x[2] = -LOWEST, -1e38
        got = check(dev, x, min(vocab, 20), temperature, tokens=[0, vocab - 1, vocab // 2])
        assert np.allclose(got[1], np.log(vocab), rtol=1e-5)
    x = np.full((2, 9000), 3e38, np.float32)
    x[0, 8000], x[1, :5000] = 3.2e38, LOWEST
    check(dev, x, 20, temperature)


@pytest.mark.parametrize("temperature", [0.3, 2.5])
def test_numbers_that_are_not_finite_over_a_temperature(dev, temperature):
    """A NaN, a +inf or nothing but -inf make a row NaN, and no other; -inf among others has probability 0."""
    say("not finite", temperature)
    rng = np.random.default_rng(3)
    for vocab in (700, 9000):
        x = P.logits(rng, 7, vocab)
        x[1, vocab - 1], x[2, 5], x[3], x[4, ::2], x[5, :600] = np.nan, np.inf, -np.inf, -np.inf, LOWEST
        x[6, :600] = -np.inf
        c = P.Call(dev, x, [0] * 7, 9, float(np.float32(temperature)))
        got = c.run().result()
        c.free()
        assert np.array_equal(np.isnan(got[1]), [False, True, True, True, False, False, False])
        assert np.array_equal(got[2], np.stack([P.order(r)[:9] for r in x]))
        fine = [0, 4, 5, 6]
        finite = np.where(np.isneginf(x), -3e38, x).astype(np.float32)     # -inf as a number of probability 0
        want, tol = reference(finite[fine], [0] * 4, 9, float(np.float32(temperature)))
        P.compare(got[1][fine], want[1], tol[1])
        P.compare(got[3][fine], want[3], tol[3])
        assert np.isneginf(got[0][[4, 6]]).all() and np.isnan(got[0][[1, 2, 3]]).all()
