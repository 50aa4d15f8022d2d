"""opure_logprobs against its definition in 64 bits: rows and vocabularies of any
size, masked logits, ties, NaN, infinities, tokens outside, capture and replay."""
import ctypes as C

import numpy as np
import pytest

import opure_hip as H
from gpu_util import say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = H.Dev(0)
    yield d
    d.close()


class Call:
    def __init__(self, dev, x, tokens=None, top=0, temperature=1.0, entropy=True, stride=None):
        self.dev, self.top, (self.rows, self.vocab) = dev, top, x.shape
        stride = stride or self.vocab
        wide = np.full((self.rows, stride), np.nan, np.float32)
        wide[:, :self.vocab] = x
        R = self.rows
        self.logits = dev.upload(wide)
        self.tokens = dev.upload(np.asarray(tokens, np.int32)) if tokens is not None else None
        guard = np.full(R * max(1, top) + 64, 0x12345678, np.uint32)
        self.out = [dev.upload(guard) for _ in range(4)]
        a = self.args = H.LogprobsArgs()
        a.rows, a.vocab, a.logits, a.logits_stride, a.temperature = R, self.vocab, int(self.logits), stride, temperature
        if tokens is not None:
            a.tokens, a.logprob = int(self.tokens), int(self.out[0])
        if entropy:
            a.entropy = int(self.out[1])
        a.top = top
        if top:
            a.top_tokens, a.top_logprobs = int(self.out[2]), int(self.out[3])

    def run(self, sync=True):
        H.check(H.lib().opure_logprobs(self.dev.h, C.byref(self.args)))
        if sync:
            self.dev.sync()
        return self

    def result(self):
        R, t = self.rows, self.top
        d = self.dev.download
        for buf, n, there in zip(self.out, (R, R, R * t, R * t), (self.args.logprob, self.args.entropy, t, t)):
            assert (d(buf, np.uint32, (64,), 4 * n if there else 0) == 0x12345678).all()        # nothing past the outputs
        return (d(self.out[0], np.float32, (R,)), d(self.out[1], np.float32, (R,)), d(self.out[2], np.int32, (R, t)), d(self.out[3], np.float32, (R, t)))

    def free(self):
        for b in [self.logits, *self.out] + ([self.tokens] if self.tokens else []):
            b.free()


def order(row):
    """Tokens by falling logit: NaN before every number, -0 as 0, ties by index."""
    r = np.where(np.isnan(row), np.inf, row) + 0.0
    return np.lexsort((np.arange(len(row)), -r, ~np.isnan(row)))


def reference(x, tokens, top, temperature):
    """(log p of tokens, entropy, top tokens, theirs) in 64 bits, and bounds of the errors.  With y = x / T off
    by half a step of fp32 (T other than 1), y - m off by half a step of its magnitude and the two rounded y's,
    each e^(y - m) is relatively off by that and 2^-21 (the hardware's exponential and its argument's product);
    sums of n positive terms by 2^-24 times the longest chain: a lane's share of the vocabulary, or the whole of
    a small one, and 32 joins."""
    R, V = x.shape
    x = x.astype(np.float64)
    bad = ~(x < np.inf).all(1) | ~(x > -np.inf).any(1)
    with np.errstate(all="ignore"):
        y = x / temperature
        m = y.max(1, keepdims=True)
        d = y - m
        e = np.exp(d)
        s = e.sum(1)
        ent = np.log(s) - np.where(e > 0, e * d, 0).sum(1) / s
        lp = d - np.log(s)[:, None]
    u = 2.0 ** -24
    scale = np.abs(np.where(np.isfinite(y), y, 0)).max(1) * (2 * u if temperature != 1 else 0)
    chain = (min(V, -(-V // 256) + 16) + 64) * u
    with np.errstate(all="ignore"):
        de = u * np.where(e > 0, np.abs(d), 0) + scale[:, None] + 2.0 ** -21 + np.where(e > 0, np.abs(d), 0) * u       # relative, of each term
        rel = (e * de).sum(1) / s + chain
        ls = np.abs(np.log(s))
        tol_norm = rel + 4 * u * (ls + 1)
        dm = np.where(e > 0, -d, 0)
        ent_tol = tol_norm + (e * (de * dm + u * dm + scale[:, None])).sum(1) / s + 2 * (chain + rel) * (e * dm).sum(1) / s + 4 * u * np.abs(ent) + 2.0 ** -126 * V
        lp_tol = tol_norm[:, None] + scale[:, None] + 2 * u * (np.abs(np.where(np.isfinite(d), d, 0)) + ls[:, None] + 1)
    lp[bad], ent[bad] = np.nan, np.nan
    tops = np.stack([order(r)[:top] for r in x]) if top else np.zeros((R, 0), int)
    pick = lambda a, i: np.take_along_axis(a, i, 1)  # noqa: E731
    t = np.asarray(tokens)
    inside = (t >= 0) & (t < V)
    at = np.where(inside, t, 0)[:, None]
    lpt = np.where(inside, pick(lp, at)[:, 0], np.nan)
    return (lpt, ent, tops, pick(lp, tops)), (pick(lp_tol, at)[:, 0], ent_tol, None, pick(lp_tol, tops))


def compare(got, want, tol):
    got = got.astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want)), (got, want)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    off = np.where(fine, np.abs(np.where(fine, got, 0) - np.where(fine, want, 0)) - np.where(fine, tol, 0), 0)
    assert not (off > 0).any(), (off.max(), got[off > 0][:3], want[off > 0][:3])


def check(dev, x, top, temperature=1.0, seed=0, tokens=None, stride=None):
    x = np.asarray(x, np.float32)
    rng = np.random.default_rng(seed)
    tokens = rng.integers(0, x.shape[1], x.shape[0]) if tokens is None else tokens
    c = Call(dev, x, tokens, top, temperature, stride=stride)
    got = c.run().result()
    want, tol = reference(x, tokens, top, temperature)
    assert np.array_equal(got[2], want[2]), (np.argwhere(got[2] != want[2])[:3], got[2][got[2] != want[2]][:3], want[2][got[2] != want[2]][:3])
    for i in (0, 1, 3):
        compare(got[i], want[i], tol[i])
    again = c.run().result()
    for a, b in zip(got, again):
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
    c.free()
    return got


def logits(rng, rows, vocab, spread=2.5):
    x = rng.standard_normal((rows, vocab), dtype=np.float32) * np.float32(spread)
    return x + (rng.random((rows, vocab)) > 0.99) * rng.random((rows, vocab)).astype(np.float32) * np.float32(8)


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 255, 1000, 1023, 1024, 1025, 4095, 4096, 4097, 5000, 8193, 49152, 128256, 151936])
@pytest.mark.parametrize("rows", [1, 3, 70])
def test_sizes(dev, rows, vocab):
    say("sizes", rows, vocab)
    rng = np.random.default_rng(vocab + rows)
    for top in (0, 1, 5, 20, 64):
        if top <= vocab and (rows < 70 or vocab < 10000 or top in (0, 20)):
            check(dev, logits(rng, rows, vocab), top, seed=top)


@pytest.mark.parametrize("rows", [200, 300, 600])
def test_many_rows(dev, rows):
    """One slice a row and more."""
    say("rows", rows)
    rng = np.random.default_rng(rows)
    for top, vocab in ((0, 9000), (1, 9000), (33, 20011)):
        check(dev, logits(rng, rows, vocab), top)


@pytest.mark.parametrize("seed", range(30))
def test_at_random(dev, seed):
    r = np.random.default_rng(seed)
    rows, vocab = int(2 ** r.uniform(0, 8)), int(2 ** r.uniform(0, 15))
    top = min(vocab, int(r.choice([0, 1, int(2 ** r.uniform(0, 6)), 64])))
    temperature = float(np.float32(r.choice([1.0, 0.7, 1.9, 0.05])))
    x = logits(r, rows, vocab)
    if r.random() < 0.4:
        x[r.random(x.shape) < 0.97] = -np.inf
        x[:, 0] = 1.0
    say("random", seed, rows, vocab, top, temperature)
    check(dev, x, top, temperature, seed, stride=vocab + int(r.integers(0, 9)))


@pytest.mark.parametrize("rows,vocab", [(1, 5000), (1, 128256), (520, 6001)])
def test_orders(dev, rows, vocab):
    """Rising and falling logits, equal ones, two values, zeros of both signs: every way that the largest arrive."""
    say("orders", rows, vocab)
    rng = np.random.default_rng(1)
    ramp = np.linspace(-20, 10, vocab, dtype=np.float32)
    kinds = [ramp, ramp[::-1], np.zeros(vocab), np.full(vocab, -np.inf), (np.arange(vocab) % 7).astype(np.float32), np.where(np.arange(vocab) % 2, 0.0, -0.0),
             np.round(rng.standard_normal(vocab)), np.where(np.arange(vocab) % 1000 == 999, 5.0, -np.inf)]
    if rows == 1:
        for k in kinds:
            for top in (1, 7, 64):
                check(dev, np.asarray(k, np.float32)[None], top)
    else:
        check(dev, np.stack([np.asarray(kinds[i % len(kinds)], np.float32) for i in range(rows)]), 40)


def test_nan_and_infinities(dev):
    """A row with a NaN or +inf reads NaN; others are not touched by it; a NaN counts as the largest."""
    say("nan")
    rng = np.random.default_rng(2)
    for vocab in (700, 9000):
        x = logits(rng, 12, vocab)
        x[1, 5], x[2, vocab - 1], x[3, 3] = np.nan, np.inf, -np.inf
        x[4, ::2] = np.nan
        x[5, :] = -np.inf
        x[6, :] = np.nan
        x[7, 10:400] = np.inf
        x[8, [4, 600]] = [np.nan, np.inf]
        x[9] = 3e38
        x[10] = -3e38
        x[11] *= np.float32(1e-30)
        got = check(dev, x, 64)
        assert np.isfinite(got[1][[0, 3, 9, 10, 11]]).all() and np.isnan(got[1][[1, 2, 4, 5, 6, 7, 8]]).all()


def test_masked_tokens(dev):
    """A token of probability 0 reads -inf; alternatives past the allowed tokens are -inf, the lowest first."""
    say("masked")
    x = np.full((2, 6000), -np.inf, np.float32)
    x[0, [17, 4000]], x[1, 5999] = [1.0, 2.0], 0.5
    got = check(dev, x, 6, tokens=[16, 5999])
    assert got[0][0] == -np.inf and got[0][1] == 0 and got[1][1] == 0
    assert got[2].tolist() == [[4000, 17, 0, 1, 2, 3], [5999, 0, 1, 2, 3, 4]]


@pytest.mark.parametrize("bad", [-1, 500, 0x7FFFFFFF, -0x80000000])
def test_tokens_outside(dev, bad):
    say("outside", bad)
    x = logits(np.random.default_rng(3), 3, 500)
    c = Call(dev, x, [3, bad, 499], 2)
    with pytest.raises(H.OpureError) as e:
        c.run()
    assert e.value.code == H.E_INVALID
    got = c.result()
    want, tol = reference(x, [3, bad, 499], 2, 1.0)
    assert np.array_equal(got[2], want[2])
    for i in (0, 1, 3):
        compare(got[i], want[i], tol[i])
    dev.sync()
    c.free()


def test_parts_left_out(dev):
    say("parts")
    x = logits(np.random.default_rng(4), 5, 3001)
    full = check(dev, x, 9, tokens=[1, 2, 3, 4, 5])
    for tokens, entropy, top in (([1, 2, 3, 4, 5], False, 0), (None, True, 0), (None, False, 9), ([1, 2, 3, 4, 5], False, 9)):
        c = Call(dev, x, tokens, top, entropy=entropy)
        got = c.run().result()
        if tokens:
            assert np.array_equal(got[0], full[0])
        if entropy:
            assert np.array_equal(got[1], full[1])
        if top:
            assert np.array_equal(got[2], full[2]) and np.array_equal(got[3], full[3])
        c.free()


@pytest.mark.parametrize("temperature", [0.01, 0.6, 1.0, 3.0, 100.0])
def test_temperatures(dev, temperature):
    say("temperature", temperature)
    check(dev, logits(np.random.default_rng(5), 20, 7000), 10, float(np.float32(temperature)))


def test_capture_and_replay(dev):
    say("graph")
    rng = np.random.default_rng(6)
    calls = []
    for rows, vocab, top in ((1, 50000, 20), (3, 20000, 64)):
        c = Call(dev, logits(rng, rows, vocab), rng.integers(0, vocab, rows), top)
        H.check(H.lib().opure_logprobs_reserve(dev.h, C.byref(c.args)))
        dev.graph_begin()
        c.run(sync=False)
        calls.append((c, dev.graph_end()))
    for _ in range(4):
        new = []
        for c, g in calls:
            x, t = logits(rng, c.rows, c.vocab), rng.integers(0, c.vocab, c.rows)
            dev.write(c.logits, x)
            dev.write(c.tokens, t.astype(np.int32))
            new.append((x, t))
            dev.graph_launch(g)
        dev.sync()
        for (c, g), (x, t) in zip(calls, new):
            got = c.result()
            want, tol = reference(x, t, c.top, 1.0)
            assert np.array_equal(got[2], want[2])
            for i in (0, 1, 3):
                compare(got[i], want[i], tol[i])
            for a, b in zip(got, c.run().result()):
                assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
    for c, g in calls:
        dev.graph_destroy(g)
        c.free()


def test_offsets_past_32_bits(dev):
    """Rows that lie past 4 GB."""
    say("large")
    rng = np.random.default_rng(7)
    rows, vocab, stride = 3, 5000, 3 << 28
    x = logits(rng, rows, vocab)
    c = Call(dev, x, [1, 2, 3], 4)
    want = c.run().result()
    far = dev.alloc(((rows - 1) * stride + vocab) * 4)
    for r in range(rows):
        dev.write(far, x[r], r * stride * 4)
    c.args.logits, c.args.logits_stride = int(far), stride
    for a, b in zip(want, c.run().result()):
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
    far.free()
    c.free()
