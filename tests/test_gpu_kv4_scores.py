"""opure_attn_kv4_paged where scores are large, up to those that 32 bits just hold: rows
with one number other than 0, whose scores are exact in 32 bits, so that what the
softmax makes of them is held to the definition by a bound that does not grow with them."""
import numpy as np
import pytest

import kv4_ref as K
import opure_hip as H
import window_ref as R
from gpu_util import say
from test_gpu_kv4_attn import compare

pytestmark = pytest.mark.gpu

F32, F16, BF16 = H.A_F32, H.A_F16, H.A_BF16

# |q| scale of a row: a score is that times a key's channel, 4 at most
SIZES = [1.0, 2.0 ** 9, 2.0 ** 14, 1.5 * 2.0 ** 17, 2.0 ** 20, 2.0 ** 22, 1.5 * 2.0 ** 24, 2.0 ** 27, 2.0 ** 28, 1.5 * 2.0 ** 28, 2.0 ** 29, 2.0 ** 30, 2.0 ** 33,
         2.0 ** 40, 2.0 ** 63, 2.0 ** 100, 2.0 ** 113]


@pytest.fixture(scope="module")
def dev():
    d = H.Dev(0)
    yield d
    d.close()


def reference(cache, q, afmt, heads, seq, rows, window, sinks, scale):
    """(out, bound) in 64 bits.  Scores are exact; a weight's exponent, of its distance d from the row's largest score, is
    off by 2^-22 |d| (the factor's rounding, log2 e's, a product's and a sum's) and its weight by 2^-20 (the exponential
    and the sums of positive terms), by its rounding (2^-11 as one fp16 number, 2^-22 as two) and by fp16's smallest
    step, 2^-37 of the row's largest weight; the result is rounded once."""
    out = np.zeros((len(seq), rows, heads, cache.hd))
    tol = np.zeros_like(out)
    G = heads // cache.n_kv
    for b, n0 in enumerate(seq):
        n = n0 + rows
        m = R.sees(n0, rows, n, window, sinks)
        for h in range(cache.n_kv):
            k, v = (cache.get(b, 0, h, i, n) for i in (0, 1))
            for g in range(G):
                s = np.where(m, q[b, :, h * G + g].astype(np.float64) @ k.T * scale, -np.inf)
                d = np.where(m, s - s.max(1, keepdims=True), -np.inf)
                e = np.exp(d)
                w = e / e.sum(1, keepdims=True)
                dw = w * (2.0 ** -22 * np.where(m, np.abs(d), 0) + 2.0 ** -20 + (2.0 ** -11 if afmt == BF16 else 2.0 ** -22)) + m * 2.0 ** -37
                o = w @ v
                out[b, :, h * G + g] = o
                tol[b, :, h * G + g] = (R.HALF_STEP[afmt] * (1 + 2.0 ** -10) * np.abs(o) + dw @ np.abs(v) + np.abs(o) * dw.sum(1, keepdims=True)
                                        + (2.0 ** -24 if afmt == F16 else 1e-30))
    return out, tol


def one_hot(shape, sizes):
    """Rows with one number, of the sizes in turn and of either sign, its channel another one each time."""
    q = np.zeros(shape, np.float32)
    flat = q.reshape(-1, shape[-1])
    i = np.arange(len(flat))
    flat[i, (7 * i + i // len(sizes)) % shape[-1]] = np.array(sizes, np.float32)[i % len(sizes)] * np.where(i // len(sizes) % 2, -1, 1)
    return q


def check(dev, afmt, heads, n_kv, hd, seq, rows, window=0, sinks=0, positive=False, sizes=SIZES, seed=0):
    rng = np.random.default_rng(seed)
    cache = K.Kv4Cache(rng, 1, n_kv, hd, [n + rows for n in seq])
    if positive:                                            # with negative queries every score is below -1 times their size
        for b, n in enumerate(seq):
            cache.put(b, np.arange(n + rows), 0, 0, np.abs(rng.standard_normal((n + rows, n_kv, hd)).astype(np.float32)) + 1)
    shape = (len(seq), rows, heads, hd)
    # fp16 has not the range: the scale has it there
    calls = [(one_hot(shape, [16.0]), size / 16) for size in sizes if size < 2.0 ** 101] if afmt == F16 else [(one_hot(shape, np.array(sizes) * 8), 0.125), (one_hot(shape, np.array(sizes) * 4), -0.25)]
    for q, scale in calls:
        c = K.Call(dev, cache, q, afmt, heads, seq, rows, window, sinks, scale)
        got = c.run().result()
        compare(got, *reference(cache, q, afmt, heads, seq, rows, window, sinks, scale))
        assert np.array_equal(got.view(np.uint32), c.run().result().view(np.uint32))
        c.free()


SHAPES = {  # sequences, rows, heads, KV heads
    "few": ([90, 0, 33], 6, 4, 2),                          # k_kv4_one
    "more": ([50], 40, 4, 2),                               # in blocks of 32 rows
    "long": ([2500], 2, 6, 2),                              # k_kv4_split and k_kv4_join
    "long-more": ([2500], 20, 4, 2),                        # in blocks of 32 rows
    "prompt": ([2650], 70, 64, 8),                          # k_kv4_rows in parts
    "prompt-short": ([900, 900], 100, 64, 16),              # and in one
}


@pytest.mark.parametrize("afmt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_sizes_of_scores(dev, shape, afmt):
    seq, rows, heads, n_kv = SHAPES[shape]
    say("scores", shape, afmt)
    check(dev, afmt, heads, n_kv, 64, seq, rows, sizes=SIZES if "prompt" not in shape or afmt != F16 else SIZES[3::3])
    check(dev, afmt, heads, n_kv, 32, seq, rows, 70, 3, positive="prompt" not in shape, sizes=SIZES[2::2], seed=1)
