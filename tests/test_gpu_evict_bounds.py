"""What opure_kv_evict promises beyond its definition's values: every missing page is reported,
and scores_out may lie between the rows of scores."""
import numpy as np
import pytest

import opure_hip as H
import window_ref as R
from gpu_util import say
from test_gpu_evict import Evict, check

pytestmark = pytest.mark.gpu

F32, F16, BF16 = H.A_F32, H.A_F16, H.A_BF16


@pytest.fixture(scope="module")
def dev():
    d = H.Dev(0)
    yield d
    d.close()


@pytest.mark.parametrize("seq,budget,page", [([40, 30], (4, 30, 30), 1),       # nothing to evict
                                             ([1300, 20], (600, 300, 300), 0),  # before the sinks' last run
                                             ([3000, 20], (2, 0, 40), 180),     # far behind the last kept position
                                             ([3000, 1600], (700, 2, 3), 187)])
@pytest.mark.parametrize("afmt", [F32, F16], ids=["f32", "f16"])
def test_every_missing_page_is_reported(dev, afmt, seq, budget, page):
    """Also of a sequence that keeps all its positions, and where no position moves."""
    say("missing page", afmt, seq, budget, page)
    rng = np.random.default_rng(page)
    for value in (-1, 1 << 30):
        cache = R.Cache(rng, afmt, 1, 2, 32, seq)
        scores = rng.random((2, 1, 2, max(seq)), dtype=np.float32)
        scores[..., 200:] *= 0.001                              # the heavy ones lie in front
        cache.table[0, page] = value
        e = Evict(dev, cache, seq, scores, *budget, True)
        with pytest.raises(H.OpureError) as err:
            e.run()
        assert err.value.code == H.E_CAPACITY
        e.done()
    # pages past a sequence's positions are not its pages: missing in every shorter row of the table
    check(dev, afmt, 1, 2, 32, seq, *budget)


def test_scores_out_between_the_rows_of_scores(dev):
    rng = np.random.default_rng(1)
    n = 300
    cache = R.Cache(rng, F16, 2, 2, 32, [n, 200])
    scores = rng.random((2, 2, 2, 2 * n), dtype=np.float32)
    apart = Evict(dev, cache, [n, 200], scores, 2, 40, 50, True).run()
    e = Evict(dev, cache, [n, 200], scores, 2, 40, 50, True, with_scores=False)
    e.args.scores_out = int(e.scores) + 4 * n
    e.run()
    got = dev.download(e.scores, np.float32, scores.shape)
    want = apart.get()
    assert np.array_equal(got[..., :n], scores[..., :n])
    for b, length in enumerate((n, 200)):
        assert np.array_equal(got[b, ..., n:n + length], want["scores"][b, ..., :length])
        assert np.array_equal(got[b, ..., n + length:], scores[b, ..., n + length:])
    assert np.array_equal(e.get()["kept"], want["kept"]) and np.array_equal(e.get()["pool"], want["pool"])
    e.done()
    apart.done()


def test_scores_past_32_bits(dev):
    """Scores whose six planes lie 2^30 elements apart."""
    say("scores past 32 bits")
    rng = np.random.default_rng(2)
    n, stride = 250, (1 << 30) + 3
    cache = R.Cache(rng, BF16, 3, 2, 32, [n])
    scores = rng.random((1, 3, 2, n), dtype=np.float32)
    near = Evict(dev, cache, [n], scores, 2, 40, 50, True, in_place=True).run()
    far = dev.alloc((5 * stride + n) * 4)
    for plane in range(6):
        dev.write(far, scores.reshape(6, n)[plane], plane * stride * 4)
    e = Evict(dev, cache, [n], scores, 2, 40, 50, True)
    e.args.scores = e.args.scores_out = int(far)
    e.args.scores_stride = stride
    e.run()
    got, want = e.get(), near.get()
    assert np.array_equal(got["kept"], want["kept"]) and np.array_equal(got["pool"], want["pool"])
    for plane in range(6):
        assert np.array_equal(dev.download(far, np.float32, (n,), plane * stride * 4), want["scores"].reshape(6, n)[plane])
    e.done()
    near.done()
    far.free()
