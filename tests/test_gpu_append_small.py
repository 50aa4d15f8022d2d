"""opure_kv_append to 4 bits of groups whose range is small for fp16's smallest steps, and
the bound of a value's error that the header states."""
import numpy as np
import pytest

import kv4_ref as K
import opure_hip as H
import test_gpu_append as A
from gpu_util import say

pytestmark = pytest.mark.gpu

F32 = H.A_F32


@pytest.fixture(scope="module")
def dev():
    d = H.Dev(0)
    yield d
    d.close()


def rounding(v):
    """What rounding v to fp16 is off by at most."""
    return np.maximum(2.0 ** -11 * np.abs(v), 2.0 ** -25)


def errors(dev, edit, seed):
    """Errors of the values held, and their groups' bounds: half a scale, 15 times the scale's rounding, base's and the
    value's (and fp32's own in the differences, 2^-22 of the largest magnitude)."""
    c = A.Append(dev, F32, F32, True, 1, 2, 128, [3], 40, rotate=False, seed=seed, edit=edit)
    c.run()
    c.expect()
    c.check()
    got = K.Kv4Pool(np.random.default_rng(0), 1, c.n_pages, 2, 128)
    got.words = dev.download(c.pool_buf, np.uint32, got.words.shape)
    pos = np.arange(3, 43)
    page, slot = c.table[0, pos // H.PAGE_SIZE], pos % H.PAGE_SIZE
    off, bound = [], []
    for which in (0, 1):
        for h in range(2):
            x = c.x[:, 128 * (1 + 2 * which + h):][:, :128].astype(np.float64)
            y = got.get(0, page, slot, h, which)
            g = x.reshape(40, 4, 32)
            lo, step, big = g.min(-1), (g.max(-1) - g.min(-1)) / 15, np.abs(g).max(-1)
            at_most = step + rounding(step)                  # the scale as it is held
            b = at_most / 2 + 15 * rounding(step) + rounding(np.abs(lo) + 16 * at_most) + rounding(big + at_most) + 2.0 ** -22 * (big + 16 * step)
            off.append(np.abs(x - y))
            bound.append(b.repeat(32, 1))
    c.free()
    return np.stack(off), np.stack(bound)


@pytest.mark.parametrize("spread", [1e-2, 1e-4, 1e-5, 1e-6, 3e-7, 1e-7, 1e-8, 1e-12])
@pytest.mark.parametrize("offset", [0.0, 1e-5, 1.0])
def test_error_of_small_ranges(dev, spread, offset):
    say("small", spread, offset)
    off, bound = errors(dev, lambda x: np.add(x * np.float32(spread), np.float32(offset), out=x), 9)
    assert (off <= bound).all(), float((off / bound).max())


def test_a_scale_of_one_smallest_step(dev):
    """0 .. 15 (1.49 2^-24): the scale is held as 2^-24, the largest value 7.35 of them too low."""
    say("step")

    def edit(x):
        g = x.reshape(len(x), -1, 32)
        g[...] = np.float32(1.49 * 2.0 ** -24) * (np.arange(32) % 16).astype(np.float32)

    off, bound = errors(dev, edit, 1)
    assert (off <= bound).all()
    assert off.max() > 7 * 2.0 ** -24                       # half a scale and the roundings of base and value are below 2 of them
