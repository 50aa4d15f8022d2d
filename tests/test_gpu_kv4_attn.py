"""opure_attn_kv4_paged against its definition in 64 bits: every format, head size
and layout, one row to a prompt's, windows and sinks of any length, what is masked
holding NaN, missing pages, capture and replay."""
import numpy as np
import pytest

import kv4_ref as K
import opure_hip as H
from gpu_util import say
from npref import act_to_f32, f32_to_act

pytestmark = pytest.mark.gpu

F32, F16, BF16 = H.A_F32, H.A_F16, H.A_BF16


@pytest.fixture(scope="module")
def dev():
    d = H.Dev(0)
    yield d
    d.close()


def compare(got, ref, tol):
    got = got.astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    fine = np.isfinite(ref)
    assert np.array_equal(got[~fine & ~np.isnan(ref)], ref[~fine & ~np.isnan(ref)])
    off = np.where(fine, np.abs(np.where(fine, got, 0) - np.where(fine, ref, 0)) - np.where(fine, tol, 0), 0)
    assert not np.isnan(off).any() and not (off > 0).any(), (float(off.max()), np.argwhere(off > 0)[:4])


def check(dev, afmt, heads, n_kv, hd, seq, rows, window=0, sinks=0, layers=1, seed=0, edit=None, spread=1.5, max_ctx=None, scale=None):
    rng = np.random.default_rng(seed)
    layer = layers - 1
    cache = K.Kv4Cache(rng, layers, n_kv, hd, [n + rows for n in seq], cap=max_ctx)
    q = act_to_f32(f32_to_act(rng.standard_normal((len(seq), rows, heads, hd), dtype=np.float32) * np.float32(spread), afmt), afmt)
    if edit:
        edit(cache, q)
    scale = hd ** -0.5 if scale is None else scale
    c = K.Call(dev, cache, q, afmt, heads, seq, rows, window, sinks, scale, layer, max_ctx)
    got = c.run().result()
    compare(got, *K.attention(cache, layer, q, afmt, heads, seq, rows, window, sinks, scale))
    assert np.array_equal(got.view(np.uint32), c.run().result().view(np.uint32))     # the same call, the same bits
    c.free()
    return got


@pytest.mark.parametrize("afmt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", list(range(16, 257, 16)))
def test_head_sizes(dev, hd, afmt):
    say("head size", hd, afmt)
    check(dev, afmt, 6, 2, hd, [0, 37, 150], 3, seed=hd)
    check(dev, afmt, 6, 2, hd, [0, 37, 150], 3, 50, 5, seed=hd)


SHAPES = {  # sequences, rows, heads: every way a call is run, at every head size
    "one-row": ([700, 3, 511], 1, 6),                    # a few query rows a KV head over a long cache
    "two-blocks": ([1200, 40], 12, 6),                   # 36: blocks of 32
    "prompt": ([70], 130, 4),                            # 260 over a short one
    "wide": ([30, 0, 64, 5] * 20, 40, 4),                # 80 sequences: more workgroups than the device has CUs
}


@pytest.mark.parametrize("shape,afmt", [(s, f) for s in SHAPES for f in (F32, F16, BF16) if s != "wide" or f == F16])
@pytest.mark.parametrize("hd", list(range(16, 257, 16)))
def test_every_kernel(dev, shape, hd, afmt):
    seq, rows, heads = SHAPES[shape]
    say("kernel", shape, hd, afmt)
    check(dev, afmt, heads, 2, hd, seq, rows, 333 if shape != "wide" else 40, 6, seed=hd)


@pytest.mark.parametrize("scale", [0.0, -0.11, 1.0, 3.0])
@pytest.mark.parametrize("rows,n", [(2, 700), (90, 20)])
def test_scales(dev, rows, n, scale):
    """attn_scale of either sign, and 0, where every visible position weighs the same."""
    say("scale", scale, rows)
    for afmt in (F32, F16, BF16):
        check(dev, afmt, 4, 2, 64, [n], rows, 50, 3, seed=rows, spread=0.3, scale=scale)


@pytest.mark.parametrize("spread", [1e-20, 1e-3, 30.0, 1e4, 1e20])
def test_query_magnitudes(dev, spread):
    """Rows far from 1, and rows of numbers of very different size (fp16 has neither)."""
    say("magnitude", spread)

    def uneven(cache, q):
        q[..., ::3] *= np.float32(1e-6)
        q[:, 1] = 0.0

    for afmt in (F32, BF16):
        for edit in (None, uneven):
            check(dev, afmt, 4, 2, 64, [90], 3, seed=3, spread=spread, scale=0.125 / spread, edit=edit)


@pytest.mark.parametrize("seed", range(60))
def test_shapes_at_random(dev, seed):
    r = np.random.default_rng(1000 + seed)
    n_kv, G = int(r.choice([1, 2, 3, 5, 8])), int(r.choice([1, 2, 3, 4, 7, 8]))
    afmt, hd = int(r.integers(0, 3)), 16 * int(r.integers(1, 17))
    rows = int(r.choice([1, 1, 2, 5, 9, 16, 33, 70, 150]))
    batch = int(r.integers(1, 6)) if rows < 33 else int(r.integers(1, 3))
    most = int(2 ** r.uniform(3, 11))
    seq = [int(r.integers(0, most)) for _ in range(batch)]
    window, sinks = int(r.choice([0, 0, 1, 15, 16, 63, 64, int(2 ** r.uniform(0, 11))])), int(r.choice([0, 0, 1, 4, 16, 33, 200]))
    say("random", seed, afmt, n_kv, G, hd, seq, rows, window, sinks)
    check(dev, afmt, n_kv * G, n_kv, hd, seq, rows, window, sinks, seed=seed, max_ctx=max(seq) + rows + int(r.choice([0, 0, 7, 500])))


def test_most_sequences(dev):
    say("256 sequences")
    rng = np.random.default_rng(12)
    check(dev, F16, 8, 2, 64, [int(n) for n in rng.integers(0, 300, 256)], 1, 100, 4)
    check(dev, BF16, 4, 1, 32, [int(n) for n in rng.integers(0, 60, 256)], 3)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (1, 40), (7, 0), (16, 4), (17, 3), (33, 16), (64, 70), (100, 0), (129, 33),
                                          (400, 2), (0, 0), (0, 9), (1 << 31, 5), (0xFFFFFFFF, 0xFFFF)])
@pytest.mark.parametrize("rows", [1, 5, 40])
def test_windows(dev, rows, window, sinks):
    say("window", rows, window, sinks)
    check(dev, BF16 if rows == 5 else F16, 8, 2, 64, [0, 1, 15, 16, 200, 333], rows, window, sinks, seed=rows)
    check(dev, F32, 3, 3, 32, [0, 15, 131], rows, window, sinks, seed=rows)


@pytest.mark.parametrize("heads,n_kv", [(1, 1), (7, 1), (9, 3), (16, 2), (40, 8), (5, 5), (33, 1)])
@pytest.mark.parametrize("rows", [1, 4, 16, 23])
def test_layouts(dev, heads, n_kv, rows):
    say("layout", heads, n_kv, rows)
    check(dev, F16, heads, n_kv, 64, [3, 77, 260], rows, 96, 4, layers=2, seed=heads)
    check(dev, BF16, heads, n_kv, 128, [90], rows, layers=3, seed=heads)


@pytest.mark.parametrize("afmt,hd", [(F16, 64), (BF16, 128), (F16, 96), (BF16, 80), (F32, 64), (F16, 256), (BF16, 16)])
@pytest.mark.parametrize("rows,start,window,sinks", [(17, 0, 0, 0), (130, 0, 50, 4), (333, 0, 0, 0), (200, 517, 128, 4), (260, 90, 1, 0),
                                                     (129, 700, 300, 70), (65, 64, 0, 0)])
def test_prompts(dev, afmt, hd, rows, start, window, sinks):
    say("prompt", afmt, hd, rows, start, window, sinks)
    check(dev, afmt, 8, 2, hd, [start], rows, window, sinks, seed=rows)
    check(dev, afmt, 8, 2, hd, [start, start // 2], rows, window, sinks, seed=rows + 1)


@pytest.mark.parametrize("afmt,hd,rows,n", [(F16, 64, 1, 5000), (BF16, 128, 2, 3000), (F32, 64, 1, 2500), (F16, 64, 1500, 600)])
def test_long(dev, afmt, hd, rows, n):
    """Caches and prompts long enough for every way of splitting the work; a
    spread of scores that a few positions dominate."""
    say("long", afmt, hd, rows, n)
    check(dev, afmt, 4, 1, hd, [n], rows, seed=n, spread=6.0)
    check(dev, afmt, 4, 1, hd, [n], rows, 1031, 4, seed=n + 1, spread=6.0)
    check(dev, afmt, 8, 2, hd, [n, n // 7, 9], rows, 700, 20, seed=n + 2)


@pytest.mark.parametrize("afmt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,window,sinks", [(6, 20, 3), (70, 33, 2)])
def test_masked_positions_may_hold_anything(dev, afmt, rows, window, sinks):
    """Groups of NaN at positions that some rows see and others do not: the rows
    that do not see them are not touched by them."""
    say("masked", afmt, rows)
    n0 = 100

    def edit(cache, q):
        rng = np.random.default_rng(1)
        for t, value in ((n0 + 2, np.nan), (n0 - window + 1, np.inf), (n0 + rows - 2, -np.inf)):
            k, v = (rng.standard_normal((1, cache.n_kv, cache.hd)).astype(np.float32) for _ in range(2))
            v[0, 0, 5] = value                              # V of one KV head
            k[0, 1, 3] = value                              # K of the other
            cache.put(0, [t], 0, 0, k)
            cache.put(0, [t], 0, 1, v)
        # positions between the sinks and every window: nothing of them is read
        hidden = np.arange(sinks, n0 - window)
        for which in (0, 1):
            cache.put(0, hidden, 0, which, np.full((len(hidden), cache.n_kv, cache.hd), np.nan, np.float32))

    got = check(dev, afmt, 4, 2, 64, [n0], rows, window, sinks, edit=edit, spread=0.5)
    assert np.isfinite(got).any() and not np.isfinite(got).all()


@pytest.mark.parametrize("afmt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_queries_that_are_not_finite(dev, afmt):
    """A NaN or an infinity in one row's query stays in that row; scores of -inf weigh nothing."""
    say("queries", afmt)

    def edit(cache, q):
        q[0, 1, 2, 7], q[0, 3, 0, 0] = np.nan, np.inf
        cache.put(0, np.arange(60), 0, 0, np.abs(np.random.default_rng(3).standard_normal((60, 2, 64)).astype(np.float32)) + 0.5)
        q[0, 4, 1] = np.abs(q[0, 4, 1]) + 1
        q[0, 4, 1, 9] = -np.inf                             # every score of this row is -inf: 0

    got = check(dev, afmt, 4, 2, 64, [52], 8, edit=edit)
    assert (got[0, 4, 1] == 0).all() and np.isnan(got[0, 1, 2]).all()


@pytest.mark.parametrize("rows", [1, 4, 60])
def test_pages_that_are_missing(dev, rows):
    """Pages that no row sees may be missing; a row that sees a missing one is NaN."""
    say("missing", rows)
    rng = np.random.default_rng(5)
    n0, window, sinks = 300, 70, 5
    for afmt in (F16, F32):
        cache = K.Kv4Cache(rng, 1, 2, 64, [n0 + rows])
        q = act_to_f32(f32_to_act(rng.standard_normal((1, rows, 4, 64), dtype=np.float32), afmt), afmt)
        ref, tol = K.attention(cache, 0, q, afmt, 4, [n0], rows, window, sinks, 0.125)
        cache.table[0, 1:(n0 - window + 1) // 16] = -1
        c = K.Call(dev, cache, q, afmt, 4, [n0], rows, window, sinks, 0.125)
        compare(c.run().result(), ref, tol)
        # the page of the first row's own position
        table = cache.table.copy()
        table[0, n0 // 16] = -1
        dev.write(c.bufs[1], table)
        got = c.run().result()
        pos = n0 + np.arange(rows)
        sees = pos - window < n0 // 16 * 16 + 15
        assert np.isnan(got[0, sees]).all()
        if not sees.all():
            compare(got[:, ~sees], ref[:, ~sees], tol[:, ~sees])
        c.free()


def test_lengths_past_the_capacity(dev):
    say("lengths")
    rng = np.random.default_rng(6)
    cache = K.Kv4Cache(rng, 1, 2, 64, [40, 70])
    q = rng.standard_normal((2, 2, 4, 64), dtype=np.float32)
    ref, tol = K.attention(cache, 0, q, F32, 4, [38, 68], 2, 0, 0, 0.125)
    c = K.Call(dev, cache, q, F32, 4, [38, 68], 2, 0, 0, 0.125)
    for bad in (-1, 69, 0x7FFFFFFF, -0x80000000):
        dev.write(c.bufs[2], np.array([38, bad], np.int32))
        with pytest.raises(H.OpureError) as e:
            c.run()
        assert e.value.code == H.E_CAPACITY
        compare(c.result()[:1], ref[:1], tol[:1])
    c.free()


def test_capture_and_replay(dev):
    """Two captured shapes share the workspace; lengths change between replays."""
    say("graph")
    rng = np.random.default_rng(8)
    cache = K.Kv4Cache(rng, 1, 2, 64, [900, 500])
    calls = []
    for afmt, rows in ((F16, 1), (BF16, 9)):
        q = act_to_f32(f32_to_act(rng.standard_normal((2, rows, 8, 64), dtype=np.float32), afmt), afmt)
        c = K.Call(dev, cache, q, afmt, 8, [800, 400], rows, 0, 0, 0.125, max_ctx=900)
        H.check(H.lib().opure_attn_kv4_reserve(dev.h, K.C.byref(c.args)))
        dev.graph_begin()
        c.run(sync=False)
        calls.append((c, dev.graph_end(), q, afmt, rows))
    for seq in ([800, 400], [10, 0], [891, 491], [333, 100]):
        for c, g, q, afmt, rows in calls:
            dev.write(c.bufs[2], np.array(seq, np.int32))
            dev.graph_launch(g)
        dev.sync()
        for c, g, q, afmt, rows in calls:
            got = c.result()
            compare(got, *K.attention(cache, 0, q, afmt, 8, seq, rows, 0, 0, 0.125))
            assert np.array_equal(got.view(np.uint32), c.run().result().view(np.uint32))
    for c, g, *_ in calls:
        dev.graph_destroy(g)
        c.free()


def test_offsets_past_32_bits(dev):
    """A cache whose pages lie past 4 GB."""
    say("large")
    rng = np.random.default_rng(9)
    cache = K.Kv4Cache(rng, 1, 8, 128, [200])
    q = act_to_f32(f32_to_act(rng.standard_normal((1, 2, 8, 128), dtype=np.float32), BF16), BF16)
    c = K.Call(dev, cache, q, BF16, 8, [198], 2, 0, 0, 0.09)
    want = c.run().result()
    block = 640 * 4 * 8
    n_pages = (5 << 30) // block
    pool = dev.alloc(n_pages * block)
    used = [int(p) for p in cache.table[0] if p >= 0]
    for i, p in enumerate(used):
        dev.write(pool, cache.pool.words[0, p], (n_pages - 1 - i) * block)
    table = np.full_like(cache.table, -1)
    table[0, :len(used)] = n_pages - 1 - np.arange(len(used))
    dev.write(c.bufs[1], table)
    c.kv.pool, c.kv.n_pages = int(pool), n_pages
    assert np.array_equal(want.view(np.uint32), c.run().result().view(np.uint32))
    pool.free()
    c.free()
