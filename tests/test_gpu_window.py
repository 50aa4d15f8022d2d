"""opure_attn_window_paged against its definition in 64 bits: every format, head
size and layout, one row to a prompt's, windows and sinks of any length, what is
masked holding NaN, the accumulated weights, capture and replay."""
import ctypes as C

import numpy as np
import pytest

import opure_hip as H
import window_ref as R
from gpu_util import say

pytestmark = pytest.mark.gpu

F32, F16, BF16 = H.A_F32, H.A_F16, H.A_BF16


@pytest.fixture(scope="module")
def dev():
    d = H.Dev(0)
    yield d
    d.close()


def check(dev, afmt, heads, n_kv, hd, seq, rows, window, sinks, weights=False, layers=1, seed=0, edit=None, spread=1.5, max_ctx=None, scale=None):
    rng = np.random.default_rng(seed)
    layer = layers - 1
    cache = R.Cache(rng, afmt, layers, n_kv, hd, [n + rows for n in seq], cap=max_ctx)
    q = R.act_to_f32(R.f32_to_act(rng.standard_normal((len(seq), rows, heads, hd), dtype=np.float32) * np.float32(spread), afmt), afmt)
    if edit:
        edit(cache, q)
    scale = hd ** -0.5 if scale is None else scale
    cap = max_ctx or max(seq) + rows
    w0 = rng.random((len(seq), layers, n_kv, cap + 5), dtype=np.float32) if weights else None
    c = R.Call(dev, cache, q, heads, seq, rows, window, sinks, scale, layer, cap, w0)
    if weights:
        c.args.weights = int(c.weights) + layer * n_kv * (cap + 5) * 4
    c.run()
    got = c.result().astype(np.float64)
    ref, tol, ws, wt = R.attention(cache, layer, q, heads, seq, rows, window, sinks, scale)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    assert np.array_equal(np.isinf(got), np.isinf(ref)) and np.array_equal(got[np.isinf(ref)], ref[np.isinf(ref)])
    with np.errstate(invalid="ignore"):
        off = np.where(np.isfinite(ref), np.abs(got - ref) - tol, 0)
    assert not np.isnan(off).any() and not (off > 0).any(), (float(np.nanmax(off)), float(np.nanmax(np.abs(got - ref))), np.argwhere(off > 0)[:4])
    if weights:
        sums = c.sums()
        want = w0.astype(np.float64).copy()
        for b, n in enumerate(seq):
            want[b, layer, :, :n + rows] += ws[b]
        bound = np.zeros_like(want)
        for b, n in enumerate(seq):
            bound[b, layer, :, :n + rows] = wt[b] + 2.0 ** -23 * want[b, layer, :, :n + rows]
        assert np.array_equal(np.isnan(sums), np.isnan(want))
        fine = np.isfinite(want)
        assert not np.isnan(bound[fine]).any()
        assert not (np.abs(sums - want)[fine] > bound[fine]).any(), float(np.max((np.abs(sums - want) - bound)[fine]))
    first = c.result()
    if weights:
        c.dev.write(c.weights, w0)
    c.run()
    assert np.array_equal(first.view(np.uint32), c.result().view(np.uint32))     # the same call, the same bits
    if weights:
        assert np.array_equal(sums.view(np.uint32), c.sums().view(np.uint32))
    c.free()
    return got


@pytest.mark.parametrize("weights", [False, True], ids=["", "weights"])
@pytest.mark.parametrize("afmt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", list(range(16, 257, 16)))
def test_head_sizes(dev, hd, afmt, weights):
    say("head size", hd, afmt, weights)
    check(dev, afmt, 6, 2, hd, [0, 37, 150], 3, 50, 5, weights, seed=hd)


SHAPES = {  # sequences, rows, heads: every way a call is run, at every head size
    "one-block": ([900, 3, 511], 3, 6),                  # up to 16 query rows a KV head over a long cache
    "two-blocks": ([1200, 40], 12, 6),                   # 36: blocks of 32
    "prompt": ([70], 130, 4),                            # 260 over a short one
    "wide": ([30, 0, 64, 5] * 20, 70, 8),                # 280 in 80 sequences: more workgroups than the device has CUs
}


@pytest.mark.parametrize("shape,afmt,weights", [(s, f, w) for s in SHAPES for f in (F32, F16, BF16) for w in (False, True)
                                                if s != "wide" or not (w or f == F32)])   # there, as the prompt's
@pytest.mark.parametrize("hd", list(range(16, 257, 16)))
def test_every_kernel(dev, shape, hd, afmt, weights):
    seq, rows, heads = SHAPES[shape]
    say("kernel", shape, hd, afmt, weights)
    check(dev, afmt, heads, 2, hd, seq, rows, 333 if shape != "wide" else 40, 6, weights, seed=hd)


@pytest.mark.parametrize("scale", [0.0, -0.11, 1.0, 3.0])
@pytest.mark.parametrize("rows,n", [(2, 700), (90, 20)])
def test_scales(dev, rows, n, scale):
    """attn_scale of either sign, and 0, where every visible position weighs the same."""
    say("scale", scale, rows)
    for afmt in (F32, F16, BF16):
        check(dev, afmt, 4, 2, 64, [n], rows, 50, 3, True, seed=rows, spread=0.3, scale=scale)


@pytest.mark.parametrize("seed", range(60))
def test_shapes_at_random(dev, seed):
    r = np.random.default_rng(1000 + seed)
    n_kv, G = int(r.choice([1, 2, 3, 5, 8])), int(r.choice([1, 2, 3, 4, 7, 8]))
    afmt, hd = int(r.integers(0, 3)), 16 * int(r.integers(1, 17))
    rows = int(r.choice([1, 1, 2, 5, 9, 16, 33, 70, 150]))
    batch = int(r.integers(1, 6)) if rows < 33 else int(r.integers(1, 3))
    most = int(2 ** r.uniform(3, 11))
    seq = [int(r.integers(0, most)) for _ in range(batch)]
    window, sinks = int(r.choice([0, 1, 15, 16, 63, 64, int(2 ** r.uniform(0, 11))])), int(r.choice([0, 0, 1, 4, 16, 33, 200]))
    say("random", seed, afmt, n_kv, G, hd, seq, rows, window, sinks)
    check(dev, afmt, n_kv * G, n_kv, hd, seq, rows, window, sinks, bool(r.integers(0, 2)), seed=seed,
          max_ctx=max(seq) + rows + int(r.choice([0, 0, 7, 500])))


def test_most_sequences(dev):
    rng = np.random.default_rng(12)
    check(dev, F16, 8, 2, 64, [int(n) for n in rng.integers(0, 400, 256)], 1, 100, 4, True)
    check(dev, BF16, 4, 1, 32, [int(n) for n in rng.integers(0, 60, 256)], 3, 0, 0, False)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (1, 40), (7, 0), (16, 4), (17, 3), (33, 16), (64, 70), (100, 0), (129, 33),
                                          (400, 2), (0, 0), (0, 9), (1 << 31, 5), (0xFFFFFFFF, 0xFFFF)])
@pytest.mark.parametrize("rows", [1, 5, 40])
def test_windows(dev, rows, window, sinks):
    say("window", rows, window, sinks)
    check(dev, BF16 if rows == 5 else F16, 8, 2, 64, [0, 1, 15, 16, 200, 333], rows, window, sinks, True, seed=rows)
    check(dev, F32, 3, 3, 32, [0, 15, 131], rows, window, sinks, True, seed=rows)


@pytest.mark.parametrize("heads,n_kv", [(1, 1), (7, 1), (9, 3), (16, 2), (40, 8), (5, 5), (33, 1)])
@pytest.mark.parametrize("rows", [1, 4, 16, 23])
def test_layouts(dev, heads, n_kv, rows):
    say("layout", heads, n_kv, rows)
    check(dev, F16, heads, n_kv, 64, [3, 77, 260], rows, 96, 4, rows % 2 == 0, layers=2, seed=heads)
    check(dev, BF16, heads, n_kv, 128, [90], rows, 41, 2, rows % 2 == 1, layers=3, seed=heads)


@pytest.mark.parametrize("afmt,hd", [(F16, 64), (BF16, 128), (F16, 96), (BF16, 80), (F32, 64), (F16, 256), (BF16, 16)])
@pytest.mark.parametrize("rows,start,window,sinks", [(17, 0, 0, 0), (130, 0, 50, 4), (333, 0, 0, 0), (200, 517, 128, 4), (260, 90, 1, 0),
                                                     (129, 700, 300, 70), (65, 64, 0, 0)])
def test_prompts(dev, afmt, hd, rows, start, window, sinks):
    say("prompt", afmt, hd, rows, start, window, sinks)
    check(dev, afmt, 8, 2, hd, [start], rows, window, sinks, True, seed=rows)
    check(dev, afmt, 8, 2, hd, [start, start // 2], rows, window, sinks, False, seed=rows + 1)


@pytest.mark.parametrize("afmt,hd,rows,n", [(F16, 64, 1, 5000), (BF16, 128, 2, 3000), (F32, 64, 1, 2500), (F16, 64, 1500, 600)])
def test_long(dev, afmt, hd, rows, n):
    """Caches and prompts long enough for every way of splitting the work; a
    spread of scores that a few positions dominate."""
    say("long", afmt, hd, rows, n)
    check(dev, afmt, 4, 1, hd, [n], rows, 0, 0, True, seed=n, spread=6.0)
    check(dev, afmt, 4, 1, hd, [n], rows, 1031, 4, True, seed=n + 1, spread=6.0)
    check(dev, afmt, 8, 2, hd, [n, n // 7, 9], rows, 700, 20, False, seed=n + 2)


@pytest.mark.parametrize("afmt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,window,sinks", [(6, 20, 3), (70, 33, 2)])
def test_masked_positions_may_hold_anything(dev, afmt, rows, window, sinks):
    """NaN and infinities at positions that some rows see and others do not: the
    rows that do not see them are not touched by them."""
    say("masked", afmt, rows)
    n0 = 100

    def edit(cache, q):
        rng = np.random.default_rng(1)
        n = n0 + rows
        for t, value in ((n0 + 2, np.nan), (n0 - window + 1, np.inf), (n0 + rows - 2, -np.inf)):
            x = rng.standard_normal((1, 2, cache.n_kv, 1, cache.hd)).astype(np.float32)
            x[0, 1, 0, 0, 5] = value                        # V of one KV head
            x[0, 0, 1, 0, 3] = value                        # K of the other
            cache.put(0, [t], x)
        # positions between the sinks and every window: nothing of them is read
        hidden = np.arange(sinks, n0 - window)
        cache.put(0, hidden, np.full((1, 2, cache.n_kv, len(hidden), cache.hd), np.nan, np.float32))

    # spread 0.5: an infinite score of either sign is a definite value on both sides
    got = check(dev, afmt, 4, 2, 64, [n0], rows, window, sinks, True, edit=edit, spread=0.5)
    assert np.isfinite(got).any() and not np.isfinite(got).all()


@pytest.mark.parametrize("afmt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [2, 50])
def test_rows_of_infinite_scores(dev, afmt, rows):
    """Every visible score -inf: the row gives 0 and its positions get nothing."""
    say("-inf rows", afmt, rows)

    def edit(cache, q):
        q[...] = np.abs(q) + 0.25
        n = 40 + rows
        x = np.random.default_rng(2).standard_normal((1, 2, 1, n, 64)).astype(np.float32)
        x[0, 0] = -np.inf
        cache.put(0, slice(0, n), x)

    q = check(dev, afmt, 3, 1, 64, [40], rows, 24, 3, True, edit=edit)
    assert (q == 0).all()


@pytest.mark.parametrize("afmt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 4, 90])
def test_released_pages(dev, afmt, rows):
    """Pages that no row sees may be missing; a missing page that a row sees makes
    that row NaN and no other."""
    say("released", afmt, rows)
    window, sinks, n0 = 30, 3, 200

    def edit(cache, q):
        cache.table[0, 1:(n0 - window + 1) // 16] = -1

    check(dev, afmt, 4, 2, 64, [n0, 10], rows, window, sinks, rows == 4, edit=edit)

    rng = np.random.default_rng(4)
    cache = R.Cache(rng, afmt, 1, 2, 64, [n0 + rows])
    q = rng.standard_normal((1, rows, 4, 64), dtype=np.float32)
    q = R.act_to_f32(R.f32_to_act(q, afmt), afmt)
    ref = R.attention(cache, 0, q, 4, [n0], rows, window, sinks, 0.125)
    gone = n0 // 16                                         # positions 192 .. 207
    for value in (-1, cache.n_pages, 1 << 30):
        cache.table[0, gone] = value
        c = R.Call(dev, cache, q, 4, [n0], rows, window, sinks, 0.125).run()
        got = c.result()
        c.free()
        touched = R.sees(n0, rows, n0 + rows, window, sinks)[:, gone * 16:gone * 16 + 16].any(1)
        assert np.isnan(got[0, touched]).all()
        assert (np.abs(got[0, ~touched] - ref[0][0, ~touched]) <= ref[1][0, ~touched]).all()


@pytest.mark.parametrize("rows", [1, 16, 100])
def test_positions_past_the_capacity(dev, rows):
    """A length past max_ctx or below zero is reported at the next sync, and the
    device goes on; weights past max_ctx stay."""
    say("capacity", rows)
    rng = np.random.default_rng(5)
    cache = R.Cache(rng, F16, 1, 2, 64, [300], cap=300)
    q = rng.standard_normal((1, rows, 4, 64), dtype=np.float32)
    for seq, max_ctx in (([250], 120), ([5000], 300), ([2 ** 31 - 1], 300), ([-1], 300), ([-2 ** 31], 300)):
        w = np.zeros((1, 1, 2, 400), np.float32)
        c = R.Call(dev, cache, q, 4, seq, rows, 0, 0, 0.125, max_ctx=max_ctx, weights=w)
        with pytest.raises(H.OpureError) as e:
            c.run()
        assert e.value.code == H.E_CAPACITY
        assert (c.sums()[..., max_ctx:] == 0).all()
        c.free()
    check(dev, F16, 4, 2, 64, [100], rows, 0, 0)


def test_agrees_with_decode_attention(dev):
    """No window: the same as opure_attn_decode_paged, to the bounds of both."""
    rng = np.random.default_rng(6)
    for afmt, hd in ((F32, 64), (F16, 64), (BF16, 128), (F16, 96)):
        seq, rows = [5, 400, 77], 4
        cache = R.Cache(rng, afmt, 1, 2, hd, [n + rows for n in seq])
        q = R.act_to_f32(R.f32_to_act(rng.standard_normal((3, rows, 8, hd), dtype=np.float32), afmt), afmt)
        c = R.Call(dev, cache, q, 8, seq, rows, 0, 0, hd ** -0.5).run()
        a = c.result()
        d = H.AttnArgs(c.args.model, c.args.kv, 0, 3, rows, c.args.seq_len, c.args.max_ctx, c.args.q, c.args.out)
        H.check(H.lib().opure_attn_decode_paged(dev.h, C.byref(d)))
        dev.sync()
        tol = R.attention(cache, 0, q, 8, seq, rows, 0, 0, hd ** -0.5)[1]
        assert (np.abs(a - c.result()) <= 2 * tol).all()
        c.free()


@pytest.mark.parametrize("rows,weights", [(1, True), (5, True), (5, False), (80, True), (80, False)])
def test_captured_and_replayed(dev, rows, weights):
    """Captured once, replayed several times with eager calls of another shape and
    new inputs between: every replay has the eager call's bits."""
    say("graph", rows, weights)
    rng = np.random.default_rng(7)
    seq = [300, 31]
    cache = R.Cache(rng, BF16, 1, 2, 128, [n + rows for n in seq])
    w0 = np.zeros((2, 1, 2, 300 + rows), np.float32) if weights else None

    def fresh():
        return rng.standard_normal((2, rows, 8, 128), dtype=np.float32)

    q = fresh()
    c = R.Call(dev, cache, q, 8, seq, rows, 100, 4, 0.09, weights=w0)
    other = R.Call(dev, cache, fresh(), 8, seq, rows, 60, 2, 0.09, weights=w0)
    H.check(H.lib().opure_attn_window_reserve(dev.h, C.byref(c.args)))
    dev.graph_begin()
    c.run(sync=False)
    g = dev.graph_end()
    dev.graph_begin()
    other.run(sync=False)
    g2 = dev.graph_end()
    for k in range(4):
        q = fresh()
        dev.write(c.bufs[3], R.f32_to_act(q, BF16))
        if weights:
            dev.write(c.weights, w0)
        dev.graph_launch(g2)
        dev.graph_launch(g)
        dev.sync()
        got, sums = c.result(), c.sums() if weights else None
        check(dev, F16, 4, 2, 64, [500 + 200 * k], 3, 0, 0, True, seed=k)      # may replace the workspace
        if weights:
            dev.write(c.weights, w0)
        c.run()
        assert np.array_equal(got.view(np.uint32), c.result().view(np.uint32))
        if weights:
            assert np.array_equal(sums, c.sums())
    dev.graph_destroy(g)
    dev.graph_destroy(g2)
    c.free()
    other.free()


def test_two_handles_at_once(dev):
    """Calls of two device handles, queued without waiting, each with its own workspace."""
    rng = np.random.default_rng(8)
    second = H.Dev(0)
    calls = []
    for d in (dev, second):
        cache = R.Cache(rng, F16, 1, 8, 64, [3000])
        q = R.act_to_f32(R.f32_to_act(rng.standard_normal((1, 1, 32, 64), dtype=np.float32), F16), F16)
        calls.append((R.Call(d, cache, q, 32, [2999], 1, 0, 0, 0.125, weights=np.zeros((1, 1, 8, 3000), np.float32)), cache, q))
    for _ in range(5):
        for c, _, _ in calls:
            c.run(sync=False)
    for d in (dev, second):
        d.sync()
    for c, cache, q in calls:
        ref, tol, ws, wt = R.attention(cache, 0, q, 32, [2999], 1, 0, 0, 0.125)
        assert (np.abs(c.result() - ref) <= tol).all()
        assert (np.abs(c.sums()[0, 0] - 5 * ws[0]) <= 5 * wt[0] + 2.0 ** -21 * ws[0]).all()
        c.free()
    second.close()


def test_offsets_past_32_bits(dev):
    """A pool whose last pages lie past 2^32 bytes (and elements)."""
    rng = np.random.default_rng(9)
    heads, n_kv, hd, rows, n = 8, 8, 128, 3, 90
    cache = R.Cache(rng, F16, 1, n_kv, hd, [n + rows])
    page_bytes = 2 * n_kv * 16 * hd * 2
    big = (5 << 31) // page_bytes                            # 10 GiB of pages
    pool = dev.alloc(big * page_bytes)
    first = big - cache.n_pages
    dev.write(pool, cache.pool, first * page_bytes)
    q = R.act_to_f32(R.f32_to_act(rng.standard_normal((1, rows, heads, hd), dtype=np.float32), F16), F16)
    c = R.Call(dev, cache, q, heads, [n], rows, 40, 4, 0.09, weights=np.zeros((1, 1, n_kv, n + rows), np.float32))
    table = np.where(cache.table >= 0, cache.table + first, -1).astype(np.int32)
    dev.write(c.bufs[1], table)
    c.kv.pool, c.kv.n_pages = int(pool), big
    c.run()
    ref, tol, ws, wt = R.attention(cache, 0, q, heads, [n], rows, 40, 4, 0.09)
    assert (np.abs(c.result() - ref) <= tol).all()
    assert (np.abs(c.sums()[0, 0] - ws[0]) <= wt[0] + 2.0 ** -23 * ws[0]).all()
    c.free()
    pool.free()
