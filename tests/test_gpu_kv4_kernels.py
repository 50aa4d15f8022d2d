"""Every kernel of opure_attn_kv4_paged, asked for by name and not by the shape that would
choose it: every head size and format, one block of query rows and several, one part and
several, ragged batches with empty sequences, and all that the masks, pages, queries and
scores of the other tests hold."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as K
import opure_hip as H
import test_gpu_kv4_attn as A
import test_gpu_kv4_scores as S
from gpu_util import say
from npref import act_to_f32, f32_to_act

pytestmark = pytest.mark.gpu

F32, F16, BF16 = H.A_F32, H.A_F16, H.A_BF16
FORMATS = pytest.mark.parametrize("afmt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
KERNELS = {"one": H.KV4_ONE, "split": H.KV4_SPLIT, "pieces": H.KV4_PIECES, "rows": H.KV4_ROWS}


@pytest.fixture(scope="module")
def handle():
    d = H.Dev(0)
    yield d
    d.close()


@pytest.fixture
def dev(handle):
    yield handle
    force(handle, H.KV4_BEST)


def force(dev, kernels):
    H.check(H.lib().opure_debug_set_kv4_kernels(dev.h, kernels))


def taken(dev, call):
    """(kernels, parts) of a call, or None where its shape does not allow those asked for."""
    k, n = C.c_uint32(), C.c_uint32()
    rc = H.lib().opure_debug_kv4_kernels(dev.h, C.byref(call.args), C.byref(k), C.byref(n))
    if rc == H.E_UNSUPPORTED:
        assert H.lib().opure_attn_kv4_paged(dev.h, C.byref(call.args)) == rc
        return None
    H.check(rc)
    return k.value, n.value


def each(dev, afmt, heads, n_kv, hd, seq, rows, window, sinks, kernels, seed, spread=1.5, max_ctx=None):
    """A call through each of the kernels, which are held to one reference; the parts that each took."""
    rng = np.random.default_rng(seed)
    cache = K.Kv4Cache(rng, 1, n_kv, hd, [n + rows for n in seq], cap=max_ctx)
    q = act_to_f32(f32_to_act(rng.standard_normal((len(seq), rows, heads, hd), dtype=np.float32) * np.float32(spread), afmt), afmt)
    want = K.attention(cache, 0, q, afmt, heads, seq, rows, window, sinks, hd ** -0.5)
    c = K.Call(dev, cache, q, afmt, heads, seq, rows, window, sinks, hd ** -0.5, max_ctx=max_ctx)
    parts = {}
    for name in kernels:
        say("  through", name)
        force(dev, KERNELS[name])
        got = taken(dev, c)
        if got is None:
            assert name == "pieces" and heads // n_kv * rows > 16
            continue
        assert got[0] == KERNELS[name]
        parts[name] = got[1]
        dev.fill_u32(c.out, 0x7FC07FC0, q.size // (1 if afmt == F32 else 2))
        out = c.run().result()
        A.compare(out, *want)
        assert np.array_equal(out.view(np.uint32), c.run().result().view(np.uint32))
    c.free()
    return parts


SHAPES = {  # sequences, rows, heads, KV heads, the parts that it has at least and at most through each of the kernels
    "few-rows": ([700, 0, 130, 333, 5], 2, 6, 2, dict(one=(1, 1), split=(2, 64), pieces=(10, 4096), rows=(2, 64))),
    "16-rows": ([211, 3], 4, 4, 1, dict(one=(1, 1), split=(2, 64), pieces=(4, 4096), rows=(1, 1))),
    "short-blocks": ([90, 0], 70, 4, 2, dict(one=(1, 1), split=(1, 64), rows=(1, 1))),           # 140 query rows a KV head: 2 of 128, 5 of 32, 9 of 16
    "long-blocks": ([1000, 64], 50, 8, 2, dict(one=(1, 1), split=(1, 64), rows=(2, 64))),         # 200
}


@FORMATS
@pytest.mark.parametrize("hd", list(range(16, 257, 16)))
@pytest.mark.parametrize("shape", SHAPES)
def test_every_kernel(dev, shape, hd, afmt):
    seq, rows, heads, n_kv, parts = SHAPES[shape]
    window, sinks = ((0, 0), (77, 6))[(hd // 16 + afmt) % 2]
    say("every kernel", shape, hd, afmt, window)
    got = each(dev, afmt, heads, n_kv, hd, seq, rows, window, sinks, KERNELS, hd)
    for name, (least, most) in parts.items():
        assert (least if not window else 1) <= got[name] <= most, (name, got[name])


@pytest.mark.parametrize("seed", range(40))
def test_shapes_at_random(dev, seed):
    """Through every kernel that the shape allows."""
    r = np.random.default_rng(2000 + seed)
    n_kv, G = int(r.choice([1, 2, 3, 5, 8])), int(r.choice([1, 2, 3, 4, 7, 8]))
    afmt, hd = int(r.integers(0, 3)), 16 * int(r.integers(1, 17))
    rows = int(r.choice([1, 1, 2, 3, 5, 16, 33, 70, 150]))
    batch = int(r.integers(1, 40)) if rows < 5 else int(r.integers(1, 4))
    most = int(2 ** r.uniform(3, 10.5))
    seq = [int(r.integers(0, most)) for _ in range(batch)]
    window, sinks = int(r.choice([0, 0, 1, 15, 16, 63, 64, int(2 ** r.uniform(0, 10))])), int(r.choice([0, 0, 1, 4, 16, 33, 200]))
    say("random", seed, afmt, n_kv, G, hd, seq, rows, window, sinks)
    each(dev, afmt, n_kv * G, n_kv, hd, seq, rows, window, sinks, KERNELS, seed, max_ctx=max(seq) + rows + int(r.choice([0, 0, 7, 500])))


@FORMATS
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 40), (33, 16), (1000, 3)])
def test_pieces_of_ragged_batches(dev, window, sinks, afmt):
    """Pieces that hold the end of a sequence, whole ones and the begin of one; 256 sequences; one."""
    say("pieces", afmt, window, sinks)
    rng = np.random.default_rng(5)
    for hd, seq, rows in ((64, [0, 0, 900, 1, 15, 16, 17, 31, 32, 33, 0, 450], 1), (48, [int(n) for n in rng.integers(0, 100, 256)], 1),
                          (128, [1500], 3), (160, [5, 0, 700, 0, 64], 2)):
        got = each(dev, afmt, 4, 2, hd, seq, rows, window, sinks, ["pieces", "split"], hd)
        assert "pieces" in got


MASKED = {"one": [(6, 20, 3), (70, 33, 2)], "split": [(6, 20, 3), (70, 33, 2)], "pieces": [(6, 20, 3)], "rows": [(6, 20, 3), (70, 33, 2)]}


@FORMATS
@pytest.mark.parametrize("name", KERNELS)
def test_what_rows_do_not_see(dev, name, afmt):
    """NaN in masked slots, missing pages, queries that are not finite: the other test's cases through each kernel."""
    say("unseen", name, afmt)
    force(dev, KERNELS[name])
    for rows, window, sinks in MASKED[name]:
        A.test_masked_positions_may_hold_anything(dev, afmt, rows, window, sinks)
    A.test_queries_that_are_not_finite(dev, afmt)


def numbers_not_finite(dev, hd, afmt, rows, window, sinks):
    """V of one KV head and K of the other with a group of NaN where some rows see it, missing pages where none does."""
    rng = np.random.default_rng(hd)
    n0 = 300
    cache = K.Kv4Cache(rng, 1, 2, hd, [n0 + rows])
    for t in (n0 - window + 1, n0 + rows - 1):
        k, v = (rng.standard_normal((1, 2, hd)).astype(np.float32) for _ in range(2))
        v[0, 0, hd - 1], k[0, 1, 3] = np.nan, np.inf
        cache.put(0, [t], 0, 0, k)
        cache.put(0, [t], 0, 1, v)
    q = act_to_f32(f32_to_act(rng.standard_normal((1, rows, 4, hd), dtype=np.float32), afmt), afmt)
    want = K.attention(cache, 0, q, afmt, 4, [n0], rows, window, sinks, 0.1)
    cache.table[0, (sinks + 15) // 16:(n0 - window + 1) // 16] = -1
    c = K.Call(dev, cache, q, afmt, 4, [n0], rows, window, sinks, 0.1)
    got = c.run().result()
    A.compare(got, *want)
    assert np.isnan(got).any() and np.isfinite(got).any()
    c.free()


@FORMATS
@pytest.mark.parametrize("hd", [16, 48, 128, 144, 256])
@pytest.mark.parametrize("name", KERNELS)
def test_numbers_not_finite_at_head_sizes(dev, name, hd, afmt):
    say("not finite", name, hd, afmt)
    force(dev, KERNELS[name])
    numbers_not_finite(dev, hd, afmt, 6, 50, 3)
    if name != "pieces":
        numbers_not_finite(dev, hd, afmt, 68, 90, 20)


@pytest.mark.parametrize("name", KERNELS)
def test_pages_and_lengths(dev, name):
    """Missing pages that rows see, lengths past the capacity, pages past 4 GB."""
    say("pages", name)
    force(dev, KERNELS[name])
    for rows in (1, 4) + ((60,) if name != "pieces" else ()):
        A.test_pages_that_are_missing(dev, rows)
    A.test_lengths_past_the_capacity(dev)
    A.test_offsets_past_32_bits(dev)


@pytest.mark.parametrize("name", KERNELS)
def test_scales_and_queries(dev, name):
    """Scales of either sign and 0, rows far from 1."""
    say("scales", name)
    force(dev, KERNELS[name])
    for scale in (0.0, -0.11, 3.0):
        A.test_scales(dev, 2, 700, scale)
        if name != "pieces":
            A.test_scales(dev, 90, 20, scale)
    for spread in (1e-20, 30.0, 1e20):
        A.test_query_magnitudes(dev, spread)


@FORMATS
@pytest.mark.parametrize("hd", [32, 80, 128, 208])
@pytest.mark.parametrize("name", KERNELS)
def test_large_scores(dev, name, hd, afmt):
    """Exact scores up to fp32's largest, in a ragged batch and in one part and several."""
    say("scores", name, hd, afmt)
    force(dev, KERNELS[name])
    S.check(dev, afmt, 4, 2, hd, [90, 0, 260], 6, positive=True, sizes=S.SIZES[1::2])
    S.check(dev, afmt, 4, 2, hd, [700], 3, 200, 3, sizes=S.SIZES[::2], seed=1)
    if name != "pieces":
        S.check(dev, afmt, 4, 2, hd, [40], 70, sizes=S.SIZES[2::3], seed=2)


@pytest.mark.parametrize("name", KERNELS)
def test_capture_and_replay(dev, name):
    """Two captured shapes share the workspace; lengths change between replays."""
    say("graph", name)
    force(dev, KERNELS[name])
    rng = np.random.default_rng(8)
    cache = K.Kv4Cache(rng, 1, 2, 64, [900, 500])
    calls = []
    for afmt, rows in ((F16, 1), (BF16, 4 if name == "pieces" else 40)):
        q = act_to_f32(f32_to_act(rng.standard_normal((2, rows, 8, 64), dtype=np.float32), afmt), afmt)
        c = K.Call(dev, cache, q, afmt, 8, [800, 400], rows, 0, 0, 0.125, max_ctx=900)
        H.check(H.lib().opure_attn_kv4_reserve(dev.h, C.byref(c.args)))
        dev.graph_begin()
        c.run(sync=False)
        calls.append((c, dev.graph_end(), q, afmt, rows))
    for seq in ([800, 400], [10, 0], [860, 460], [333, 100]):
        for c, g, q, afmt, rows in calls:
            dev.write(c.bufs[2], np.array(seq, np.int32))
            dev.graph_launch(g)
        dev.sync()
        for c, g, q, afmt, rows in calls:
            got = c.result()
            A.compare(got, *K.attention(cache, 0, q, afmt, 8, seq, rows, 0, 0, 0.125))
            assert np.array_equal(got.view(np.uint32), c.run().result().view(np.uint32))
    for c, g, *_ in calls:
        dev.graph_destroy(g)
        c.free()


def test_what_shapes_choose(dev):
    """Without being asked for, each is what some shape takes."""
    force(dev, H.KV4_BEST)
    got = set()
    for heads, n_kv, batch, rows, ctx in ((8, 2, 1, 1, 100), (8, 2, 1, 1, 8000), (32, 8, 32, 1, 16384), (32, 8, 1, 256, 8000), (64, 16, 2, 100, 1000)):
        m = H.Model()
        m.n_layers, m.n_heads, m.n_kv_heads, m.head_dim, m.afmt = 1, heads, n_kv, 64, F16
        kv = H.KV(1 << 40, 4, H.PAGE_SIZE, 1 << 41, 4096)
        a = H.AttnKv4Args(C.pointer(m), C.pointer(kv), 0, batch, rows, None, ctx, 0, 0, None, None)
        k, n = C.c_uint32(), C.c_uint32()
        H.check(H.lib().opure_debug_kv4_kernels(dev.h, C.byref(a), C.byref(k), C.byref(n)))
        got.add((k.value, n.value > 1))
    assert got == {(H.KV4_ONE, False), (H.KV4_SPLIT, True), (H.KV4_PIECES, True), (H.KV4_ROWS, True), (H.KV4_ROWS, False)}, got
