"""What opure_attn_window_paged promises beyond its definition's values: weights
that meet V with their rounding's rest, in every kernel."""
import ctypes as C

import numpy as np
import pytest

import opure_hip as H
import window_ref as R
from gpu_util import say
from test_gpu_window import check

pytestmark = pytest.mark.gpu

F32, F16, BF16 = H.A_F32, H.A_F16, H.A_BF16


@pytest.fixture(scope="module")
def dev():
    d = H.Dev(0)
    yield d
    d.close()


def sizes(cache, seq, q, heads, rows, window, sinks, scale):
    """Sum of w |v| of every output and sum of |v| over what its row sees, in 64 bits."""
    G = heads // cache.n_kv
    mag, flat = np.zeros(q.shape), np.zeros(q.shape)
    for b, n0 in enumerate(seq):
        n = n0 + rows
        m = R.sees(n0, rows, n, window, sinks)
        for h in range(heads):
            k, v = (cache.get(b, 0, h // G, i, n).astype(np.float64) for i in (0, 1))
            s = np.where(m, q[b, :, h].astype(np.float64) @ k.T * scale, -np.inf)
            e = np.exp(s - s.max(1, keepdims=True))
            mag[b, :, h] = e / e.sum(1, keepdims=True) @ np.abs(v)
            flat[b, :, h] = m @ np.abs(v)
    return mag, flat


# rows, sequences, window, and which positions' V are not 0 (about twelve a window, so that
# roundings of single weights show): 4 query rows a KV head and 36 behind a long window, a
# prompt of few workgroups and of many
KERNELS = {"decode": (1, [900, 1300, 750], 700, 60), "verify": (9, [900, 20], 700, 60), "prompt": (130, [50], 12, 1),
           "prompts": (260, [30, 5] * 20, 12, 1)}


@pytest.mark.parametrize("afmt,hd", [(F16, 64), (BF16, 64), (F16, 128), (BF16, 128), (F16, 80), (BF16, 208)])
@pytest.mark.parametrize("kernel", KERNELS)
def test_weights_keep_their_rest(dev, kernel, afmt, hd):
    """A weight of a 16-bit cache meets V as two numbers of its format: its rounding, off by
    at most half a step u, and the rest, rounded by as much: u^2 of the weight in all (and in
    fp16 half of the smallest step, 2^-25, where the row's largest weight is 1 or more).  So
    the bound of the definition's test without its one rounding of the weights."""
    rows, seq, window, every = KERNELS[kernel]
    say("rest", kernel, afmt, hd)
    rng = np.random.default_rng(hd + rows)
    heads, n_kv, sinks, scale = 8, 2, 2, hd ** -0.5
    cache = R.Cache(rng, afmt, 1, n_kv, hd, [n + rows for n in seq])
    for b, n in enumerate(seq):
        x = rng.standard_normal((1, 2, n_kv, n + rows, hd), dtype=np.float32)
        x[0, 1, :, np.arange(n + rows) % every != 0] = 0
        cache.put(b, slice(0, n + rows), x)
    q = R.act_to_f32(R.f32_to_act(rng.standard_normal((len(seq), rows, heads, hd), dtype=np.float32) * np.float32(0.5), afmt), afmt)
    ref, tol, _, _ = R.attention(cache, 0, q, heads, seq, rows, window, sinks, scale)
    mag, flat = sizes(cache, seq, q, heads, rows, window, sinks, scale)
    u = R.HALF_STEP[afmt]
    tol = tol - u * mag + u * u * mag + (2.0 ** -25 * flat if afmt == F16 else 0)
    c = R.Call(dev, cache, q, heads, seq, rows, window, sinks, scale).run()
    off = np.abs(c.result() - ref)
    c.free()
    assert not (off > tol).any(), (int((off > tol).sum()), float((off - tol).max()))


@pytest.mark.parametrize("afmt,heads,n_kv,hd", [(F16, 32, 8, 64), (BF16, 32, 8, 128), (F32, 9, 3, 64), (F16, 64, 8, 16)])
@pytest.mark.parametrize("batch,rows,ctx", [(1, 1, 131072), (16, 24, 16000), (256, 12, 2000), (64, 4, 16000), (4, 256, 30000), (1, 2048, 60000)])
def test_workspace_is_bounded(afmt, heads, n_kv, hd, batch, rows, ctx):
    """What a call with weights asks of the workspace: no more than the keys of its
    positions take in the layer, or 64 MiB, beside what it takes without weights."""
    say("workspace", afmt, heads, n_kv, hd, batch, rows, ctx)
    model = H.Model()
    model.n_layers, model.n_heads, model.n_kv_heads, model.head_dim, model.afmt, model.attn_scale = 1, heads, n_kv, hd, afmt, 0.1
    kv = H.KV(4096, 1 << 20, R.PAGE, 4096, (ctx + rows + 15) // 16)
    need = []
    for weights in (None, 4096):
        d = H.Dev(0)
        a = H.AttnWindowArgs(C.pointer(model), C.pointer(kv), 0, batch, rows, None, ctx + rows, 0, 0, None, None, weights, ctx + rows,
                             n_kv * (ctx + rows))
        H.check(H.lib().opure_attn_window_reserve(d.h, C.byref(a)))
        ptr, size = C.c_void_p(), C.c_uint64()
        H.check(H.lib().opure_debug_workspace(d.h, C.byref(ptr), C.byref(size)))
        need.append(size.value)
        d.close()
    eb = 4 if afmt == F32 else 2
    keys, q = batch * n_kv * (ctx + rows + 31) * hd * eb, batch * rows * heads * hd * 4
    assert need[0] <= max(64 << 20, 2 * q) + (1 << 20)
    assert need[1] <= max(64 << 20, 2 * q) + max(64 << 20, keys) + (1 << 20), (need[1] >> 20, keys >> 20)


def reserve(dev, afmt, heads, n_kv, hd, batch, rows, ctx, window=0, weights=True):
    model = H.Model()
    model.n_layers, model.n_heads, model.n_kv_heads, model.head_dim, model.afmt, model.attn_scale = 1, heads, n_kv, hd, afmt, 0.1
    kv = H.KV(4096, 1 << 20, R.PAGE, 4096, (ctx + 15) // 16)
    a = H.AttnWindowArgs(C.pointer(model), C.pointer(kv), 0, batch, rows, None, ctx, window, 0, None, None, 4096 if weights else None, ctx,
                         n_kv * ctx)
    return H.lib().opure_attn_window_reserve(dev.h, C.byref(a))


def test_large_calls_are_refused_where_a_launch_cannot_be(dev):
    """Launches of up to 2^24 workgroups are taken, larger ones refused."""
    say("large calls")
    assert reserve(dev, F16, 32, 8, 64, 32, 2048, 32768) == H.OK       # 0.8 million workgroups
    assert reserve(dev, F16, 64, 8, 64, 256, 2048, 4096, 512, False) == H.OK
    assert reserve(dev, F16, 64, 8, 64, 256, 2048, 65536) == H.E_CAPACITY
    assert b"workgroups" in H.lib().opure_last_error()
    assert reserve(dev, F16, 65, 5, 64, 256, 2048, 4096, 512, False) == H.E_CAPACITY


def test_more_than_four_million_workgroups(dev):
    """A max_ctx of 2^26 for 4,800 query rows: 2^22 workgroups over the positions, of which a few have any."""
    say("2^22 workgroups")
    check(dev, F16, 16, 1, 32, [50], 300, 100, 3, True, max_ctx=1 << 26)


@pytest.mark.parametrize("captured", [False, True])
def test_a_workspace_that_cannot_be_had(captured):
    """A call whose workspace is larger than the memory (scores of 2^33 positions, 512 GiB) is
    OPURE_E_OOM; the handle keeps the workspace that it had, and its next calls run."""
    say("no room", captured)
    d = H.Dev(0)
    rng = np.random.default_rng(3)
    cache = R.Cache(rng, F16, 1, 2, 64, [500])
    q = R.act_to_f32(R.f32_to_act(rng.standard_normal((1, 1, 8, 64), dtype=np.float32), F16), F16)
    c = R.Call(d, cache, q, 8, [499], 1, 0, 0, 0.125, weights=np.zeros((1, 1, 2, 500), np.float32)).run()
    first, size, ptr, after = c.result(), C.c_uint64(), C.c_void_p(), C.c_uint64()
    H.check(H.lib().opure_debug_workspace(d.h, C.byref(ptr), C.byref(size)))
    if captured:
        d.graph_begin()
        c.run(sync=False)
        g = d.graph_end()
    for _ in range(2):
        assert reserve(d, F16, 128, 32, 64, 256, 4, 1 << 20) == H.E_OOM
        H.check(H.lib().opure_debug_workspace(d.h, C.byref(ptr), C.byref(after)))
        assert after.value == size.value and ptr.value
    if not captured:
        d.graph_begin()
        c.run(sync=False)                                   # no reserve in between
        g = d.graph_end()
    for run in (c.run, lambda: d.graph_launch(g)):
        d.write(c.out, np.zeros(first.size, np.uint16))
        run()
        d.sync()
        assert np.array_equal(first.view(np.uint32), c.result().view(np.uint32))
    d.graph_destroy(g)
    c.free()
    d.close()


@pytest.mark.parametrize("weights", [False, True], ids=["", "weights"])
@pytest.mark.parametrize("scale", [0.0, 0.125, -0.2])
@pytest.mark.parametrize("afmt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n", [(3, 900), (12, 900), (70, 40), (300, 10)])
def test_queries_that_are_not_finite(dev, rows, n, afmt, scale, weights):
    """NaN and infinities in a query are its own row's and head's: NaN there (also with a scale of 0), the others exact."""
    say("queries", rows, n, afmt, scale, weights)

    def edit(cache, q):
        q[0, 0, 0, 3], q[0, rows - 1, 1, 63], q[0, rows // 2, 2, 17] = np.nan, np.inf, -np.inf

    got = check(dev, afmt, 4, 2, 64, [n], rows, 600, 3, weights, seed=rows, edit=edit, spread=0.5, scale=scale)
    assert np.isnan(got[0, 0, 0]).all() and np.isfinite(got[0, :, 3]).all()
    if scale == 0:
        assert np.isnan(got[0, rows - 1, 1]).all() and np.isnan(got[0, rows // 2, 2]).all()


# batch, max_ctx, window: calls whose weights are added four positions a thread (at least two
# workgroups a CU of 1,024 positions): with up to 8 parts a KV head, and with more
FOUR = {"few parts": (64, 1111, 0), "windowed": (64, 3001, 1100), "many parts": (10, 7007, 0)}


@pytest.mark.parametrize("group,rows", [(3, 3), (5, 2), (1, 16), (17, 1), (7, 3)])
@pytest.mark.parametrize("afmt,hd", [(F32, 64), (F32, 128), (F32, 192), (F32, 256), (F16, 64), (BF16, 128), (F16, 192), (BF16, 256)])
@pytest.mark.parametrize("form", FOUR)
def test_weights_four_positions_a_thread(dev, form, afmt, hd, group, rows):
    """9 to 21 query rows a KV head: several turns of the eight that a workgroup adds at a time, the last one not full."""
    batch, cap, window = FOUR[form]
    say("four", form, afmt, hd, group, rows)
    rng = np.random.default_rng(hd + group)
    seq = [int(n) for n in rng.integers(0, 60, batch)]
    seq[3], seq[batch // 2] = cap - rows, cap // 3                # two long ones
    check(dev, afmt, 8 * group, 8, hd, seq, rows, window, 5 if window else 0, True, seed=hd, max_ctx=cap)


def test_weights_past_32_bits(dev):
    """Sums whose heads and sequences lie 2^31 and 2^32 elements apart."""
    say("weights past 32 bits")
    rng = np.random.default_rng(14)
    for rows, seq, heads in ((2, [300, 41], 4), (90, [33, 0], 4)):
        cache = R.Cache(rng, F16, 1, 2, 64, [n + rows for n in seq])
        q = R.act_to_f32(R.f32_to_act(rng.standard_normal((2, rows, heads, 64), dtype=np.float32), F16), F16)
        c = R.Call(dev, cache, q, heads, seq, rows, 50, 4, 0.125)
        stride, batch = (1 << 31) + 7, (1 << 32) + 1000
        far = dev.alloc((batch + stride + 1000) * 4)
        c.args.weights, c.args.weights_stride, c.args.weights_batch_stride = int(far), stride, batch
        ref, tol, ws, wt = R.attention(cache, 0, q, heads, seq, rows, 50, 4, 0.125)
        for b in range(2):
            for h in range(2):
                dev.write(far, np.zeros(1000, np.float32), (b * batch + h * stride) * 4)
        c.run()
        assert (np.abs(c.result() - ref) <= tol).all()
        for b, n in enumerate(seq):
            for h in range(2):
                got = dev.download(far, np.float32, (1000,), (b * batch + h * stride) * 4)
                assert (np.abs(got[:n + rows] - ws[b][h]) <= wt[b][h] + 2.0 ** -23 * ws[b][h]).all() and (got[n + rows:] == 0).all()
        c.free()
        far.free()


@pytest.mark.parametrize("what", ["q", "out", "weights"])
def test_buffers_in_the_workspace_are_refused(dev, what):
    """The call writes its parts there, and a larger one replaces it."""
    say("in the workspace", what)
    rng = np.random.default_rng(5)
    cache = R.Cache(rng, F16, 1, 2, 64, [700])
    q = R.act_to_f32(R.f32_to_act(rng.standard_normal((1, 1, 8, 64), dtype=np.float32), F16), F16)
    c = R.Call(dev, cache, q, 8, [699], 1, 0, 0, 0.125, weights=np.zeros((1, 1, 2, 700), np.float32)).run()
    ptr, size = C.c_void_p(), C.c_uint64()
    H.check(H.lib().opure_debug_workspace(dev.h, C.byref(ptr), C.byref(size)))
    for at in (ptr.value, ptr.value + size.value - 256):
        old = getattr(c.args, what)
        setattr(c.args, what, at)
        with pytest.raises(H.OpureError) as e:
            c.run()
        assert e.value.code == H.E_INVALID and "workspace" in str(e.value)
        setattr(c.args, what, old)
    c.run()
    c.free()
