"""What opure_kv_evict promises beyond its definition's values: every missing page is reported,
and scores_out may lie between the rows of scores."""
import ctypes as C

import numpy as np
import pytest

import opure_hip as H
import oracle as O
import window_ref as R
from gpu_util import device_model, say
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


@pytest.mark.parametrize("wfmt,afmt", [(O.W_F32, O.A_F32), (O.W_I8PC, O.A_F16), (O.W_I4G128, O.A_BF16)], ids=["f32", "i8-f16", "i4-bf16"])
def test_a_models_own_queries(dev, wfmt, afmt):
    """The set over a model's layers: opure_verify_layer leaves its rotated queries and its
    attention in the workspace; on a copy of those queries the windowed attention without a
    window gives what the layer's own attention gave, and the weights that the eviction goes
    by; the layers then go on at the new lengths, over keys that it turned."""
    say("own queries", wfmt, afmt)
    rng = np.random.default_rng(17)
    m = O.HostModel(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn=512, vocab=512, wfmt=wfmt, afmt=afmt,
                    attn_scale=0.125, theta=10000.0, max_pos=256, tied=True, seed=6)
    B, rows, cap, L, kvh = 2, 8, 128, 2, 2
    okv = O.HostKV(m, n_pages=20, batch=B, max_pages_per_seq=cap // 16)
    okv.page_table[...] = rng.permutation(20)[:B * cap // 16].reshape(B, -1)
    dm = device_model(dev, m)
    dkv = H.DeviceKV(dev, m.cfg, okv.n_pages, B, okv.max_pages)
    dkv.set_pool(okv.pool)
    dkv.set_page_table(okv.page_table)
    H.check(H.lib().opure_verify_reserve(dev.h, C.byref(dm.desc), B, rows, cap))
    offsets, ws, size = (C.c_uint64 * 5)(), C.c_void_p(), C.c_uint64()
    H.check(H.lib().opure_debug_verify_offsets(C.byref(dm.desc), B, rows, cap, offsets))
    dt, eb = H.act_dtype(afmt), 4 if afmt == F32 else 2
    sums, lens = dev.upload(np.zeros((B, L, kvh, cap), np.float32)), dev.upload(np.zeros(B, np.int32))
    q, out = dev.alloc(B * rows * 256 * eb), dev.alloc(B * rows * 256 * eb)
    kept = dev.alloc(B * L * kvh * 40 * 4)
    a = H.AttnWindowArgs(C.pointer(dm.desc), C.pointer(dkv.desc), 0, B, rows, int(lens), cap, 0, 0, int(q), int(out), None, cap, L * kvh * cap)
    ev = H.EvictArgs(C.pointer(dm.desc), C.pointer(dkv.desc), B, int(lens), cap, int(sums), cap, 2, 20, 18, 1, int(kept), int(sums), int(lens))
    n = [0, 0]
    for step in range(8):
        x = dev.upload(rng.standard_normal((B * rows, 256), dtype=np.float32))
        dev.write(lens, np.array(n, np.int32))
        total = dev.download(sums, np.float32, (B, L, kvh, cap)).astype(np.float64)
        for layer in range(L):
            va = H.VerifyLayerArgs(C.pointer(dm.desc), C.pointer(dkv.desc), layer, B, rows, int(lens), cap, int(x))
            H.check(H.lib().opure_verify_layer(dev.h, C.byref(va)))
            dev.sync()
            H.check(H.lib().opure_debug_workspace(dev.h, C.byref(ws), C.byref(size)))
            bits, own = (dev.download(ws.value, dt, (B, rows, 4, 64), offsets[i]) for i in (2, 3))
            dev.write(q, bits)
            a.layer, a.weights = layer, int(sums) + layer * kvh * cap * 4
            H.check(H.lib().opure_attn_window_paged(dev.h, C.byref(a)))
            dev.sync()
            got = R.act_to_f32(dev.download(out, dt, (B, rows, 4, 64)), afmt)
            cache = R.Cache(rng, afmt, L, kvh, 64, [k + rows for k in n], cap=cap)
            cache.pool, cache.table, cache.n_pages = dkv.get_pool(), okv.page_table, okv.n_pages
            ref, tol, w, wt = R.attention(cache, layer, R.act_to_f32(bits, afmt), 4, n, rows, 0, 0, 0.125)
            assert (np.abs(got - ref) <= tol).all() and (np.abs(R.act_to_f32(own, afmt) - ref) <= tol).all()
            now = dev.download(sums, np.float32, (B, L, kvh, cap))
            for b in range(B):
                want = total[b, layer, :, :n[b] + rows] + w[b]
                assert (np.abs(now[b, layer, :, :n[b] + rows] - want) <= wt[b] + 2.0 ** -23 * want).all()
        n = [k + rows for k in n]
        x.free()
        if n[0] == 48:
            dev.write(lens, np.array(n, np.int32))
            H.check(H.lib().opure_kv_evict(dev.h, C.byref(ev)))
            n = dev.download(lens, np.int32, (B,)).tolist()
            assert n == [40, 40]
    for buf in (sums, lens, q, out, kept):
        buf.free()
