"""opure_kv_evict against its definition in 64 bits, and a run of the whole set:
prompt, windowed attention with its weights, eviction, a verify step that goes on."""
import ctypes as C

import numpy as np
import pytest

import opure_hip as H
import oracle as O
import window_ref as R
from gpu_util import VerifyRunner, device_model, say

pytestmark = pytest.mark.gpu

F32, F16, BF16 = H.A_F32, H.A_F16, H.A_BF16
THETA = 10000.0


@pytest.fixture(scope="module")
def dev():
    d = H.Dev(0)
    yield d
    d.close()


class Evict:
    def __init__(self, dev, cache, seq, scores, sinks, recent, heavy, turn, max_ctx=None, in_place=False, free=True, alias_len=False,
                 with_scores=True):
        self.dev, self.cache, self.keep = dev, cache, sinks + recent + heavy
        B, self.cap = len(seq), max_ctx or max(seq)
        cos, sin = H.rope_table(THETA, cache.hd, max(1, self.cap), H.ROPE_GPU)
        up = dev.upload
        m = self.model = H.Model()
        m.n_layers, m.n_heads, m.n_kv_heads, m.head_dim, m.afmt = cache.layers, cache.n_kv, cache.n_kv, cache.hd, cache.afmt
        self.cos, self.sin = up(cos), up(sin)
        if turn:
            m.rope_cos, m.rope_sin, m.rope_max_pos = int(self.cos), int(self.sin), cos.shape[0]
        self.pool, self.table, self.len, self.scores = up(cache.pool), up(cache.table), up(np.asarray(seq, np.int32)), up(scores)
        self.sshape, self.kshape = scores.shape, (*scores.shape[:3], self.keep)
        self.kept = up(np.full(self.kshape, -7, np.int32))
        self.sout = self.scores if in_place else up(np.full(scores.shape, 5.0, np.float32))
        self.new_len = self.len if alias_len else dev.alloc(4 * B)
        self.stride = (self.cap + 15) // 16
        self.freed, self.n_freed = up(np.full((B, self.stride), -9, np.int32)), dev.alloc(4 * B)
        self.kv = H.KV(int(self.pool), cache.n_pages, R.PAGE, int(self.table), cache.table.shape[1])
        self.args = H.EvictArgs(C.pointer(m), C.pointer(self.kv), B, int(self.len), self.cap, int(self.scores), scores.shape[-1], sinks,
                                recent, heavy, 1 if turn else 0, int(self.kept), int(self.sout) if with_scores else None, int(self.new_len),
                                int(self.freed) if free else None, self.stride, int(self.n_freed))
        self.B = B

    def run(self, sync=True):
        H.check(H.lib().opure_kv_evict(self.dev.h, C.byref(self.args)))
        if sync:
            self.dev.sync()
        return self

    def get(self):
        d = self.dev.download
        return dict(pool=d(self.pool, H.act_dtype(self.cache.afmt), self.cache.pool.shape), table=d(self.table, np.int32, self.cache.table.shape),
                    kept=d(self.kept, np.int32, self.kshape), scores=d(self.sout, np.float32, self.sshape),
                    new_len=d(self.new_len, np.int32, (self.B,)), freed=d(self.freed, np.int32, (self.B, self.stride)),
                    n_freed=d(self.n_freed, np.int32, (self.B,)))

    def done(self):
        for b in {id(x): x for x in (self.cos, self.sin, self.pool, self.table, self.len, self.scores, self.kept, self.sout, self.new_len,
                                     self.freed, self.n_freed)}.values():
            b.free()


def check(dev, afmt, layers, n_kv, hd, seq, sinks, recent, heavy, turn=True, seed=0, scores=None, extra=0, **kw):
    rng = np.random.default_rng(seed)
    cap = max(seq) + extra
    cache = R.Cache(rng, afmt, layers, n_kv, hd, seq, cap=cap)
    if scores is None:
        scores = np.exp(rng.standard_normal((len(seq), layers, n_kv, cap + 3), dtype=np.float32) * 2)
    e = Evict(dev, cache, seq, scores, sinks, recent, heavy, turn, max_ctx=cap, **kw).run()
    got = e.get()
    kept, planes, lens = R.evict(cache, seq, scores, sinks, recent, heavy, THETA, turn)
    keep = sinks + recent + heavy
    assert got["new_len"].tolist() == lens
    u = R.HALF_STEP[afmt]
    touched = np.zeros(cache.pool.shape, bool)
    tk, tv = O.kv_planes(touched)
    for (b, layer, h), idx in kept.items():
        row = np.full(keep, -1)
        row[:len(idx)] = idx
        assert np.array_equal(got["kept"][b, layer, h], row), (b, layer, h)
        k, v = planes[b, layer, h]
        gk, gv = (cache.get(b, layer, h, i, len(idx), got["pool"]).astype(np.float64) for i in (0, 1))
        assert np.array_equal(gv, v)
        same = idx == np.arange(len(idx))
        old = cache.get(b, layer, h, 0, seq[b])[idx]
        assert np.array_equal(gk[same], old[same].astype(np.float64))            # unmoved keys keep their bits
        if not turn:
            assert np.array_equal(gk, k)
        # the table's cos and sin are rounded to 32 bits, as are the two products and
        # their sum: at most 4 roundings of |x| + |y|; then one to the format
        mag = np.abs(old[:, 0::2]) + np.abs(old[:, 1::2])
        bound = u * np.abs(k) * 1.01 + np.repeat(mag, 2, 1) * 4 * 2.0 ** -24 + (2.0 ** -25 if afmt == F16 else 0)
        assert not (np.abs(gk - k) > bound).any(), float(np.max(np.abs(gk - k) - bound))
        if kw.get("with_scores", True):
            s = got["scores"][b, layer, h]
            assert np.array_equal(s[:len(idx)], scores[b, layer, h, idx], equal_nan=True)
            assert (s[len(idx):seq[b]] == 0).all()
            beyond = scores[b, layer, h, seq[b]:] if kw.get("in_place") else 5.0
            assert np.array_equal(s[seq[b]:], np.broadcast_to(beyond, s[seq[b]:].shape), equal_nan=True)
        page, slot = cache.slots(b, np.arange(len(idx)))
        tk[layer, page, h, slot] = tv[layer, page, h, slot] = True
    bits = np.uint32 if afmt == F32 else np.uint16
    assert np.array_equal(got["pool"].view(bits)[~touched], cache.pool.view(bits)[~touched])   # nothing else is written
    for b, n in enumerate(seq):
        first, last = (lens[b] + 15) // 16, (n + 15) // 16
        if kw.get("free", True):
            want = cache.table[b].copy()
            out = want[first:last].copy()
            want[first:last] = -1
            assert np.array_equal(got["table"][b], want)
            assert np.array_equal(got["freed"][b, :len(out)], out) and (got["freed"][b, len(out):] == -9).all()
            assert got["n_freed"][b] == len(out)
        else:
            assert np.array_equal(got["table"][b], cache.table[b]) and got["n_freed"][b] == 0
    e.done()


@pytest.mark.parametrize("turn", [True, False], ids=["turn", "move"])
@pytest.mark.parametrize("afmt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", list(range(16, 257, 16)))
def test_head_sizes(dev, hd, afmt, turn):
    say("evict head size", hd, afmt, turn)
    check(dev, afmt, 2, 3, hd, [100, 3, 47, 161], 2, 21, 24, turn, seed=hd)


@pytest.mark.parametrize("afmt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", list(range(16, 257, 16)))
def test_caches_past_the_last_level_cache(dev, hd, afmt):
    """What a cache could hold (max_ctx) decides how it is moved: 256 MB and more
    whole lines at a time, here with few positions in it; 600 of them take several runs."""
    say("evict large", hd, afmt)
    eb = 4 if afmt == F32 else 2
    extra = (300 << 20) // (2 * hd * eb * 2 * 2)
    check(dev, afmt, 1, 2, hd, [600, 90], 3, 100, 130, hd % 32 == 0 and extra < 400000, seed=hd, extra=extra)


@pytest.mark.parametrize("sinks,recent,heavy", [(0, 1, 0), (0, 0, 1), (1, 0, 0), (4, 30, 0), (0, 0, 50), (16, 16, 16), (5, 1, 250), (0, 299, 0),
                                                (0, 0, 300), (100, 100, 99), (1000, 2, 3), (0, 40, 1)])
def test_budgets(dev, sinks, recent, heavy):
    say("budget", sinks, recent, heavy)
    check(dev, F16, 1, 2, 64, [300, 0, 1, 16, 17, 299, 50], sinks, recent, heavy, seed=sinks)
    check(dev, BF16, 2, 1, 32, [300, 16], sinks, recent, heavy, seed=sinks, free=False, in_place=True, extra=40)


@pytest.mark.parametrize("seed", range(40))
def test_shapes_at_random(dev, seed):
    r = np.random.default_rng(2000 + seed)
    seq = [int(r.integers(0, int(2 ** r.uniform(3, 12.5)))) for _ in range(int(r.integers(1, 5)))]
    keep = 1 + int(r.integers(0, max(seq) + 20))
    sinks = int(r.integers(0, min(keep, 40) + 1))
    recent = int(r.integers(0, keep - sinks + 1))
    afmt, hd = int(r.integers(0, 3)), 16 * int(r.integers(1, 9))
    say("evict random", seed, afmt, hd, seq, sinks, recent, keep)
    check(dev, afmt, int(r.integers(1, 4)), int(r.integers(1, 4)), hd, [max(1, n) for n in seq], sinks, recent, keep - sinks - recent,
          bool(r.integers(0, 2)), seed=seed, in_place=bool(r.integers(0, 2)), free=bool(r.integers(0, 2)), extra=int(r.choice([0, 5, 5000])))


@pytest.mark.parametrize("n,keep", [(1024, 1000), (1025, 64), (2049, 1500), (5000, 1100), (9000, 4500), (20000, 300)])
def test_long(dev, n, keep):
    say("evict long", n, keep)
    check(dev, F16, 1, 2, 32, [n, n // 3], 4, keep // 3, keep - 4 - keep // 3, seed=n, in_place=n % 2 == 0)


@pytest.mark.parametrize("afmt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", list(range(16, 257, 16)))
def test_more_parts_than_fit_at_a_time(dev, hd, afmt):
    """Four a CU of 64 bytes of a key or 16 channels of V: shorter runs of keys."""
    say("evict many parts", hd, afmt)
    parts = -(-hd * (4 if afmt == F32 else 2) // 64) + hd // 16
    check(dev, afmt, -(-1024 // (6 * parts)), 2, hd, [161, 300, 40], 1, 30, 60, seed=hd)


@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in place"])
def test_long_of_many_heads(dev, in_place):
    """More heads than CUs, whose selection takes its sequences in blocks of 2,048."""
    say("evict long, many heads", in_place)
    check(dev, BF16, 33, 4, 16, [5000, 4096, 2049], 4, 300, 800, seed=7, in_place=in_place)


def test_scores_of_every_kind(dev):
    """Ties (the lowest positions stay), negative scores, zeros of both signs,
    infinities, NaN, denormal numbers, values that share their leading bits."""
    rng = np.random.default_rng(3)
    n = 700
    rows = [np.zeros(n), np.full(n, 2.5), rng.integers(0, 4, n).astype(float), -rng.random(n), np.where(rng.random(n) < 0.5, 0.0, -0.0),
            np.where(rng.random(n) < 0.1, np.inf, np.where(rng.random(n) < 0.1, -np.inf, rng.standard_normal(n))),
            np.where(rng.random(n) < 0.05, np.nan, np.where(rng.random(n) < 0.05, np.inf, rng.standard_normal(n))), np.full(n, np.nan),
            np.full(n, -np.inf), rng.integers(0, 30, n) * 1e-44, 1.0 + rng.integers(0, 40, n) * 2.0 ** -23,
            np.sign(rng.standard_normal(n)) * rng.integers(0, 3, n) * 1e30]
    scores = np.stack(rows).astype(np.float32).reshape(1, 4, 3, n)
    for heavy in (1, 130, 500):
        check(dev, F16, 4, 3, 16, [n], 3, 20, heavy, scores=scores)
        check(dev, F16, 4, 3, 16, [n], 0, 0, heavy, scores=scores, in_place=True, alias_len=True)


@pytest.mark.parametrize("kw", [dict(alias_len=True), dict(free=False), dict(free=False, alias_len=True), dict(with_scores=False),
                                dict(in_place=True, extra=37)])
def test_forms_of_the_call(dev, kw):
    check(dev, BF16, 2, 2, 128, [200, 90, 64], 3, 30, 31, **kw)


def test_nothing_to_evict(dev):
    check(dev, F16, 2, 2, 64, [64, 1, 0, 33], 4, 30, 30)


def test_bad_lengths_and_pages(dev):
    """A length past max_ctx, below zero, or over a missing page: reported, in bounds."""
    rng = np.random.default_rng(4)
    for what in ("long", "negative", "missing", "beyond"):
        say("bad", what)
        cache = R.Cache(rng, F16, 1, 2, 64, [200])
        scores = rng.random((1, 1, 2, 200), dtype=np.float32)
        if what == "missing":
            cache.table[0, 3] = -1
        if what == "beyond":
            cache.table[0, 3] = cache.n_pages
        e = Evict(dev, cache, [200], scores, 2, 70, 30, True)
        if what == "long":
            dev.write(e.len, np.array([201], np.int32))
        if what == "negative":
            dev.write(e.len, np.array([-5], np.int32))
        with pytest.raises(H.OpureError) as err:
            e.run()
        assert err.value.code == H.E_CAPACITY
        e.done()
    check(dev, F16, 1, 2, 64, [200], 2, 70, 30)


def test_captured_and_replayed(dev):
    """Replays on restored caches, with eager work between, have the eager call's bits."""
    rng = np.random.default_rng(5)
    cache = R.Cache(rng, BF16, 3, 2, 128, [400, 100, 222])
    scores = rng.random((3, 3, 2, 400), dtype=np.float32)
    e = Evict(dev, cache, [400, 100, 222], scores, 4, 50, 60, True).run()
    want = e.get()
    g = None
    for k in range(4):
        dev.write(e.pool, cache.pool)
        dev.write(e.table, cache.table)
        if g is None:
            dev.graph_begin()
            e.run(sync=False)
            g = dev.graph_end()
        dev.graph_launch(g)
        dev.sync()
        got = e.get()
        for name in want:
            assert np.array_equal(want[name], got[name], equal_nan=name == "scores"), name
        check(dev, F16, 1, 2, 64, [300], 1, 20, 40, seed=k)
    dev.graph_destroy(g)
    e.done()


def test_offsets_past_32_bits(dev):
    """A pool whose last pages lie past 2^32 bytes (and elements)."""
    rng = np.random.default_rng(6)
    n_kv, hd, n = 8, 128, 150
    cache = R.Cache(rng, F16, 1, n_kv, hd, [n])
    scores = rng.random((1, 1, n_kv, n), dtype=np.float32)
    e = Evict(dev, cache, [n], scores, 4, 30, 40, True)
    page_bytes = 2 * n_kv * 16 * hd * 2
    big = (5 << 31) // page_bytes
    pool = dev.alloc(big * page_bytes)
    first = big - cache.n_pages
    dev.write(pool, cache.pool, first * page_bytes)
    dev.write(e.table, np.where(cache.table >= 0, cache.table + first, -1).astype(np.int32))
    e.kv.pool, e.kv.n_pages = int(pool), big
    e.run()
    got = dev.download(pool, np.uint16, cache.pool.shape, first * page_bytes)
    small = Evict(dev, cache, [n], scores, 4, 30, 40, True).run()
    assert np.array_equal(got, small.get()["pool"]) and np.array_equal(e.get()["kept"], small.get()["kept"])
    e.done()
    small.done()
    pool.free()


@pytest.mark.parametrize("wfmt,afmt,bar", [(O.W_F32, O.A_F32, 1e-4), (O.W_I8PC, O.A_F16, 2e-2), (O.W_I4G128, O.A_BF16, 2e-2)],
                         ids=["f32", "i8-f16", "i4-bf16"])
def test_prompt_weights_eviction_and_on(dev, wfmt, afmt, bar):
    """The set as a server uses it: prompts through verify steps, windowed attention
    that scores the cached positions of each layer, an eviction that turns the kept
    keys, then verify steps on the shorter cache against the oracle on the same
    cache; and again, so that the second eviction finds the first's keys."""
    say("run", wfmt, afmt)
    rng = np.random.default_rng(11)
    m = O.HostModel(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn=512, vocab=512, wfmt=wfmt, afmt=afmt,
                    attn_scale=0.125, theta=THETA, max_pos=256, tied=True, seed=5)
    B, rows, cap, L, kvh = 2, 8, 128, 2, 2
    okv = O.HostKV(m, n_pages=20, batch=B, max_pages_per_seq=cap // 16)
    perm = rng.permutation(20)
    okv.page_table[...] = perm[:B * cap // 16].reshape(B, -1)
    dm = device_model(dev, m)
    dkv = H.DeviceKV(dev, m.cfg, okv.n_pages, B, okv.max_pages)
    dkv.set_pool(okv.pool)
    dkv.set_page_table(okv.page_table)
    run = VerifyRunner(dev, dm, dkv, B, rows, max_ctx=cap)
    sums = dev.upload(np.zeros((B, L, kvh, cap), np.float32))
    q, out = dev.alloc(B * rows * 256 * 4), dev.alloc(B * rows * 256 * 4)
    n = np.array([0, 0], np.int32)
    kept, new_len = dev.alloc(B * L * kvh * 40 * 4), dev.alloc(B * 4)
    a = H.AttnWindowArgs()
    a.model, a.kv, a.batch, a.rows, a.seq_len, a.max_ctx = C.pointer(dm.desc), C.pointer(dkv.desc), B, rows, int(run.seq_len), cap
    a.window, a.sinks, a.q, a.out = 24, 2, int(q), int(out)
    a.weights_stride, a.weights_batch_stride = cap, L * kvh * cap
    ev = H.EvictArgs()
    ev.model, ev.kv, ev.batch, ev.seq_len, ev.max_ctx = a.model, a.kv, B, int(run.seq_len), cap
    ev.scores = ev.scores_out = int(sums)
    ev.scores_stride, ev.sinks, ev.recent, ev.heavy, ev.turn = cap, 2, 20, 18, 1
    ev.kept, ev.new_seq_len = int(kept), int(run.seq_len)
    for turn in range(2):
        for _ in range(6 if turn == 0 else 4):
            toks = rng.integers(0, 512, (B, rows)).astype(np.int32)
            okv.pool[...] = dkv.get_pool()
            run.step(toks, n)
            want = O.verify_forward(m, okv, toks, n)
            assert np.abs(run.get_logits() - want).max() <= bar
            for layer in range(L):
                dev.write(q, R.f32_to_act(rng.standard_normal((B, rows, 4, 64), dtype=np.float32), afmt))
                a.layer, a.weights = layer, int(sums) + layer * kvh * cap * 4
                H.check(H.lib().opure_attn_window_paged(dev.h, C.byref(a)))
            n = n + rows
        dev.write(run.seq_len, n)
        before, s = dkv.get_pool(), dev.download(sums, np.float32, (B, L, kvh, cap))
        cache = R.Cache(rng, afmt, L, kvh, 64, n, cap=cap)
        cache.pool, cache.table, cache.n_pages = before, okv.page_table, okv.n_pages
        H.check(H.lib().opure_kv_evict(dev.h, C.byref(ev)))
        dev.sync()
        idx, planes, lens = R.evict(cache, n, s, 2, 20, 18, THETA, True)
        got = dkv.get_pool()
        for key, (k, v) in planes.items():
            b, layer, h = key
            mag = np.abs(k).max() + 1e-3
            gk, gv = (cache.get(b, layer, h, i, lens[b], got).astype(np.float64) for i in (0, 1))
            assert np.array_equal(gv, v) and np.abs(gk - k).max() <= mag * (2 * R.HALF_STEP[afmt] + 2.0 ** -21)
        n = dev.download(run.seq_len, np.int32, (B,))
        assert n.tolist() == lens == [40, 40]
