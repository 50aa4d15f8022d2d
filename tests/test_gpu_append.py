"""opure_kv_append against the formulas, bit for bit: every format, head size and
layout, rows that begin and end anywhere in a page, padded batches, 4-bit words
that hold tokens of before, what cannot be written, capture and replay."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as K
import opure_hip as H
import oracle as O
from gpu_util import say
from npref import act_to_f32, f32_to_act

pytestmark = pytest.mark.gpu

PAGE = H.PAGE_SIZE
F32, F16, BF16 = H.A_F32, H.A_F16, H.A_BF16


@pytest.fixture(scope="module")
def dev():
    d = H.Dev(0)
    yield d
    d.close()


class Append:
    """One append's host state, buffers and arguments, and what it has to leave."""

    def __init__(self, dev, afmt, xfmt, i4, heads, n_kv, hd, seq, rows, counts=None, layers=1, rotate=True, seed=0, fused=True, edit=None,
                 max_ctx=None, spare=2, cols=None):
        self.__dict__.update(dev=dev, afmt=afmt, xfmt=xfmt, i4=i4, heads=heads, n_kv=n_kv, hd=hd, seq=list(seq), rows=rows, layers=layers,
                             rotate=rotate)
        rng = np.random.default_rng(seed)
        self.counts = list(counts) if counts is not None else [rows] * len(seq)
        self.layer = layers - 1
        self.cap = max_ctx or max(n + c for n, c in zip(seq, self.counts))
        need = [(n + c + PAGE - 1) // PAGE for n, c in zip(seq, self.counts)]
        self.n_pages = sum(need) + spare
        perm, at = rng.permutation(self.n_pages), 0
        self.table = np.full((len(seq), cols or max(max(need), (self.cap + PAGE - 1) // PAGE)), -1, np.int32)
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at:at + n]
            at += n
        if i4:
            self.pool = K.Kv4Pool(rng, layers, self.n_pages, n_kv, hd)
            w = self.pool.words[..., 128 * self.pool.ng:]
            w[...] = rng.standard_normal(w.shape + (2,)).astype(np.float16).view(np.uint32)[..., 0]
        else:
            self.pool = f32_to_act(rng.standard_normal((layers, self.n_pages, 2, n_kv, PAGE, hd), dtype=np.float32), afmt)
        x = rng.standard_normal((len(seq) * rows, (heads + 2 * n_kv) * hd), dtype=np.float32) * np.float32(2)
        x[:, heads * hd:] += rng.standard_normal(2 * n_kv * hd, dtype=np.float32)
        if edit:
            edit(x)
        with np.errstate(over="ignore"):
            self.x = act_to_f32(f32_to_act(x, xfmt), xfmt)
        ang = np.arange(self.cap)[:, None] * 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
        self.cos, self.sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
        self.q0 = f32_to_act(rng.standard_normal((len(seq) * rows, heads * hd), dtype=np.float32), afmt)
        # ---- the device's
        up, xb = dev.upload, 4 if xfmt == F32 else 2
        m = self.model = H.Model()
        m.n_layers, m.n_heads, m.n_kv_heads, m.head_dim, m.afmt = layers, heads, n_kv, hd, afmt
        a = self.args = H.KvAppendArgs()
        if fused:
            parts, width = [f32_to_act(self.x, xfmt)], self.x.shape[1]
        else:
            # rows apart, with room between them
            cut = np.cumsum([0, heads * hd, n_kv * hd, n_kv * hd])
            parts = [np.pad(f32_to_act(np.ascontiguousarray(self.x[:, i:j]), xfmt), ((0, 0), (0, 24))) for i, j in zip(cut, cut[1:])]
        self.bufs = [up(p) for p in parts] + [up(self.pool.words if i4 else self.pool), up(self.table), up(np.asarray(seq, np.int32)),
                                              up(np.asarray(self.counts, np.int32)), up(self.cos), up(self.sin), up(self.q0)]
        n = len(parts)
        self.pool_buf, self.table_buf, self.len_buf, self.count_buf, cos, sin, self.q_buf = self.bufs[n:]
        m.rope_cos, m.rope_sin, m.rope_max_pos = int(cos), int(sin), self.cap
        self.kv = H.KV(int(self.pool_buf), self.n_pages, PAGE, int(self.table_buf), self.table.shape[1])
        if fused:
            a.q, a.k = int(self.bufs[0]), int(self.bufs[0]) + heads * hd * xb
            a.v = a.k + n_kv * hd * xb
            a.q_stride = a.k_stride = a.v_stride = width
        else:
            a.q, a.k, a.v = (int(x) for x in self.bufs[:3])
            a.q_stride, a.k_stride, a.v_stride = (p.shape[1] for p in parts)
        a.q_out = int(self.q_buf)
        a.model, a.kv, a.kvfmt, a.layer, a.batch, a.rows = C.pointer(m), C.pointer(self.kv), int(i4), self.layer, len(seq), rows
        a.seq_len, a.max_ctx, a.rotate, a.xfmt = int(self.len_buf), self.cap, int(rotate), xfmt
        if counts is not None:
            a.row_count = int(self.count_buf)

    def run(self):
        H.check(H.lib().opure_kv_append(self.dev.h, C.byref(self.args)))

    def expect(self, seq=None):
        """The pool's bits and q's after the call, on the host's copies (q0 and pool change)."""
        heads, n_kv, hd, R = self.heads, self.n_kv, self.hd, self.rows
        x = self.x.reshape(-1, R, heads + 2 * n_kv, hd)
        for b, (n0, n) in enumerate(zip(seq or self.seq, self.counts)):
            if not n:
                continue
            pos = np.arange(n0, n0 + n)
            with np.errstate(all="ignore"):
                t = K.turn(x[b, :n, :heads + n_kv], self.cos[pos], self.sin[pos]) if self.rotate else x[b, :n, :heads + n_kv]
                self.q0.reshape(-1, R, heads * hd)[b, :n] = f32_to_act(np.ascontiguousarray(t[:, :heads]).reshape(n, -1), self.afmt)
            page, slot = self.table[b, pos // PAGE], pos % PAGE
            for which, y in ((0, t[:, heads:]), (1, x[b, :n, heads + n_kv:])):
                if self.i4:
                    self.pool.put(self.layer, page, slot, which, y)
                else:
                    with np.errstate(all="ignore"):
                        O.kv_planes(self.pool)[which][self.layer, page, :, slot] = f32_to_act(np.ascontiguousarray(y), self.afmt)

    def check(self):
        dt = np.uint32 if self.afmt == F32 else np.uint16
        if self.i4:
            got = self.dev.download(self.pool_buf, np.uint32, self.pool.words.shape)
            want = self.pool.words
        else:
            got, want = self.dev.download(self.pool_buf, dt, self.pool.shape), self.pool.view(dt)
        same = got == want
        if not self.i4:
            f = [act_to_f32(np.ascontiguousarray(y).view(np.float32) if self.afmt == F32 else np.ascontiguousarray(y), self.afmt) for y in (got, want)]
            same |= np.isnan(f[0]) & np.isnan(f[1])
        else:
            # a base of 0 of either sign
            half = [np.ascontiguousarray(y[..., 128 * self.pool.ng:]).view(np.float16) for y in (got, want)]
            eq = (half[0] == half[1]) | (np.isnan(half[0]) & np.isnan(half[1]))
            same[..., 128 * self.pool.ng:] |= eq.reshape(eq.shape[:-1] + (-1, 2)).all(-1)
        assert same.all(), (np.argwhere(~same)[:4], got[~same][:4], want[~same][:4])
        q = self.dev.download(self.q_buf, dt, self.q0.shape)
        qw = self.q0.view(dt)
        if self.args.q:
            f = [act_to_f32(y.view(np.float32) if self.afmt == F32 else y, self.afmt) for y in (q, qw)]
            assert ((q == qw) | (np.isnan(f[0]) & np.isnan(f[1]))).all()

    def free(self):
        for b in self.bufs:
            b.free()


def check(dev, *a, **kw):
    c = Append(dev, *a, **kw)
    for _ in range(2):                      # again over its own results: the same
        c.run()
        dev.sync()
    c.expect()
    c.check()
    c.free()


@pytest.mark.parametrize("i4", [False, True], ids=["act", "i4"])
@pytest.mark.parametrize("afmt,xfmt", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("hd", list(range(16, 257, 16)))
def test_head_sizes(dev, hd, afmt, xfmt, i4):
    say("append", hd, afmt, xfmt, i4)
    check(dev, afmt, xfmt, i4, 6, 2, hd, [0, 13, 37], 5, seed=hd)
    check(dev, afmt, xfmt, i4, 3, 3, hd, [7], 21, seed=hd + 1, fused=False)


@pytest.mark.parametrize("i4", [False, True], ids=["act", "i4"])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 15, 16, 17, 18, 33, 64])
def test_rows_and_slots(dev, rows, i4):
    """Every first slot of a page."""
    say("rows", rows, i4)
    check(dev, F16, F16, i4, 2, 1, 64, list(range(16)), rows, seed=rows)
    check(dev, BF16, F32, i4, 5, 5, 80, [16 * s + s for s in range(0, 16, 3)], rows, seed=rows, layers=3)


@pytest.mark.parametrize("i4", [False, True], ids=["act", "i4"])
@pytest.mark.parametrize("heads,n_kv", [(1, 1), (7, 1), (9, 3), (16, 2), (40, 8), (33, 1)])
def test_layouts(dev, heads, n_kv, i4):
    say("layout", heads, n_kv, i4)
    check(dev, BF16, BF16, i4, heads, n_kv, 48, [3, 77], 6, seed=heads, fused=False)
    check(dev, F32, F32, i4, heads, n_kv, 16, [15], 9, seed=heads, rotate=False)


@pytest.mark.parametrize("seed", range(40))
def test_shapes_at_random(dev, seed):
    r = np.random.default_rng(500 + seed)
    n_kv, G = int(r.choice([1, 2, 3, 5, 8])), int(r.choice([1, 2, 3, 4, 7]))
    afmt, hd = int(r.integers(0, 3)), 16 * int(r.integers(1, 17))
    rows = int(r.choice([1, 1, 2, 5, 9, 16, 33, 70, 150]))
    batch = int(r.integers(1, 6))
    seq = [int(r.integers(0, int(2 ** r.uniform(1, 10)))) for _ in range(batch)]
    counts = [int(r.integers(0, rows + 1)) for _ in range(batch)] if r.random() < 0.5 else None
    if counts is not None and not any(counts):
        counts[0] = 1
    i4 = bool(r.integers(0, 2))
    say("random", seed, afmt, n_kv, G, hd, seq, rows, counts, i4)
    check(dev, afmt, int(r.choice([F32, afmt])), i4, n_kv * G, n_kv, hd, seq, rows, counts, seed=seed, rotate=bool(r.integers(0, 2)),
          fused=bool(r.integers(0, 2)), layers=int(r.integers(1, 3)))


@pytest.mark.parametrize("i4", [False, True], ids=["act", "i4"])
def test_prompt(dev, i4):
    say("prompt", i4)
    check(dev, F16, F16, i4, 4, 2, 128, [29], 600, seed=3)
    check(dev, BF16, F32, i4, 4, 2, 64, [0, 5, 100], 333, [333, 222, 111], seed=4)
    check(dev, F16, F32, i4, 1, 1, 16, [9], 2048, seed=5)


@pytest.mark.parametrize("i4", [False, True], ids=["act", "i4"])
def test_padded_batch(dev, i4):
    """Sequences with none of their rows there, counts outside 0..rows."""
    say("padded", i4)
    check(dev, F16, F16, i4, 4, 2, 64, [5, 60, 7, 31], 20, [0, 20, 3, 1], seed=1)
    c = Append(dev, F16, F16, i4, 4, 2, 64, [5, 60, 7], 20, [0, 20, 3], seed=2)
    dev.write(c.count_buf, np.array([-7, 99, 3], np.int32))
    c.run()
    dev.sync()
    c.expect()
    c.check()
    c.free()


@pytest.mark.parametrize("i4", [False, True], ids=["act", "i4"])
def test_extremes(dev, i4):
    """NaN, infinities, magnitudes past what 4 bits hold, constant and tiny groups."""
    say("extremes", i4)

    def edit(x):
        x[0, 5], x[1, 300], x[2, 420] = np.nan, np.inf, -np.inf
        x[3, 256:288], x[3, 384:416] = 0.0, 3.25
        x[4, 256:320] *= 1e-8
        x[5, 256:288] = 1e9
        x[5, 288:320] *= 1e6
        x[6, 384:400] = -1e30
        x[7, 384:512] = 100 + 1e-3 * x[7, 384:512]
        x[8, 384:512] = -0.0

    for afmt, xfmt in ((BF16, F32), (F32, F32), (BF16, BF16)):
        check(dev, afmt, xfmt, i4, 4, 2, 64, [10], 12, seed=8, edit=edit)
        check(dev, afmt, xfmt, i4, 4, 2, 64, [10], 12, seed=8, edit=edit, rotate=False)


def test_scales_between_two_halves(dev):
    """Ranges whose fifteenth is, rounded to fp32, half way between two fp16 numbers, and is not without that rounding."""
    say("ties")
    r = np.random.default_rng(11).uniform(1, 2, 1 << 21).astype(np.float32)
    f = np.float32(1.0 / 15.0)
    p = r * f
    tie = ((p.view(np.uint32) & 0x1FFF) == 0x1000) & (r.astype(np.float64) * np.float64(f) != p)
    r = r[tie][:160]
    assert len(r) == 160

    def edit(x):
        # a group of 32: 0, the range, and numbers between them
        for which in (1, 2):
            g = x[:, 128 * which:128 * which + 128].reshape(20, 4, 32)
            top = r.reshape(2, 20, 4)[which - 1]
            g[...] = np.abs(g) % 1 * top[..., None]
            g[..., 3], g[..., 17] = 0, top

    check(dev, BF16, F32, True, 1, 1, 128, [5], 20, seed=3, rotate=False, edit=edit)


@pytest.mark.parametrize("spread,offset", [(1.0, 0.0), (30.0, 0.0), (1.0, 40.0), (1e-3, 0.0)])
def test_error_of_4_bits(dev, spread, offset):
    """A value is off by half a scale, half a step of fp16 in the scale (times 31) and in base and one in the value."""
    say("error", spread, offset)
    c = Append(dev, F32, F32, True, 1, 2, 128, [3], 40, rotate=False, seed=9, edit=lambda x: np.add(x * np.float32(spread), np.float32(offset), out=x))
    c.run()
    got = K.Kv4Pool(np.random.default_rng(0), 1, c.n_pages, 2, 128)
    got.words = dev.download(c.pool_buf, np.uint32, got.words.shape)
    pos = np.arange(3, 43)
    page, slot = c.table[0, pos // PAGE], pos % PAGE
    for which in (0, 1):
        for h in range(2):
            x = c.x[:, 128 * (1 + 2 * which + h):][:, :128].astype(np.float64)
            y = got.get(0, page, slot, h, which)
            g = x.reshape(40, 4, 32)
            step = ((g.max(-1) - g.min(-1)) / 15).repeat(32, 1)
            big = np.abs(g).max(-1).repeat(32, 1)
            # the base is at most big + 16 steps; fp16 rounds to 2^-11 of a value, its smallest steps are 2^-24
            bound = step / 2 + 2.0 ** -11 * (31 * step + (big + 16 * step) + big) + 2.0 ** -22
            assert (np.abs(x - y) <= bound).all()
    c.free()


@pytest.mark.parametrize("i4", [False, True], ids=["act", "i4"])
def test_queries_in_place_and_left_out(dev, i4):
    say("in place", i4)
    for afmt in (F32, F16, BF16):
        c = Append(dev, afmt, afmt, i4, 4, 2, 64, [7, 30], 6, seed=4, fused=False)
        q = np.ascontiguousarray(f32_to_act(c.x[:, :256], afmt))
        dev.write(c.q_buf, q)
        c.args.q, c.args.q_stride = int(c.q_buf), 256
        c.run()
        c.expect()
        c.check()
        c.free()
        c = Append(dev, afmt, F32, i4, 4, 2, 64, [7, 30], 6, seed=5)
        before = c.q0.copy()
        c.args.q = c.args.q_out = None
        c.model.n_heads = 0
        c.run()
        c.expect()
        c.q0 = before
        c.check()
        c.free()


@pytest.mark.parametrize("i4", [False, True], ids=["act", "i4"])
def test_rows_that_cannot_be_written(dev, i4):
    """Past max_ctx, a negative length, a missing or wrong page: reported, nothing of them written."""
    say("errors", i4)

    def failing(c, seq=None):
        c.run()
        with pytest.raises(H.OpureError) as e:
            dev.sync()
        assert e.value.code == H.E_CAPACITY
        dev.sync()                           # reported once

    # the third sequence's last rows lie past max_ctx
    c = Append(dev, F16, F16, i4, 2, 2, 32, [4, 9, 40], 10, seed=1)
    c.args.max_ctx = 45
    failing(c)
    c.counts[2] = 5
    c.expect()
    c.check()
    c.free()
    # a negative length writes nothing of its sequence
    c = Append(dev, F16, F16, i4, 2, 2, 32, [4, 9], 10, seed=2)
    dev.write(c.len_buf, np.array([-1, 9], np.int32))
    failing(c)
    c.counts[0] = 0
    c.expect()
    c.check()
    c.free()
    # lengths at the end of 32 bits
    c = Append(dev, F16, F16, i4, 2, 2, 32, [4, 9], 10, seed=2)
    dev.write(c.len_buf, np.array([0x7FFFFFFF, 9], np.int32))
    failing(c)
    c.counts[0] = 0
    c.expect()
    c.check()
    c.free()
    # a page that is missing, and one past the pool: the rows' q is written, their K and V are not
    for bad in (-1, 1 << 20):
        c = Append(dev, F16, F16, i4, 2, 2, 32, [4, 9], 30, seed=3)
        table = c.table.copy()
        table[0, 1] = bad
        dev.write(c.table_buf, table)
        failing(c)
        gone = c.table[0, 1]
        words = (c.pool.words if i4 else c.pool)[:, gone].copy()
        c.expect()
        (c.pool.words if i4 else c.pool)[:, gone] = words
        c.check()
        c.free()


@pytest.mark.parametrize("i4", [False, True], ids=["act", "i4"])
def test_capture_and_replay(dev, i4):
    """A captured append follows its lengths; eager work and syncs between the replays."""
    say("graph", i4)
    c = Append(dev, F16, F16, i4, 4, 2, 64, [7, 30], 3, seed=6, max_ctx=64, cols=4, spare=8)
    c.table[...] = np.random.default_rng(7).permutation(8).reshape(2, 4)
    dev.write(c.table_buf, c.table)
    dev.graph_begin()
    c.run()
    g = dev.graph_end()
    for step in range(4):
        seq = [7 + 3 * step, 30 + 3 * step]
        dev.write(c.len_buf, np.array(seq, np.int32))
        dev.graph_launch(g)
        dev.sync()
        c.expect(seq)
        c.check()
    dev.graph_destroy(g)
    c.free()


@pytest.mark.parametrize("i4", [False, True], ids=["act", "i4"])
def test_offsets_past_32_bits(dev, i4):
    """Pages and rows that lie past 4 GB."""
    say("large", i4)
    n_kv, hd = 8, 128
    block = 640 * 4 * n_kv if i4 else 2 * n_kv * PAGE * hd * 2
    n_pages = (5 << 30) // block
    c = Append(dev, F16, F16, i4, 8, n_kv, hd, [5], 20, seed=6)
    small = c.n_pages
    pool = dev.alloc(n_pages * block)
    table = c.table.copy()
    used = [int(p) for p in table[0] if p >= 0]
    far = {p: n_pages - 1 - i for i, p in enumerate(used)}
    size = 160 * 4 * n_kv if i4 else 2 * n_kv * PAGE * hd
    host = c.pool.words if i4 else c.pool
    for p, f in far.items():
        dev.write(pool, host[0, p], f * block)
    dev.write(c.table_buf, np.array([[far.get(int(p), -1) for p in table[0]]], np.int32))
    c.kv.pool, c.kv.n_pages = int(pool), n_pages
    c.run()
    dev.sync()
    c.expect()
    for p, f in far.items():
        got = dev.download(pool, host.dtype, (size,), f * block)
        assert np.array_equal(got, host[0, p].ravel())
    assert small == len(used) + 2
    pool.free()
    c.free()
