"""Appending to a paged cache, attention over it and log probabilities as a user
runs them: layers of opure_gemv_batched_f32 -> opure_kv_append -> attention ->
opure_gemv_batched_f32, a prompt and then one row at a time, eagerly and replayed.
Every operator is held to its definition on the inputs that the device gave it."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as K
import opure_hip as H
import oracle as O
import test_gpu_logprobs as P
import window_ref as R
from gpu_util import say

pytestmark = pytest.mark.gpu

PAGE = H.PAGE_SIZE
HEADS, KV, HD, LAYERS, VOCAB, CAP, TOP = 8, 2, 64, 2, 1008, 200, 5
DIM = HEADS * HD
WIDTH = (HEADS + 2 * KV) * HD


@pytest.fixture(scope="module")
def dev():
    d = H.Dev(0)
    yield d
    d.close()


class Server:
    """Weights, a cache for `batch` sequences and the buffers of a step of `rows` rows."""

    def __init__(self, dev, i4, batch, rows, seed=0):
        rng = np.random.default_rng(seed)
        self.dev, self.i4, self.batch, self.rows = dev, i4, batch, rows
        self.keep = []
        cols = (CAP + PAGE - 1) // PAGE
        self.n_pages = batch * cols + 1
        self.table = rng.permutation(self.n_pages)[:batch * cols].reshape(batch, cols).astype(np.int32)
        m = self.model = H.Model()
        m.n_layers, m.n_heads, m.n_kv_heads, m.head_dim, m.afmt, m.attn_scale = LAYERS, HEADS, KV, HD, H.A_F32, HD ** -0.5
        ang = np.arange(CAP)[:, None] * 10000.0 ** (-2.0 * np.arange(HD // 2) / HD)
        self.cos, self.sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
        m.rope_cos, m.rope_sin, m.rope_max_pos = self.up(self.cos), self.up(self.sin), CAP
        size = C.c_uint64()
        H.check(H.lib().opure_kv_pool_bytes(C.byref(m), int(i4), self.n_pages, C.byref(size)))
        # no slot holds a number yet
        self.pool0 = np.full(size.value // 4, 0x7E007E00 if i4 else 0x7FC00000, np.uint32)
        self.pool, table = self.up(self.pool0), self.up(self.table)
        self.kv = H.KV(self.pool, self.n_pages, PAGE, table, cols)
        self.w = [[self.linear(rng, WIDTH, DIM), self.linear(rng, DIM, DIM)] for _ in range(LAYERS)]
        self.head = self.linear(rng, VOCAB, DIM)
        n = batch * rows
        self.seq, self.count, self.given = self.up(np.zeros(batch, np.int32)), self.up(np.zeros(batch, np.int32)), self.up(np.zeros(n, np.int32))
        self.x = [self.up(np.zeros((n, DIM), np.float32)) for _ in range(LAYERS + 1)]
        self.qkv = [self.up(np.zeros((n, WIDTH), np.float32)) for _ in range(LAYERS)]
        self.q, self.out = ([self.up(np.zeros((n, DIM), np.float32)) for _ in range(LAYERS)] for _ in range(2))
        self.logits = self.up(np.zeros((n, VOCAB), np.float32))
        self.answers = [self.up(np.zeros(n * k, np.float32)) for k in (1, 1, TOP, TOP)]

    def up(self, x):
        b = self.dev.upload(x)
        self.keep.append(b)
        return int(b)

    def linear(self, rng, out, n):
        w = H.Linear()
        w.out, w.in_, w.w = out, n, self.up(rng.standard_normal((out, n), dtype=np.float32) * np.float32(2.0 / n ** 0.5))
        tiled, kept = self.dev.tile(H.W_F32, w)
        self.keep += [b for b in kept if b]
        return tiled

    def appended(self, layer):
        a = H.KvAppendArgs()
        a.model, a.kv, a.kvfmt, a.layer, a.batch, a.rows = C.pointer(self.model), C.pointer(self.kv), H.KV_I4 if self.i4 else H.KV_ACT, layer, self.batch, self.rows
        a.seq_len, a.row_count, a.max_ctx, a.rotate, a.xfmt = self.seq, self.count, CAP, 1, H.A_F32
        a.q, a.k, a.v = (self.qkv[layer] + 4 * at * HD for at in (0, HEADS, HEADS + KV))
        a.q_stride = a.k_stride = a.v_stride = WIDTH
        a.q_out = self.q[layer]
        return a

    def attended(self, layer):
        a = H.AttnKv4Args() if self.i4 else H.AttnWindowArgs()
        a.model, a.kv, a.layer, a.batch, a.rows = C.pointer(self.model), C.pointer(self.kv), layer, self.batch, self.rows
        a.seq_len, a.max_ctx, a.window, a.sinks, a.q, a.out = self.seq, CAP, 60, 3, self.q[layer], self.out[layer]
        return a

    def answered(self):
        a = H.LogprobsArgs()
        a.rows, a.vocab, a.logits, a.logits_stride, a.temperature, a.top = self.batch * self.rows, VOCAB, self.logits, VOCAB, 0.7, TOP
        a.tokens, (a.logprob, a.entropy, a.top_tokens, a.top_logprobs) = self.given, self.answers
        return a

    def reserve(self):
        L, h = H.lib(), self.dev.h
        H.check((L.opure_attn_kv4_reserve if self.i4 else L.opure_attn_window_reserve)(h, C.byref(self.attended(0))))
        H.check(L.opure_logprobs_reserve(h, C.byref(self.answered())))

    def gemv(self, w, x, y):
        n = self.batch * self.rows
        for r in range(0, n, H.MAX_ROWS):
            H.gemv(self.dev, H.W_F32, w, x + 4 * r * w.in_, y + 4 * r * w.out, min(H.MAX_ROWS, n - r), H.A_F32, H.A_F32, H.EPI_STORE)

    def run(self):
        L, h = H.lib(), self.dev.h
        for i, (qkv, o) in enumerate(self.w):
            self.gemv(qkv, self.x[i], self.qkv[i])
            H.check(L.opure_kv_append(h, C.byref(self.appended(i))))
            H.check((L.opure_attn_kv4_paged if self.i4 else L.opure_attn_window_paged)(h, C.byref(self.attended(i))))
            self.gemv(o, self.out[i], self.x[i + 1])
        self.gemv(self.head, self.x[-1], self.logits)
        H.check(L.opure_logprobs(h, C.byref(self.answered())))

    def put(self, x, seq, count, given):
        for to, v in ((self.x[0], x), (self.seq, np.asarray(seq, np.int32)), (self.count, np.asarray(count, np.int32)), (self.given, np.asarray(given, np.int32))):
            self.dev.write(to, v)

    def get(self, buf, shape, dtype=np.float32):
        return self.dev.download(buf, dtype, shape)

    def state(self):
        """All that a step leaves, as bits."""
        n = self.batch * self.rows
        return [self.get(self.pool, self.pool0.shape, np.uint32)] + [self.get(b, (n, w), np.uint32) for b, w in
                [*((q, DIM) for q in self.q + self.out), (self.logits, VOCAB), (self.answers[0], 1), (self.answers[1], 1), (self.answers[2], TOP), (self.answers[3], TOP)]]

    def host_cache(self, before):
        """The reference's cache object on a copy of the pool's words."""
        cache = object.__new__(K.Kv4Cache if self.i4 else R.Cache)
        cache.layers, cache.n_kv, cache.hd, cache.n_pages, cache.table = LAYERS, KV, HD, self.n_pages, self.table
        if self.i4:
            pool = object.__new__(K.Kv4Pool)
            pool.hd, pool.ng, pool.words = HD, K.groups(HD), before.copy().reshape(LAYERS, self.n_pages, KV, -1)
            cache.pool = pool
        else:
            cache.afmt, cache.pool = H.A_F32, before.copy().view(np.float32).reshape(LAYERS, self.n_pages, 2, KV, PAGE, HD)
        return cache

    def check(self, before, seq, count, given):
        """One step's every result against the definitions, on what the device computed them from."""
        B, rows = self.batch, self.rows
        cache = self.host_cache(before)
        for i in range(LAYERS):
            x = self.get(self.qkv[i], (B, rows, HEADS + 2 * KV, HD))
            q = self.get(self.q[i], (B, rows, HEADS, HD))
            for b in range(B):
                n = count[b]
                if not n:
                    continue
                pos = np.arange(seq[b], seq[b] + n)
                t = K.turn(x[b, :n, :HEADS + KV], self.cos[pos], self.sin[pos])
                assert np.array_equal(q[b, :n].view(np.uint32), t[:, :HEADS].view(np.uint32))
                page, slot = self.table[b, pos // PAGE], pos % PAGE
                for which, y in ((0, t[:, HEADS:]), (1, x[b, :n, HEADS + KV:])):
                    if self.i4:
                        cache.pool.put(i, page, slot, which, y)
                    else:
                        O.kv_planes(cache.pool)[which][i, page, :, slot] = y
        got = self.get(self.pool, self.pool0.shape, np.uint32)
        want = cache.pool.words if self.i4 else cache.pool.view(np.uint32)
        assert np.array_equal(got, want.ravel())
        for i in range(LAYERS):
            q, out = (self.get(y[i], (B, rows, HEADS, HD)) for y in (self.q, self.out))
            for b in range(B):                              # rows past a sequence's count read slots that nobody wrote
                n, sub = count[b], object.__new__(type(cache))
                if not n:
                    continue
                sub.__dict__.update(cache.__dict__, table=self.table[b:b + 1])
                if self.i4:
                    ref, tol = K.attention(sub, i, q[b:b + 1, :n], H.A_F32, HEADS, [seq[b]], n, 60, 3, HD ** -0.5)
                else:
                    ref, tol = R.attention(sub, i, q[b:b + 1, :n], HEADS, [seq[b]], n, 60, 3, HD ** -0.5)[:2]
                P.compare(out[b:b + 1, :n], ref, tol)
        logits = self.get(self.logits, (B * rows, VOCAB))
        want, tol = P.reference(logits, given, TOP, 0.7)
        shapes = ((B * rows,), (B * rows,), (B * rows, TOP), (B * rows, TOP))
        for k, (buf, shape) in enumerate(zip(self.answers, shapes)):
            if k == 2:
                assert np.array_equal(self.get(buf, shape, np.int32), want[2])
            else:
                P.compare(self.get(buf, shape), want[k], tol[k])

    def free(self):
        for b in self.keep:
            b.free()


def step(s, x, seq, count, given):
    s.put(x, seq, count, given)
    before = s.get(s.pool, s.pool0.shape, np.uint32)
    s.run()
    s.dev.sync()
    s.check(before, seq, count, given)
    return before


@pytest.mark.parametrize("i4", [False, True], ids=["act", "i4"])
def test_prompt_then_rows(dev, i4):
    """Prompts of different lengths padded to one, then steps of one row, one sequence ending early."""
    say("step", i4)
    rng = np.random.default_rng(3)
    batch, rows, lens = 3, 70, [70, 33, 1]
    s = Server(dev, i4, batch, rows)
    step(s, rng.standard_normal((batch * rows, DIM), dtype=np.float32), [0] * batch, lens, rng.integers(0, VOCAB, batch * rows))
    one = Server(dev, i4, batch, 1)                        # the same weights and table: the same seed
    one.kv.pool, one.pool = s.pool, s.pool
    seq = list(lens)
    for k in range(5):
        count = [1, 1, int(k < 2)]
        step(one, rng.standard_normal((batch, DIM), dtype=np.float32), seq, count, rng.integers(0, VOCAB, batch))
        seq = [a + c for a, c in zip(seq, count)]
    one.free()
    s.free()


@pytest.mark.parametrize("i4", [False, True], ids=["act", "i4"])
def test_captured_steps(dev, i4):
    """A captured step replayed at rising lengths, other work between, has the eager step's bits; two of different
    shapes share the workspace."""
    say("captured step", i4)
    rng = np.random.default_rng(4)
    made = [Server(dev, i4, 2, rows, seed=7 + rows) for rows in (1, 5)]
    graphs = []
    for s in made:
        s.reserve()
    for s in made:
        dev.graph_begin()
        s.run()
        graphs.append(dev.graph_end())
    seqs = [[0, 0] for _ in made]
    for k in range(4):
        todo = []
        for s, seq, g in zip(made, seqs, graphs):
            n = 2 * s.rows
            call = (rng.standard_normal((n, DIM), dtype=np.float32), list(seq), [s.rows, s.rows - (k % 2 if s.rows > 1 else 0)], rng.integers(0, VOCAB, n))
            s.put(*call)
            todo.append((call, s.get(s.pool, s.pool0.shape, np.uint32)))
            dev.graph_launch(g)
        dev.sync()
        for s, seq, (call, before) in zip(made, seqs, todo):
            s.check(before, *call[1:])
            replayed = s.state()
            dev.write(s.pool, before)
            s.run()
            dev.sync()
            for a, b in zip(replayed, s.state()):
                assert np.array_equal(a, b)
            for b in range(2):
                seq[b] += call[2][b]
    for g in graphs:
        dev.graph_destroy(g)
    for s in made:
        s.free()


def test_two_handles_at_once(dev):
    """Steps of two device handles queued without waiting, each with its stream and workspace."""
    rng = np.random.default_rng(5)
    second = H.Dev(0)
    made = [Server(d, True, 2, 9, seed=k) for k, d in enumerate((dev, second))]
    calls = [(rng.standard_normal((18, DIM), dtype=np.float32), [0, 0], [9, 4], rng.integers(0, VOCAB, 18)) for _ in made]
    for s, call in zip(made, calls):
        s.put(*call)
    for _ in range(3):                                      # the same rows at the same positions: the same step
        for s in made:
            s.run()
    for s, call in zip(made, calls):
        s.dev.sync()
        s.check(s.pool0, *call[1:])
        s.free()
    second.close()


def test_workspace_grows_behind_a_graph(dev):
    """A larger call is refused in a capture that has too little workspace, which goes on; run eagerly it replaces
    the workspace, and the graph's calls keep theirs."""
    own = H.Dev(0)
    rng = np.random.default_rng(6)
    calls = []
    for batch, rows, n in ((1, 1, 2000), (6, 4, 2500)):     # both in parts, which are joined from the workspace
        cache = K.Kv4Cache(rng, 1, KV, HD, [n] * batch)
        q = rng.standard_normal((batch, rows, HEADS, HD), dtype=np.float32)
        c = K.Call(own, cache, q, H.A_F32, HEADS, [n - rows] * batch, rows, 0, 0, 0.1)
        calls.append((c, *K.attention(cache, 0, q, H.A_F32, HEADS, [n - rows] * batch, rows, 0, 0, 0.1)))
    (small, *want), (big, *want_big) = calls
    H.check(H.lib().opure_attn_kv4_reserve(own.h, C.byref(small.args)))
    own.graph_begin()
    small.run(sync=False)
    assert H.lib().opure_attn_kv4_paged(own.h, C.byref(big.args)) == H.E_CAPACITY
    g = own.graph_end()
    for _ in range(3):
        own.graph_launch(g)
        P.compare(big.run().result(), *want_big)
        P.compare(small.result(), *want)
        own.fill_u32(small.out, 0x7FC00000, HEADS * HD)
    own.graph_destroy(g)
    P.compare(small.run().result(), *want)
    small.free()
    big.free()
    own.close()


@pytest.mark.parametrize("rows", [1, 9, 40])
def test_sequences_that_share_pages(dev, rows):
    """One cache read through three rows of the page table, its pages in the same places: the same bits in each."""
    rng = np.random.default_rng(rows)
    cache = K.Kv4Cache(rng, 1, KV, HD, [900 + rows] * 3)
    cache.table[1:] = cache.table[0]
    q = np.repeat(rng.standard_normal((1, rows, HEADS, HD), dtype=np.float32), 3, 0)
    c = K.Call(dev, cache, q, H.A_F32, HEADS, [900] * 3, rows, 0, 0, 0.1)
    got = c.run().result()
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])
    ref, tol = K.attention(cache, 0, q, H.A_F32, HEADS, [900] * 3, rows, 0, 0, 0.1)
    assert (np.abs(got - ref) <= tol).all()
    c.free()
