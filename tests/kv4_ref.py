"""Plain restatements of the 4-bit paged cache, of appending to a paged cache and of
attention over the 4-bit one, for the tests of those entry points; and the device
buffers that such calls take."""
import ctypes as C

import numpy as np

import opure_hip as H
import window_ref as R
from npref import act_to_f32, f32_to_act

PAGE = H.PAGE_SIZE
MOST = np.float32(16384.0)


def groups(hd):
    return (hd + 31) // 32


def quantise(x):
    """Codes [..][hd], scales and bases [..][ng] (fp16) of x [..][hd] in fp32, each step rounded as written."""
    x = np.asarray(x, np.float32)
    hd, ng = x.shape[-1], groups(x.shape[-1])
    codes = np.zeros(x.shape, np.int64)
    s, b = (np.zeros(x.shape[:-1] + (ng,), np.float16) for _ in range(2))
    for g in range(ng):
        part = x[..., 32 * g:min(hd, 32 * g + 32)]
        bad = ~np.isfinite(part).all(-1)
        y = np.clip(np.where(np.isfinite(part), part, np.float32(0)), -MOST, MOST)
        lo, hi = y.min(-1), y.max(-1)
        sg = ((hi - lo) * np.float32(1.0 / 15.0)).astype(np.float16)
        bg = (lo - np.float32(16.0) * sg.astype(np.float32)).astype(np.float16)
        with np.errstate(all="ignore"):
            c = np.rint((y - bg.astype(np.float32)[..., None]) / sg.astype(np.float32)[..., None] - np.float32(16.0))
        c = np.where((sg == 0)[..., None] | bad[..., None], 0, np.clip(np.nan_to_num(c), 0, 15))
        codes[..., 32 * g:min(hd, 32 * g + 32)] = c
        s[..., g], b[..., g] = np.where(bad, np.float16(np.nan), sg), np.where(bad, np.float16(np.nan), bg)
    return codes, s, b


def values(codes, s, b):
    """What codes stand for, fp16 numbers as doubles (sums of two are exact in 64 bits)."""
    hd = codes.shape[-1]
    rep = np.minimum(np.arange(hd) // 32, s.shape[-1] - 1)
    return (s.astype(np.float64)[..., rep] * (16 + codes) + b.astype(np.float64)[..., rep]).astype(np.float16).astype(np.float64)


class Kv4Pool:
    """A 4-bit pool on the host, uint32 [layers][n_pages][n_kv][160 ng], read and written slot by slot."""

    def __init__(self, rng, layers, n_pages, n_kv, hd):
        self.hd, self.ng = hd, groups(hd)
        # every slot holds codes at random and NaN scales
        self.words = rng.integers(0, 1 << 32, (layers, n_pages, n_kv, 160 * self.ng), dtype=np.uint32)
        self.words[..., 128 * self.ng:] = 0x7E007E00

    def _at(self, which, u, d):
        """(word, bit) of channel d of token u; positions of its group's scale and base among the fp16 of the block."""
        ng, g = self.ng, d // 32
        if which == 0:
            return (d % 32 // 8 * 16 + u) * ng + g, 16 * (d % 2) + 4 * (d % 8 // 2), 256 * ng + 2 * (u * ng + g), 256 * ng + 2 * (u * ng + g) + 1
        at = 288 * ng + (u // 4 * ng + g) * 8 + u % 4
        return 64 * ng + (u // 4 * 16 + d % 16) * ng + g, 16 * (u % 2) + 8 * (d % 32 // 16) + 4 * (u % 4 // 2), at, at + 4

    def put(self, layer, pages, slots, which, x):
        """x [len(pages)][n_kv][hd] quantised into those slots; of half a group the other half's codes of the token are 0."""
        codes, s, b = quantise(x)
        full = np.zeros(codes.shape[:-1] + (32 * self.ng,), np.int64)
        full[..., :self.hd] = codes
        half = self.words.view(np.float16)
        for t, (page, slot) in enumerate(zip(pages, slots)):
            d = np.arange(32 * self.ng)
            word, bit, sa, ba = self._at(which, int(slot), d)
            block = self.words[layer, page]
            for dd in d:
                clear = np.uint32(0xFFFFFFFF ^ (15 << int(bit[dd])))
                block[:, word[dd]] = (block[:, word[dd]] & clear) | (full[t, :, dd].astype(np.uint32) << np.uint32(bit[dd]))
            for g in range(self.ng):
                half[layer, page][:, sa[32 * g]], half[layer, page][:, ba[32 * g]] = s[t, :, g], b[t, :, g]

    def put_all(self, layer, pages, slots, which, x):
        """The same for many tokens of pages that hold nothing else: whole pages at a time."""
        n_kv, ng = self.words.shape[2], self.ng
        codes, s, b = quantise(x)
        for page in np.unique(pages):
            t = np.nonzero(pages == page)[0]
            u, d = slots[t][:, None], np.arange(self.hd)[None]
            word, bit, sa, ba = (np.broadcast_to(y, (len(t), self.hd)) for y in self._at(which, u, d))
            lo, hi = (0, 64 * ng) if which == 0 else (64 * ng, 128 * ng)
            self.words[layer, page, :, lo:hi] = 0
            half = self.words.view(np.float16)
            for h in range(n_kv):
                np.bitwise_or.at(self.words[layer, page, h], word, codes[t, h].astype(np.uint32) << bit.astype(np.uint32))
                half[layer, page, h][sa[:, ::32]], half[layer, page, h][ba[:, ::32]] = s[t, h], b[t, h]

    def get(self, layer, pages, slots, h, which):
        """[len(pages)][hd] values as doubles."""
        d = np.arange(self.hd)[None]
        word, bit, sa, ba = self._at(which, np.asarray(slots)[:, None], d)
        block = self.words[layer, pages, h]
        half = np.ascontiguousarray(block).view(np.float16)
        code = (np.take_along_axis(block, np.broadcast_to(word, (len(pages), self.hd)), 1) >> np.broadcast_to(bit, (len(pages), self.hd)).astype(np.uint32)) & 15
        s = np.take_along_axis(half, np.broadcast_to(sa, (len(pages), self.hd)), 1).astype(np.float64)
        b = np.take_along_axis(half, np.broadcast_to(ba, (len(pages), self.hd)), 1).astype(np.float64)
        return (s * (16 + code.astype(np.int64)) + b).astype(np.float16).astype(np.float64)


class Kv4Cache:
    """A 4-bit cache of normal keys and values over pages in no order."""

    def __init__(self, rng, layers, n_kv, hd, lens, cap=None, spare=3, spread=1.0):
        self.layers, self.n_kv, self.hd, self.lens = layers, n_kv, hd, [int(n) for n in lens]
        cols = ((cap or max(self.lens)) + PAGE - 1) // PAGE
        need = [(n + PAGE - 1) // PAGE for n in self.lens]
        self.n_pages = sum(need) + spare
        perm = rng.permutation(self.n_pages)
        self.table = np.full((len(self.lens), max(1, cols)), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at:at + n]
            at += n
        self.pool = Kv4Pool(rng, layers, self.n_pages, n_kv, hd)
        for b, n in enumerate(self.lens):
            page, slot = self.slots(b, np.arange(n))
            for layer in range(layers):
                for which in (0, 1):
                    x = rng.standard_normal((n, n_kv, hd), dtype=np.float32) * np.float32(spread)
                    self.pool.put_all(layer, page, slot, which, x)

    def slots(self, b, t):
        t = np.asarray(t)
        return self.table[b, t // PAGE], t % PAGE

    def put(self, b, t, layer, which, x):
        page, slot = self.slots(b, t)
        self.pool.put(layer, page, slot, which, x)

    def get(self, b, layer, h, which, n):
        page, slot = self.slots(b, np.arange(n))
        return self.pool.get(layer, page, slot, h, which)


def attention(cache, layer, q, afmt, heads, seq, rows, window, sinks, scale):
    """(out, bound of |out's error|) in 64 bits.  q [B][rows][heads][hd] values of the format.
    The bound counts, for each score, its 32-bit sum (hd + 2 roundings of its terms' magnitudes) and what the
    row's fp16 form leaves out (bf16: 2^-34 of the row's largest magnitude; fp32, as two numbers: 2^-22 of each
    and that), entering the weight twice (itself and the sum), 2^-20 for the exponential and the sums of
    positive terms, the weight's rounding (2^-11 as one fp16 number, 2^-22 as two) and one rounding of the result;
    and fp16's smallest step, 2^-24: a weight is held as 2^12 e^(s - m), m at least the largest score seen less
    3 ln 2, so that half a step is 2^-37 of a weight whose row sums to 1 or more.  A sum in which all that
    counts lies there (the larger weights' values are 0 exactly) is off by as much of the values' magnitudes."""
    B, hd, G = len(seq), cache.hd, heads // cache.n_kv
    out = np.zeros((B, rows, heads, hd))
    tol = np.zeros_like(out)
    u = R.HALF_STEP[afmt]
    for b, n0 in enumerate(seq):
        n = n0 + rows
        m = R.sees(n0, rows, n, window, sinks)
        live = m.any(0)
        for h in range(cache.n_kv):
            k, v = (cache.get(b, layer, h, i, n) for i in (0, 1))
            k, v = np.where(live[:, None], k, 0), np.where(live[:, None], v, 0)
            for g in range(G):
                x = q[b, :, h * G + g].astype(np.float64)
                with np.errstate(all="ignore"):
                    s = np.where(m, x @ k.T * scale, -np.inf)
                    top = s.max(1, keepdims=True)
                    e = np.where(m, np.exp(s - np.where(np.isneginf(top), 0.0, top)), 0)
                    l = e.sum(1, keepdims=True)
                    w = np.where(m & (l != 0), e / l, 0.0)
                    size = np.abs(x) @ np.abs(k).T * abs(scale)
                    ds = (hd + 2) * 2.0 ** -24 * size
                    if afmt != H.A_F16:
                        ds = ds + 2.0 ** -34 * np.abs(x).max(1, keepdims=True) * np.abs(k).sum(1)[None] * abs(scale)
                    if afmt == H.A_F32:
                        ds = ds + 2.0 ** -22 * size
                    ds = np.where(m & np.isfinite(ds), ds, 0).max(1, keepdims=True)
                    if np.isfinite(v).all():
                        out[b, :, h * G + g], mag, least = w @ v, w @ np.abs(v), m @ np.abs(v)
                    else:
                        vz = np.where(m[:, :, None], v[None], 0.0)
                        out[b, :, h * G + g], mag = np.einsum("rt,rtd->rd", w, vz), np.einsum("rt,rtd->rd", w, np.abs(vz))
                        least = np.abs(vz).sum(1)
                rel = 2 * ds + 2.0 ** -20 + (2.0 ** -11 if afmt == H.A_BF16 else 2.0 ** -22)
                tol[b, :, h * G + g] = u * np.abs(out[b, :, h * G + g]) * (1 + u) + rel * mag + 2.0 ** -37 * least + 1e-30
                if afmt == H.A_F16:
                    tol[b, :, h * G + g] += 2.0 ** -24        # half a step of fp16's smallest values
    return out, tol


class Call:
    """Device buffers and the argument structure of one attention over a 4-bit cache."""

    def __init__(self, dev, cache, q, afmt, heads, seq, rows, window, sinks, scale, layer=0, max_ctx=None):
        self.dev, self.afmt, self.shape = dev, afmt, (len(seq), rows, heads, cache.hd)
        m = self.model = H.Model()
        m.n_layers, m.n_heads, m.n_kv_heads, m.head_dim = cache.layers, heads, cache.n_kv, cache.hd
        m.attn_scale, m.afmt = scale, afmt
        up = dev.upload
        self.bufs = [up(cache.pool.words), up(cache.table), up(np.asarray(seq, np.int32)), up(f32_to_act(q, afmt))]
        self.out = dev.alloc(q.size * (4 if afmt == H.A_F32 else 2))
        self.kv = H.KV(int(self.bufs[0]), cache.n_pages, PAGE, int(self.bufs[1]), cache.table.shape[1])
        a = self.args = H.AttnKv4Args()
        a.model, a.kv, a.layer, a.batch, a.rows = C.pointer(m), C.pointer(self.kv), layer, len(seq), rows
        a.seq_len, a.max_ctx, a.window, a.sinks = int(self.bufs[2]), max_ctx or max(seq) + rows, window, sinks
        a.q, a.out = int(self.bufs[3]), int(self.out)

    def run(self, sync=True):
        H.check(H.lib().opure_attn_kv4_paged(self.dev.h, C.byref(self.args)))
        if sync:
            self.dev.sync()
        return self

    def result(self):
        return act_to_f32(self.dev.download(self.out, H.act_dtype(self.afmt), self.shape), self.afmt)

    def free(self):
        for b in self.bufs + [self.out]:
            b.free()


def turn(x, cos, sin):
    """x [n][heads][hd] in fp32 turned by its rows' cosines and sines [n][hd / 2], products and sums rounded."""
    e, o, c, s = x[..., 0::2], x[..., 1::2], cos[:, None], sin[:, None]
    y = np.empty_like(x)
    y[..., 0::2], y[..., 1::2] = e * c - o * s, e * s + o * c
    return y
