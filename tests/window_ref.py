"""Plain 64-bit restatements of windowed attention over the paged cache, its
accumulated weights, and eviction, for the tests of those entry points; and the
device buffers that such a call takes."""
import ctypes as C

import numpy as np

import opure_hip as H
import oracle as O
from npref import act_to_f32, f32_to_act

PAGE = H.PAGE_SIZE
NAMES = {H.A_F32: "f32", H.A_F16: "f16", H.A_BF16: "bf16"}
# a rounding is off by at most half a step, relative to the value
HALF_STEP = {H.A_F32: 2.0 ** -24, H.A_F16: 2.0 ** -11, H.A_BF16: 2.0 ** -8}
NAN_BITS = {H.A_F32: 0x7FC00000, H.A_F16: 0x7E00, H.A_BF16: 0x7FC0}


class Cache:
    """A paged cache on the host: K and V as [batch][layers][n_kv][n][hd] values of
    the format, scattered over pages in no order.  Every slot that holds no
    position, and every page that is nobody's, holds NaN."""

    def __init__(self, rng, afmt, layers, n_kv, hd, lens, cap=None, spare=3):
        self.afmt, self.layers, self.n_kv, self.hd, self.lens = afmt, layers, n_kv, hd, [int(n) for n in lens]
        cols = ((cap or max(self.lens)) + PAGE - 1) // PAGE
        need = [(n + PAGE - 1) // PAGE for n in self.lens]
        self.n_pages = sum(need) + spare
        perm = rng.permutation(self.n_pages)
        self.table = np.full((len(self.lens), max(1, cols)), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at:at + n]
            at += n
        dt = np.float32 if afmt == H.A_F32 else np.uint16
        self.pool = np.empty((layers, self.n_pages, 2, n_kv, PAGE, hd), dt)
        self.pool.view(np.uint32 if afmt == H.A_F32 else np.uint16)[...] = NAN_BITS[afmt]
        for b, n in enumerate(self.lens):
            self.put(b, slice(0, n), rng.standard_normal((layers, 2, n_kv, n, hd), dtype=np.float32))

    def slots(self, b, t):
        t = np.arange(self.lens[b])[t] if isinstance(t, slice) else np.asarray(t)
        return self.table[b, t // PAGE], t % PAGE

    def put(self, b, t, x):
        """x [layers][2][n_kv][len(t)][hd]"""
        page, slot = self.slots(b, t)
        k, v = O.kv_planes(self.pool)
        x = f32_to_act(x, self.afmt)
        k[:, page, :, slot] = x[:, 0].transpose(2, 0, 1, 3)
        v[:, page, :, slot] = x[:, 1].transpose(2, 0, 1, 3)

    def get(self, b, layer, h, which, n, pool=None):
        page, slot = self.slots(b, np.arange(n))
        plane = O.kv_planes(self.pool if pool is None else pool)[which]
        return act_to_f32(np.ascontiguousarray(plane[layer, page, h, slot]), self.afmt)


def sees(lens_b, rows, n, window, sinks):
    p, t = np.arange(lens_b, lens_b + rows)[:, None], np.arange(n)[None]
    m = t <= p
    return m & ((t < sinks) | (t > p - window)) if window else m


def attention(cache, layer, q, heads, seq, rows, window, sinks, scale):
    """(out, bound of |out's error|, weights, their bound), everything in 64 bits.
    q [B][rows][heads][hd] values.  The bounds count: each score's 32-bit sum
    (hd + 2 roundings of its terms' magnitudes) entering the weight twice (itself
    and the sum), 2^-20 for the exponential and the sums of positive terms, one
    rounding of the weights and one of the result to the cache's format."""
    B, hd, G = len(seq), cache.hd, heads // cache.n_kv
    out = np.zeros((B, rows, heads, hd))
    tol = np.zeros_like(out)
    wsum, wtol = [], []
    u = HALF_STEP[cache.afmt]
    for b, n0 in enumerate(seq):
        n = n0 + rows
        ws, wt = np.zeros((cache.n_kv, n)), np.zeros((cache.n_kv, n))
        m = sees(n0, rows, n, window, sinks)
        for h in range(cache.n_kv):
            k, v = (cache.get(b, layer, h, i, n).astype(np.float64) for i in (0, 1))
            live = m.any(0)
            k, v = np.where(live[:, None], k, 0), np.where(live[:, None], v, 0)
            for g in range(G):
                x = q[b, :, h * G + g].astype(np.float64)
                with np.errstate(all="ignore"):
                    s = np.where(m, x @ k.T * scale, -np.inf)
                    top = s.max(1, keepdims=True)
                    e = np.exp(s - np.where(np.isneginf(top), 0.0, top))
                    e = np.where(m, e, 0)
                    l = e.sum(1, keepdims=True)
                    w = np.where(m & (l != 0), e / l, 0.0)
                    size = np.abs(x) @ np.abs(k).T * abs(scale)
                    ds = (hd + 2) * 2.0 ** -24 * np.where(m & np.isfinite(size), size, 0).max(1, keepdims=True)
                    vz = np.where(m[:, :, None], v[None], 0.0) if not np.isfinite(v).all() else None
                    out[b, :, h * G + g] = w @ v if vz is None else np.einsum("rt,rtd->rd", w, vz)
                    mag = w @ np.abs(v) if vz is None else np.einsum("rt,rtd->rd", w, np.abs(vz))
                rel = 2 * ds + 2.0 ** -20
                tol[b, :, h * G + g] = u * np.abs(out[b, :, h * G + g]) * (1 + u) + (rel + (u if cache.afmt != H.A_F32 else 0)) * mag + 1e-30
                if cache.afmt == H.A_F16:
                    tol[b, :, h * G + g] += 2.0 ** -24        # half a step of fp16's smallest values
                ws[h] += w.sum(0)
                wt[h] += (w * (rel + 2.0 ** -20)).sum(0)
        wsum.append(ws)
        wtol.append(wt)
    return out, tol, wsum, wtol


class Call:
    """Device buffers and the argument structure of one windowed attention."""

    def __init__(self, dev, cache, q, heads, seq, rows, window, sinks, scale, layer=0, max_ctx=None, weights=None, stride=None,
                 batch_stride=None):
        self.dev, self.cache, self.shape = dev, cache, (len(seq), rows, heads, cache.hd)
        m = self.model = H.Model()
        m.n_layers, m.n_heads, m.n_kv_heads, m.head_dim = cache.layers, heads, cache.n_kv, cache.hd
        m.attn_scale, m.afmt = scale, cache.afmt
        up = dev.upload
        self.bufs = [up(cache.pool), up(cache.table), up(np.asarray(seq, np.int32)), up(f32_to_act(q, cache.afmt))]
        self.out = dev.alloc(q.size * (4 if cache.afmt == H.A_F32 else 2))
        self.kv = H.KV(int(self.bufs[0]), cache.n_pages, PAGE, int(self.bufs[1]), cache.table.shape[1])
        self.weights = up(weights) if weights is not None else None
        self.wshape = weights.shape if weights is not None else None
        a = self.args = H.AttnWindowArgs()
        a.model, a.kv, a.layer, a.batch, a.rows = C.pointer(m), C.pointer(self.kv), layer, len(seq), rows
        a.seq_len, a.max_ctx, a.window, a.sinks = int(self.bufs[2]), max_ctx or max(seq) + rows, window, sinks
        a.q, a.out = int(self.bufs[3]), int(self.out)
        if weights is not None:
            a.weights = int(self.weights)
            a.weights_stride = stride or weights.shape[-1]
            a.weights_batch_stride = batch_stride or int(np.prod(weights.shape[1:]))

    def run(self, sync=True):
        H.check(H.lib().opure_attn_window_paged(self.dev.h, C.byref(self.args)))
        if sync:
            self.dev.sync()
        return self

    def result(self):
        return act_to_f32(self.dev.download(self.out, H.act_dtype(self.cache.afmt), self.shape), self.cache.afmt)

    def sums(self):
        return self.dev.download(self.weights, np.float32, self.wshape)

    def free(self):
        for b in self.bufs + [self.out] + ([self.weights] if self.weights else []):
            b.free()


def select(scores, n, sinks, recent, heavy):
    """The kept positions of one (sequence, layer, KV head)."""
    keep = sinks + recent + heavy
    if n <= keep:
        return np.arange(n)
    s = np.asarray(scores[:n], np.float64)
    rank = np.where(np.isnan(s), np.inf, s) + 0.0
    # NaN above +inf: a second key
    cand = np.arange(sinks, n - recent)
    order = sorted(cand, key=lambda t: (not np.isnan(s[t]), -rank[t], t))
    return np.sort(np.concatenate([np.arange(sinks), np.array(order[:heavy], int), np.arange(n - recent, n)])).astype(int)


def evict(cache, seq, scores, sinks, recent, heavy, theta, turn):
    """(kept lists, per plane K and V in 64 bits of the new slots, new lengths)."""
    freq = theta ** (-2.0 * np.arange(cache.hd // 2) / cache.hd)
    kept, planes = {}, {}
    for b, n in enumerate(seq):
        for layer in range(cache.layers):
            for h in range(cache.n_kv):
                idx = select(scores[b, layer, h], n, sinks, recent, heavy)
                k, v = (cache.get(b, layer, h, i, n)[idx].astype(np.float64) for i in (0, 1))
                if turn:
                    ang = (np.arange(len(idx)) - idx)[:, None] * freq
                    x, y = k[:, 0::2].copy(), k[:, 1::2].copy()
                    k[:, 0::2], k[:, 1::2] = x * np.cos(ang) - y * np.sin(ang), x * np.sin(ang) + y * np.cos(ang)
                kept[b, layer, h], planes[b, layer, h] = idx, (k, v)
    return kept, planes, [min(n, sinks + recent + heavy) for n in seq]
