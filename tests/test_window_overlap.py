"""Refusals of opure_attn_window_paged and opure_kv_evict whose buffers overlap (no
kernel is launched: the device handle is a placeholder that refused calls never
dereference)."""
import ctypes as C

import pytest

import opure_hip as H

MIB = 1 << 20


@pytest.fixture
def at():
    raw = C.create_string_buffer(512)
    yield (C.addressof(raw) + 255) // 256 * 256


def model(at):
    m = H.Model()
    m.n_layers, m.n_heads, m.n_kv_heads, m.head_dim, m.afmt = 2, 8, 2, 64, H.A_F16
    m.rope_cos, m.rope_sin, m.rope_max_pos = at, at, 64
    return m


POOL, Q = 2 * 4 * 2 * 2 * 16 * 64 * 2, 2 * 4 * 8 * 64 * 2    # bytes of the cache and of q
SUMS = (130 + 64 + 64) * 4                                   # of weights: the last row's end


def window(at, **kw):
    """Buffers a MiB apart, those in kw at other offsets."""
    where = {n: at + i * MIB for i, n in enumerate(("pool", "table", "seq_len", "q", "out", "weights"), 1)}
    where.update({n: where[base] + off for n, (base, off) in kw.items()})
    m = model(at)
    kv = H.KV(where["pool"], 4, H.PAGE_SIZE, where["table"], 4)
    return m, kv, H.AttnWindowArgs(C.pointer(m), C.pointer(kv), 0, 2, 4, where["seq_len"], 64, 16, 2, where["q"], where["out"], where["weights"],
                                   64, 130)


@pytest.mark.parametrize("kw", [dict(weights=("q", 0)), dict(weights=("q", Q - 4)), dict(weights=("q", 4 - SUMS)), dict(weights=("out", 128)),
                                dict(weights=("pool", POOL - 4)), dict(weights=("pool", 4 - SUMS)), dict(weights=("table", 28)),
                                dict(weights=("seq_len", 4)), dict(out=("pool", 4096)), dict(out=("pool", POOL - 16)), dict(out=("table", 0)),
                                dict(out=("seq_len", 0)), dict(out=("q", 16))])
def test_window_refuses_overlaps(at, kw):
    m, kv, a = window(at, **kw)
    assert H.lib().opure_attn_window_paged(at, C.byref(a)) == H.E_INVALID
    assert b"overlaps" in H.lib().opure_last_error()


SCORES, KEPT = (7 * 70 + 64) * 4, 8 * 9 * 4                  # of scores with a stride of 70, of kept


def evict(at, stride=70, **kw):
    names = ("pool", "table", "seq_len", "scores", "kept", "scores_out", "new_seq_len", "freed", "n_freed")
    where = {n: at + i * MIB for i, n in enumerate(names, 1)}
    where.update({n: where[base] + off for n, (base, off) in kw.items()})
    m = model(at)
    kv = H.KV(where["pool"], 4, H.PAGE_SIZE, where["table"], 4)
    return m, kv, H.EvictArgs(C.pointer(m), C.pointer(kv), 2, where["seq_len"], 64, where["scores"], stride, 2, 3, 4, 1, where["kept"],
                              where["scores_out"], where["new_seq_len"], where["freed"], 4, where["n_freed"])


@pytest.mark.parametrize("kw", [dict(scores_out=("scores", 4)), dict(scores_out=("scores", -4)), dict(scores_out=("scores", 280)),
                                dict(scores_out=("scores", -63 * 4)), dict(scores_out=("scores", 7 * 280 + 63 * 4)),
                                dict(scores_out=("scores", 65 * 4)), dict(kept=("scores", SCORES - 4)), dict(kept=("scores_out", 4 - KEPT)),
                                dict(kept=("pool", 0)), dict(scores=("pool", POOL - 4)), dict(scores_out=("pool", 4 - SCORES)),
                                dict(new_seq_len=("seq_len", 4)), dict(new_seq_len=("kept", 0)), dict(n_freed=("new_seq_len", 0)),
                                dict(n_freed=("seq_len", 0)), dict(freed=("table", 16)), dict(freed=("new_seq_len", -28)),
                                dict(table=("pool", 64)), dict(new_seq_len=("table", 28))])
def test_evict_refuses_overlaps(at, kw):
    m, kv, a = evict(at, **kw)
    assert H.lib().opure_kv_evict(at, C.byref(a)) == H.E_INVALID
    assert b"overlaps" in H.lib().opure_last_error()
