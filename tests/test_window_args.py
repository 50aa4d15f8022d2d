"""Refusals and struct layouts of opure_attn_window_paged and opure_kv_evict (no
kernel is launched: the device handle is a placeholder that refused calls never
dereference)."""
import ctypes as C
import os
import subprocess

import pytest

import opure_hip as H

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_header(tmp_path):
    structs = {"opure_attn_window_args": H.AttnWindowArgs, "opure_evict_args": H.EvictArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "opure_hip.h"', "int main(void){"]
    for name, cls in structs.items():
        lines.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "probe")], check=True)
    for line in subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True, check=True).stdout.split("\n"):
        if line:
            name, field, value = line.split()
            cls = structs[name]
            assert int(value) == (C.sizeof(cls) if field == "size" else getattr(cls, field).offset), (name, field)


@pytest.fixture
def fake():
    raw = C.create_string_buffer(512)
    at = (C.addressof(raw) + 255) // 256 * 256
    m = H.Model()
    m.n_layers, m.n_heads, m.n_kv_heads, m.head_dim, m.afmt = 2, 8, 2, 64, H.A_F16
    m.rope_cos, m.rope_sin, m.rope_max_pos = at, at, 64
    kv = H.KV(at, 4, H.PAGE_SIZE, at, 4)
    return at, m, kv, raw


def window_args(fake, **kw):
    at, m, kv, _ = fake
    a = H.AttnWindowArgs(C.pointer(m), C.pointer(kv), 0, 2, 4, at, 64, 16, 2, at, at, at, 64, 2 * 64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def evict_args(fake, **kw):
    at, m, kv, _ = fake
    a = H.EvictArgs(C.pointer(m), C.pointer(kv), 2, at, 64, at, 64, 2, 3, 4, 1, at, at, at, at, 4, at)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


WINDOW = [(dict(q=None), H.E_INVALID, b"null"), (dict(out=None), H.E_INVALID, b"null"), (dict(seq_len=None), H.E_INVALID, b"null"),
          (dict(model=None), H.E_INVALID, b"null"), (dict(kv=None), H.E_INVALID, b"null"), (dict(layer=2), H.E_INVALID, b"layer"),
          (dict(batch=0), H.E_CAPACITY, b"sequences"), (dict(batch=257), H.E_CAPACITY, b"sequences"), (dict(rows=0), H.E_CAPACITY, b"rows"),
          (dict(rows=2049, max_ctx=2049), H.E_CAPACITY, b"rows"), (dict(max_ctx=3), H.E_CAPACITY, b"max_ctx"),
          (dict(max_ctx=65), H.E_CAPACITY, b"max_ctx"), (dict(max_ctx=0xFFFFFFFF), H.E_CAPACITY, b"max_ctx"),
          (dict(weights_stride=63), H.E_INVALID, b"weights_stride"), (dict(weights_batch_stride=127), H.E_INVALID, b"overlap"),
          (dict(sinks=1 << 31), H.E_INVALID, b"sinks")]


@pytest.mark.parametrize("kw,code,word", WINDOW, ids=[next(iter(w[0])) + str(i) for i, w in enumerate(WINDOW)])
def test_window_refusals(fake, kw, code, word):
    L, at = H.lib(), fake[0]
    assert L.opure_attn_window_paged(at, C.byref(window_args(fake, **kw))) == code
    assert word in L.opure_last_error()


def test_window_refuses_models_and_caches(fake):
    L, (at, m, kv, _) = H.lib(), fake
    assert L.opure_attn_window_paged(None, C.byref(window_args(fake))) == H.E_INVALID
    assert L.opure_attn_window_paged(at, None) == H.E_INVALID
    assert L.opure_attn_window_reserve(None, None) == H.E_INVALID
    assert L.opure_attn_window_reserve(at, None) == H.E_INVALID
    for what, value, code in (("n_kv_heads", 0, H.E_INVALID), ("n_kv_heads", 3, H.E_INVALID), ("head_dim", 24, H.E_UNSUPPORTED),
                              ("head_dim", 0, H.E_UNSUPPORTED), ("head_dim", 272, H.E_UNSUPPORTED), ("afmt", 3, H.E_INVALID),
                              ("n_heads", 0, H.E_INVALID)):
        old = getattr(m, what)
        setattr(m, what, value)
        assert L.opure_attn_window_paged(at, C.byref(window_args(fake))) == code, what
        assert L.opure_attn_window_reserve(at, C.byref(window_args(fake))) == code, what
        setattr(m, what, old)
    for what, value, code in (("n_pages", 0, H.E_INVALID), ("max_pages_per_seq", 0, H.E_INVALID), ("page_size", 32, H.E_UNSUPPORTED),
                              ("pool", None, H.E_INVALID), ("pool", at + 8, H.E_INVALID), ("page_table", None, H.E_INVALID),
                              ("page_table", at + 2, H.E_INVALID)):
        old = getattr(kv, what)
        setattr(kv, what, value)
        assert L.opure_attn_window_paged(at, C.byref(window_args(fake))) == code, what
        setattr(kv, what, old)
    for name, off in (("q", 8), ("out", 4), ("seq_len", 2), ("weights", 2)):
        assert L.opure_attn_window_paged(at, C.byref(window_args(fake, **{name: at + off}))) == H.E_INVALID
        assert b"aligned" in L.opure_last_error()


def test_window_refuses_out_over_q(fake):
    L, at = H.lib(), fake[0]
    size = 2 * 4 * 8 * 64 * 2
    for off in (0, 16, size - 16, -size + 16):
        assert L.opure_attn_window_paged(at, C.byref(window_args(fake, q=at + 65536, out=at + 65536 + off))) == H.E_INVALID
        assert b"overlaps" in L.opure_last_error()


EVICT = [(dict(seq_len=None), H.E_INVALID), (dict(scores=None), H.E_INVALID), (dict(kept=None), H.E_INVALID), (dict(new_seq_len=None), H.E_INVALID),
         (dict(model=None), H.E_INVALID), (dict(kv=None), H.E_INVALID), (dict(batch=0), H.E_CAPACITY), (dict(batch=257), H.E_CAPACITY),
         (dict(max_ctx=0), H.E_CAPACITY), (dict(max_ctx=65, scores_stride=65), H.E_CAPACITY), (dict(scores_stride=63), H.E_INVALID),
         (dict(sinks=0, recent=0, heavy=0), H.E_INVALID), (dict(sinks=0xFFFFFFFF, recent=2), H.E_INVALID), (dict(freed_stride=3), H.E_INVALID)]


@pytest.mark.parametrize("kw,code", EVICT, ids=[next(iter(w[0])) + str(i) for i, w in enumerate(EVICT)])
def test_evict_refusals(fake, kw, code):
    assert H.lib().opure_kv_evict(fake[0], C.byref(evict_args(fake, **kw))) == code
    assert b"opure_kv_evict" in H.lib().opure_last_error()


def test_evict_refuses_models_and_caches(fake):
    L, (at, m, kv, _) = H.lib(), fake
    for name in ("scores", "scores_out", "kept", "seq_len", "new_seq_len", "freed", "n_freed"):
        assert L.opure_kv_evict(at, C.byref(evict_args(fake, **{name: at + 2}))) == H.E_INVALID, name
        assert b"aligned" in L.opure_last_error()
    assert L.opure_kv_evict(None, C.byref(evict_args(fake))) == H.E_INVALID
    assert L.opure_kv_evict(at, None) == H.E_INVALID
    for obj, what, value, code in ((m, "n_layers", 0, H.E_INVALID), (m, "n_kv_heads", 0, H.E_INVALID), (m, "head_dim", 40, H.E_UNSUPPORTED),
                                   (m, "afmt", 3, H.E_INVALID), (m, "rope_cos", None, H.E_INVALID), (m, "rope_sin", None, H.E_INVALID),
                                   (m, "rope_max_pos", 63, H.E_INVALID), (kv, "n_pages", 0, H.E_INVALID),
                                   (kv, "max_pages_per_seq", 0, H.E_INVALID), (kv, "page_size", 8, H.E_UNSUPPORTED),
                                   (kv, "pool", at + 8, H.E_INVALID), (kv, "page_table", None, H.E_INVALID)):
        old = getattr(obj, what)
        setattr(obj, what, value)
        assert L.opure_kv_evict(at, C.byref(evict_args(fake))) == code, what
        setattr(obj, what, old)
