"""Refusals and struct layouts of opure_kv_append, opure_attn_kv4_paged and
opure_logprobs, and the bytes of a pool (no kernel is launched: the device handle
is a placeholder that refused calls never use)."""
import ctypes as C
import os
import subprocess

import pytest

import opure_hip as H

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_header(tmp_path):
    structs = {"opure_kv_append_args": H.KvAppendArgs, "opure_attn_kv4_args": H.AttnKv4Args, "opure_logprobs_args": H.LogprobsArgs}
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
    """Addresses far apart that nothing reads: 16 MB each."""
    raw = C.create_string_buffer(8192)
    dev = (C.addressof(raw) + 255) // 256 * 256
    base = 1 << 40
    at = {n: base + (i << 24) for i, n in enumerate(("pool", "table", "len", "count", "cos", "sin", "q", "k", "v", "out", "x", "tok", "lp", "ent", "tt", "tl"))}
    m = H.Model()
    m.n_layers, m.n_heads, m.n_kv_heads, m.head_dim, m.afmt = 2, 8, 2, 64, H.A_F16
    m.rope_cos, m.rope_sin, m.rope_max_pos = at["cos"], at["sin"], 64
    kv = H.KV(at["pool"], 4, H.PAGE_SIZE, at["table"], 4)
    return dev, at, m, kv, raw


def append_args(fake, **kw):
    _, at, m, kv, _ = fake
    a = H.KvAppendArgs()
    a.model, a.kv, a.kvfmt, a.layer, a.batch, a.rows = C.pointer(m), C.pointer(kv), H.KV_I4, 0, 2, 4
    a.seq_len, a.max_ctx, a.row_count, a.rotate, a.xfmt = at["len"], 64, at["count"], 1, H.A_F16
    a.q, a.k, a.v, a.q_stride, a.k_stride, a.v_stride, a.q_out = at["q"], at["k"], at["v"], 512, 128, 128, at["out"]
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def attn_args(fake, **kw):
    _, at, m, kv, _ = fake
    a = H.AttnKv4Args(C.pointer(m), C.pointer(kv), 0, 2, 4, at["len"], 64, 16, 2, at["q"], at["out"])
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def logprob_args(fake, **kw):
    at = fake[1]
    a = H.LogprobsArgs(4, 1000, at["x"], 1000, 1.0, at["tok"], at["lp"], at["ent"], 5, at["tt"], at["tl"])
    for k, v in kw.items():
        setattr(a, k, v)
    return a


APPEND = [(dict(k=None), H.E_INVALID, b"null"), (dict(v=None), H.E_INVALID, b"null"), (dict(seq_len=None), H.E_INVALID, b"null"),
          (dict(model=None), H.E_INVALID, b"null"), (dict(kv=None), H.E_INVALID, b"null"), (dict(kvfmt=2), H.E_INVALID, b"cache format"),
          (dict(layer=2), H.E_INVALID, b"layer"), (dict(batch=0), H.E_CAPACITY, b"sequences"), (dict(batch=257), H.E_CAPACITY, b"sequences"),
          (dict(rows=0), H.E_CAPACITY, b"rows"), (dict(rows=2049), H.E_CAPACITY, b"rows"), (dict(max_ctx=0), H.E_CAPACITY, b"max_ctx"),
          (dict(max_ctx=65), H.E_CAPACITY, b"max_ctx"), (dict(max_ctx=0xFFFFFFFF), H.E_CAPACITY, b"max_ctx"),
          (dict(q=None), H.E_INVALID, b"together"), (dict(q_out=None), H.E_INVALID, b"together"), (dict(xfmt=H.A_BF16), H.E_UNSUPPORTED, b"format"),
          (dict(xfmt=3), H.E_INVALID, b"format"), (dict(q_stride=504), H.E_INVALID, b"overlap"), (dict(k_stride=120), H.E_INVALID, b"overlap"),
          (dict(v_stride=0), H.E_INVALID, b"overlap"), (dict(k_stride=132), H.E_INVALID, b"aligned"), (dict(q_stride=516), H.E_INVALID, b"aligned")]


@pytest.mark.parametrize("kw,code,word", APPEND, ids=[next(iter(w[0])) + str(i) for i, w in enumerate(APPEND)])
def test_append_refusals(fake, kw, code, word):
    assert H.lib().opure_kv_append(fake[0], C.byref(append_args(fake, **kw))) == code
    assert word in H.lib().opure_last_error()


MODELS = (("n_kv_heads", 0, H.E_INVALID), ("head_dim", 24, H.E_UNSUPPORTED), ("head_dim", 0, H.E_UNSUPPORTED), ("head_dim", 272, H.E_UNSUPPORTED),
          ("afmt", 3, H.E_INVALID), ("n_heads", 0, H.E_INVALID))


def caches(at):
    return (("n_pages", 0, H.E_INVALID), ("max_pages_per_seq", 0, H.E_INVALID), ("page_size", 32, H.E_UNSUPPORTED), ("pool", None, H.E_INVALID),
            ("pool", at["pool"] + 8, H.E_INVALID), ("page_table", None, H.E_INVALID), ("page_table", at["table"] + 2, H.E_INVALID))


def test_append_refuses_models_caches_and_addresses(fake):
    L, (dev, at, m, kv, _) = H.lib(), fake
    assert L.opure_kv_append(None, C.byref(append_args(fake))) == H.E_INVALID
    assert L.opure_kv_append(dev, None) == H.E_INVALID
    for obj, what, value, code in [(m, *x) for x in MODELS] + [(kv, *x) for x in caches(at)] + [
            (m, "rope_cos", None, H.E_INVALID), (m, "rope_sin", None, H.E_INVALID), (m, "rope_max_pos", 63, H.E_INVALID), (m, "n_layers", 0, H.E_INVALID),
            (m, "rope_cos", at["cos"] + 4, H.E_INVALID), (m, "n_heads", 1 << 16, H.E_CAPACITY)]:
        old = getattr(obj, what)
        setattr(obj, what, value)
        assert L.opure_kv_append(dev, C.byref(append_args(fake, xfmt=H.A_F32 if what == "afmt" else H.A_F16))) == code, (what, value)
        setattr(obj, what, old)
    for name, off in (("q", 8), ("k", 2), ("v", 8), ("q_out", 4), ("seq_len", 2), ("row_count", 1)):
        assert L.opure_kv_append(dev, C.byref(append_args(fake, **{name: getattr(append_args(fake), name) + off}))) == H.E_INVALID
        assert b"aligned" in L.opure_last_error()


def test_append_refuses_overlaps(fake):
    L, (dev, at, m, kv, _) = H.lib(), fake
    out, pool = 8 * 512 * 2, 2 * 4 * 2 * 640 * 2
    for name, where in (("q", at["out"] + 16), ("q", at["out"] + out - 16), ("k", at["out"]), ("v", at["out"] + 64), ("seq_len", at["out"] + out - 8),
                        ("row_count", at["out"]), ("k", at["pool"]), ("v", at["pool"] + pool - 16), ("q", at["pool"]), ("q_out", at["pool"] + pool - 16),
                        ("seq_len", at["pool"] + pool - 4), ("row_count", at["pool"]), ("q_out", at["table"]), ("q_out", at["cos"]), ("q_out", at["sin"])):
        assert L.opure_kv_append(dev, C.byref(append_args(fake, **{name: where}))) == H.E_INVALID, (name, where)
        assert b"overlaps" in L.opure_last_error(), (name, where)
    # q in place: only where it is contiguous and in the model's format
    assert L.opure_kv_append(dev, C.byref(append_args(fake, q=at["out"], q_stride=520))) == H.E_INVALID
    assert L.opure_kv_append(dev, C.byref(append_args(fake, q=at["out"], xfmt=H.A_F32))) == H.E_INVALID


def test_pool_bytes(fake):
    L, (_, _, m, _, _) = H.lib(), fake
    n = C.c_uint64()
    for hd, ng in ((16, 1), (64, 2), (80, 3), (256, 8)):
        m.head_dim = hd
        assert L.opure_kv_pool_bytes(C.byref(m), H.KV_I4, 7, C.byref(n)) == H.OK and n.value == 2 * 7 * 2 * 640 * ng
        assert L.opure_kv_pool_bytes(C.byref(m), H.KV_ACT, 7, C.byref(n)) == H.OK and n.value == 2 * 7 * 2 * 2 * 16 * hd * 2
    assert L.opure_kv_pool_bytes(None, H.KV_I4, 7, C.byref(n)) == H.E_INVALID
    assert L.opure_kv_pool_bytes(C.byref(m), H.KV_I4, 7, None) == H.E_INVALID
    assert L.opure_kv_pool_bytes(C.byref(m), 2, 7, C.byref(n)) == H.E_INVALID
    m.head_dim = 40
    assert L.opure_kv_pool_bytes(C.byref(m), H.KV_I4, 7, C.byref(n)) == H.E_UNSUPPORTED


ATTN = [(dict(q=None), H.E_INVALID, b"null"), (dict(out=None), H.E_INVALID, b"null"), (dict(seq_len=None), H.E_INVALID, b"null"),
        (dict(model=None), H.E_INVALID, b"null"), (dict(kv=None), H.E_INVALID, b"null"), (dict(layer=2), H.E_INVALID, b"layer"),
        (dict(batch=0), H.E_CAPACITY, b"sequences"), (dict(batch=257), H.E_CAPACITY, b"sequences"), (dict(rows=0), H.E_CAPACITY, b"rows"),
        (dict(rows=2049, max_ctx=2049), H.E_CAPACITY, b"rows"), (dict(max_ctx=3), H.E_CAPACITY, b"max_ctx"),
        (dict(max_ctx=65), H.E_CAPACITY, b"max_ctx"), (dict(max_ctx=0xFFFFFFFF), H.E_CAPACITY, b"max_ctx"), (dict(sinks=1 << 31), H.E_INVALID, b"sinks")]


@pytest.mark.parametrize("kw,code,word", ATTN, ids=[next(iter(w[0])) + str(i) for i, w in enumerate(ATTN)])
def test_attention_refusals(fake, kw, code, word):
    L = H.lib()
    assert L.opure_attn_kv4_paged(fake[0], C.byref(attn_args(fake, **kw))) == code
    assert word in L.opure_last_error()
    if not {"q", "out", "seq_len"} & set(kw):
        assert L.opure_attn_kv4_reserve(fake[0], C.byref(attn_args(fake, **kw))) == code


def test_attention_refuses_models_caches_and_addresses(fake):
    L, (dev, at, m, kv, _) = H.lib(), fake
    for f in (L.opure_attn_kv4_paged, L.opure_attn_kv4_reserve):
        assert f(None, C.byref(attn_args(fake))) == H.E_INVALID
        assert f(dev, None) == H.E_INVALID
        for obj, what, value, code in [(m, *x) for x in MODELS] + [(m, "n_kv_heads", 3, H.E_INVALID)] + [(kv, *x) for x in caches(at)]:
            old = getattr(obj, what)
            setattr(obj, what, value)
            assert f(dev, C.byref(attn_args(fake))) == code, (what, value)
            setattr(obj, what, old)
    for name, off in (("q", 8), ("out", 4), ("seq_len", 2)):
        assert L.opure_attn_kv4_paged(dev, C.byref(attn_args(fake, **{name: getattr(attn_args(fake), name) + off}))) == H.E_INVALID
        assert b"aligned" in L.opure_last_error()
    out, pool = 8 * 512 * 2, 2 * 4 * 2 * 640 * 2
    for name, where in (("q", at["out"]), ("q", at["out"] + out - 16), ("q", at["out"] - out + 16), ("seq_len", at["out"] + 8), ("out", at["pool"]),
                        ("out", at["pool"] + pool - 8), ("out", at["table"] + 24), ("out", at["len"])):
        assert L.opure_attn_kv4_paged(dev, C.byref(attn_args(fake, **{name: where}))) == H.E_INVALID, name
        assert b"overlaps" in L.opure_last_error()


LOGPROBS = [(dict(logits=None), H.E_INVALID, b"null"), (dict(rows=0), H.E_CAPACITY, b"rows"), (dict(rows=65536), H.E_CAPACITY, b"rows"),
            (dict(vocab=0), H.E_CAPACITY, b"vocab"), (dict(vocab=(1 << 24) + 1, logits_stride=1 << 25), H.E_CAPACITY, b"vocab"),
            (dict(top=65), H.E_CAPACITY, b"top"), (dict(vocab=4), H.E_CAPACITY, b"top"), (dict(top=0), H.E_INVALID, b"together"),
            (dict(top_tokens=None), H.E_INVALID, b"together"), (dict(top_logprobs=None), H.E_INVALID, b"together"),
            (dict(tokens=None), H.E_INVALID, b"together"), (dict(logprob=None), H.E_INVALID, b"together"),
            (dict(tokens=None, logprob=None, entropy=None, top=0, top_tokens=None, top_logprobs=None), H.E_INVALID, b"nothing"),
            (dict(temperature=0.0), H.E_INVALID, b"temperature"), (dict(temperature=-1.0), H.E_INVALID, b"temperature"),
            (dict(temperature=float("nan")), H.E_INVALID, b"temperature"), (dict(temperature=float("inf")), H.E_INVALID, b"temperature"),
            (dict(logits_stride=999), H.E_INVALID, b"logits_stride")]


@pytest.mark.parametrize("kw,code,word", LOGPROBS, ids=[next(iter(w[0])) + str(i) for i, w in enumerate(LOGPROBS)])
def test_logprobs_refusals(fake, kw, code, word):
    assert H.lib().opure_logprobs(fake[0], C.byref(logprob_args(fake, **kw))) == code
    assert word in H.lib().opure_last_error()


def test_logprobs_refuses_addresses(fake):
    L, (dev, at, _, _, _) = H.lib(), fake
    assert L.opure_logprobs(None, C.byref(logprob_args(fake))) == H.E_INVALID
    assert L.opure_logprobs(dev, None) == H.E_INVALID
    assert L.opure_logprobs_reserve(None, None) == H.E_INVALID
    assert L.opure_logprobs_reserve(dev, None) == H.E_INVALID
    for kw in (dict(rows=0), dict(vocab=0), dict(top=65)):
        assert L.opure_logprobs_reserve(dev, C.byref(logprob_args(fake, **kw))) == H.E_CAPACITY
    for name in ("logits", "tokens", "logprob", "entropy", "top_tokens", "top_logprobs"):
        assert L.opure_logprobs(dev, C.byref(logprob_args(fake, **{name: getattr(logprob_args(fake), name) + 2}))) == H.E_INVALID
        assert b"aligned" in L.opure_last_error()
    for name, where in (("logprob", at["x"] + 15996), ("entropy", at["lp"] + 12), ("top_tokens", at["tok"] + 12), ("top_logprobs", at["tt"] + 76),
                        ("tokens", at["lp"]), ("logits", at["tl"] + 76), ("top_logprobs", at["ent"])):
        assert L.opure_logprobs(dev, C.byref(logprob_args(fake, **{name: where}))) == H.E_INVALID, name
        assert b"overlaps" in L.opure_last_error()
