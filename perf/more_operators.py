"""The operators of a step over a paged cache that may be held in 4 bits, as cases
to time: in plain torch, or (`own`) through the framework's entry points.

  append     opure_kv_append: the rows of one projection's output [q | k | v] turned
             to their positions (q, k), q kept in the model's format, k and v
             written to a layer of the cache, in the model's format or in 4 bits
  attention  opure_attn_kv4_paged: a row at position p sees the positions t <= p
             of a 4-bit cache with t < sinks or t > p - window (window 0: all)
  logprobs   opure_logprobs: of each row of logits the log probability of a given
             token, the entropy and the `top` most probable tokens (ties: the
             lowest) with theirs

The cache is the framework's: pages of 16 tokens, a page table a sequence.  In the
model's format a page holds K planes [16][hd] and V planes [hd][16].  In 4 bits it
holds, for each KV head and with ng = ceil(hd / 32) groups of 32 channels,
  K codes  uint32 [j 4][token 16][ng]: channels 32 g + 8 j + 2 n + h at bit 16 h + 4 n
  V codes  uint32 [j 4][c 16][ng]: channels 32 g + 16 T + c of the tokens
           4 j + 2 m + h at bit 16 h + 8 T + 4 m
  K        fp16 [token 16][ng][scale, base]
  V        fp16 [j 4][ng][scale, base][token 4 j ..]
and a code c stands for the fp16 number nearest to scale (16 + c) + base.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
THETA = 500000.0
MOST = 16384.0                                     # magnitudes past it are held as it

# head layouts and vocabularies of the models that the benchmark's configurations name
M135 = dict(heads=9, kv=3, hd=64, a="f32")
ONE_B = dict(heads=32, kv=8, hd=64, a="f16")
EIGHT_B = dict(heads=32, kv=8, hd=128, a="bf16")


def listed():
    return [
        # one new token of one sequence of a 1B model: latency alone
        dict(name="append decode 1b", kind="append", **ONE_B, x="f16", i4=False, batch=1, rows=1, ctx=2000, ragged=0, short=False),
        # a server's batch of speculative steps, fp32 accumulators in, a 4-bit cache
        dict(name="append verify 8b batch i4", kind="append", **EIGHT_B, x="f32", i4=True, batch=32, rows=5, ctx=8185, ragged=512, short=False),
        # a part of a prompt, and one that begins and ends inside a page and whose batch is padded
        dict(name="append prompt 8b", kind="append", **EIGHT_B, x="bf16", i4=False, batch=1, rows=2048, ctx=6000, ragged=0, short=False),
        dict(name="append prompt 1b i4", kind="append", **ONE_B, x="f16", i4=True, batch=3, rows=1437, ctx=700, ragged=13, short=True),
        # one new token over a 4-bit cache
        dict(name="attention i4 decode 1b", kind="attention", **ONE_B, batch=1, rows=1, ctx=2000, ragged=0, window=0, sinks=0),
        # a server's batch of new tokens, contexts from 1k to 16k
        dict(name="attention i4 decode 8b batch", kind="attention", **EIGHT_B, batch=32, rows=1, ctx=16384, ragged=1024, window=0, sinks=0),
        # a speculative step's rows of the smallest model, fp32 activations
        dict(name="attention i4 verify 135m f32", kind="attention", **M135, batch=1, rows=5, ctx=1900, ragged=0, window=0, sinks=0),
        # a batch of speculative steps behind a window, heads neither 64 nor 128 wide
        dict(name="attention i4 verify hd80 batch", kind="attention", heads=32, kv=8, hd=80, a="f16", batch=12, rows=7, ctx=3001,
             ragged=300, window=1000, sinks=5),
        # a prompt's part behind a cache
        dict(name="attention i4 prompt 8b", kind="attention", **EIGHT_B, batch=1, rows=2048, ctx=6000, ragged=0, window=0, sinks=0),
        # one sampled token's log probability and alternatives
        dict(name="logprobs decode 128k", kind="logprobs", rows=1, vocab=128256, top=20, masked=False),
        # a batch's, under a grammar that leaves few tokens
        dict(name="logprobs batch 49k masked", kind="logprobs", rows=48, vocab=49152, top=5, masked=True),
        # a prompt scored: every row's next token
        dict(name="logprobs prompt 128k", kind="logprobs", rows=1500, vocab=128256, top=1, masked=False),
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of lo..hi."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges: any head size and format, one row
    to a prompt's, windows and sinks of any length, vocabularies of any size."""
    kind = rng.choice(["append", "attention", "attention", "logprobs"])
    if kind == "logprobs":
        rows, vocab = _log(rng, 1, 1500), _log(rng, 300, 128256)
        return dict(kind=kind, rows=rows, vocab=vocab, top=min(vocab, rng.choice([0, 1, _log(rng, 2, 32), _log(rng, 2, 32)])),
                    masked=rng.random() < 0.3)
    kv = rng.choice([1, 2, 3, 4, 8, 8])
    hd = rng.choice([16, 32, 48, 64, 64, 80, 96, 112, 128, 128, 160, 192, 256])
    a = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    heads = kv * rng.choice([1, 2, 3, 4, 4, 8])
    shape = rng.choice(["decode", "verify", "prompt"])
    if shape == "prompt":
        rows, batch, ctx = _log(rng, 17, 2048), rng.choice([1, 1, 2, 3]), rng.choice([0, _log(rng, 16, 6000)])
        while rows * batch * heads * hd > 2048 * 32 * 128:
            rows, batch = max(17, rows // 2), 1
            heads = kv * max(1, heads // kv // 2) if rows == 17 else heads
    else:
        rows, batch, ctx = (1 if shape == "decode" else rng.randint(2, 16)), _log(rng, 1, 32), _log(rng, 64, 16384)
        batch = min(batch, 256 // rows)
        while batch * ctx * kv * hd > 32 * 5900 * 8 * 128:
            ctx //= 2
    ragged = max(1, ctx // rng.randint(1, 16)) if batch > 1 else 0
    if kind == "append":
        return dict(kind=kind, heads=heads, kv=kv, hd=hd, a=a, x=rng.choice(["f32", a, a]), i4=rng.random() < 0.6, batch=batch, rows=rows,
                    ctx=ctx, ragged=ragged, short=rows > 16 and rng.random() < 0.5)
    window = rng.choice([0, 0, _log(rng, 16, 4096)])
    while rows * batch * heads * hd * min(ctx + rows, window or 1 << 30) > 2048 * 32 * 128 * 6500:
        window = max(16, (window or ctx + rows) // 2)
    return dict(kind=kind, heads=heads, kv=kv, hd=hd, a=a, batch=batch, rows=rows, ctx=ctx, ragged=ragged, window=window,
                sinks=rng.choice([0, rng.randint(1, 8), _log(rng, 8, 100)]) if window else 0)


# ---- inputs --------------------------------------------------------------------


def _gen(seed, stream):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + stream * 7919 + 29) & 0x7FFFFFFFFFFFFFFF)


def _lens(case):
    """Cached tokens of each sequence: a ragged batch spreads from ragged to ctx
    evenly over the logarithm, in no order."""
    n = case["batch"]
    if not case["ragged"] or n == 1:
        return [case["ctx"]] * n
    lens = [round(case["ragged"] * (case["ctx"] / case["ragged"]) ** (i / (n - 1))) for i in range(n)]
    return [lens[i] for i in np.random.RandomState(n).permutation(n)]


def _counts(case):
    """Rows of each sequence: of a padded batch all of them, two thirds, a third."""
    return [case["rows"] * (3 - b % 3) // 3 if case["short"] else case["rows"] for b in range(case["batch"])]


def _table(case, seed):
    """A page table for the sequences' positions and the call's rows, its pages in no order."""
    need = [(n + case["rows"] + PAGE - 1) // PAGE for n in _lens(case)]
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(int(seed) + 5)).to(torch.int32)
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table.cuda(), sum(need)


def _paged(case, seed):
    table, pages = _table(case, seed)
    lens = _lens(case)
    return dict(case, table=table, pages=pages, ng=(case["hd"] + 31) // 32, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                max_ctx=max(lens) + case["rows"])


def _i4_views(st, pool):
    """The codes (as words) and the scales and bases of a 4-bit pool [...][kv][160 ng]."""
    ng = st["ng"]
    return dict(codes=pool[..., :128 * ng], scales=pool[..., 128 * ng:].view(torch.float16))


def prepare(case, seed):
    if case["kind"] == "logprobs":
        R, V = case["rows"], case["vocab"]
        x = torch.randn(R, V, generator=_gen(seed, 1), device="cuda").mul_(2.5)
        # a model is sure of a few tokens: one in a hundred stands out
        x += torch.rand(R, V, generator=_gen(seed, 2), device="cuda").sub_(0.99).clamp_(min=0).mul_(800)
        if case["masked"]:
            x.masked_fill_(torch.rand(R, V, generator=_gen(seed, 3), device="cuda") < 0.95, -math.inf)
        st = dict(case, logits=x, tokens=torch.randint(0, V, (R,), generator=_gen(seed, 4), device="cuda", dtype=torch.int32))
        st["logprob"], st["entropy"] = (torch.empty(R, device="cuda") for _ in range(2))
        st["top_tokens"] = torch.empty(R, case["top"], dtype=torch.int32, device="cuda")
        st["top_logprobs"] = torch.empty(R, case["top"], device="cuda")
        return st
    st = _paged(case, seed)
    kv, hd, ng, dt = case["kv"], case["hd"], st["ng"], DTYPE[case["a"]]
    if case["kind"] == "append":
        n = case["batch"] * case["rows"]
        x = torch.randn(n, (case["heads"] + 2 * kv) * hd, generator=_gen(seed, 1), device="cuda")
        # keys have channels that stand apart
        x[:, case["heads"] * hd:(case["heads"] + kv) * hd] += torch.randn(kv * hd, generator=_gen(seed, 2), device="cuda").mul_(1.5)
        st["qkv"] = x.to(DTYPE[case["x"]])
        st["q"] = torch.zeros(n, case["heads"] * hd, device="cuda", dtype=dt)
        if case["short"]:
            st["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device="cuda")
        ang = _angles(torch.arange(st["max_ctx"], device="cuda"), hd)
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        if case["i4"]:
            st["pool"] = torch.randint(-1 << 31, 1 << 31, (1, st["pages"], kv, 160 * ng), generator=_gen(seed, 3), device="cuda").to(torch.int32)
            st["out"] = _i4_views(st, st["pool"])
            st["out"]["scales"].copy_(torch.randn(st["out"]["scales"].shape, generator=_gen(seed, 4), device="cuda"))
        else:
            st["pool"] = torch.randn(1, st["pages"], 2, kv, PAGE * hd, generator=_gen(seed, 3), device="cuda", dtype=dt)
            st["out"] = dict(pool=st["pool"])
        return st
    # a 4-bit cache of normal keys and values, keys with channels that stand apart
    st["pool"] = torch.zeros(1, st["pages"], kv, 160 * ng, dtype=torch.int32, device="cuda")
    bias = torch.randn(kv, hd, generator=_gen(seed, 2), device="cuda").mul_(1.5)
    g = _gen(seed, 1)
    for at in range(0, st["pages"], 4096):
        n = min(4096, st["pages"] - at)
        k, v = (torch.randn(n, PAGE, kv, hd, generator=g, device="cuda") for _ in range(2))
        ck, sk, bk = _quantise(k + bias, ng)
        cv, sv, bv = _quantise(v, ng)
        st["pool"][0, at:at + n] = _pack(ck.transpose(1, 2), cv.transpose(1, 2), *(y.transpose(1, 2) for y in (sk, bk, sv, bv)))
    q = torch.randn(case["batch"] * case["rows"], case["heads"] * hd, generator=_gen(seed, 3), device="cuda")
    st["q"] = q.to(dt)
    st["out"] = torch.empty_like(st["q"])
    return st


# ---- the framework's calls -----------------------------------------------------

_dev = None


def _framework():
    """The binding and the process's one device handle: calls queue on its stream as a program's would."""
    global _dev
    import os
    import sys
    if _dev is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "opure-voxelengine_amd"))
        import opure_hip
        _dev = (opure_hip, opure_hip.Dev(0))
    return _dev


def _descriptors(st):
    """The C structures that a program keeps beside its buffers."""
    import ctypes as C
    H, dev = _framework()
    if st["kind"] == "logprobs":
        a = H.LogprobsArgs()
        a.rows, a.vocab, a.logits, a.logits_stride, a.temperature = st["rows"], st["vocab"], st["logits"].data_ptr(), st["vocab"], 1.0
        a.tokens, a.logprob, a.entropy = st["tokens"].data_ptr(), st["logprob"].data_ptr(), st["entropy"].data_ptr()
        a.top = st["top"]
        if st["top"]:
            a.top_tokens, a.top_logprobs = st["top_tokens"].data_ptr(), st["top_logprobs"].data_ptr()
        return a, C.byref(a)
    fmt = {"f32": H.A_F32, "f16": H.A_F16, "bf16": H.A_BF16}
    m = H.Model()
    m.n_layers, m.n_heads, m.n_kv_heads, m.head_dim = 1, st["heads"], st["kv"], st["hd"]
    m.attn_scale, m.afmt = st["hd"] ** -0.5, fmt[st["a"]]
    kv = H.KV(st["pool"].data_ptr(), st["pages"], PAGE, st["table"].data_ptr(), st["table"].shape[1])
    if st["kind"] == "append":
        m.rope_cos, m.rope_sin, m.rope_max_pos = st["cos"].data_ptr(), st["sin"].data_ptr(), st["cos"].shape[0]
        a = H.KvAppendArgs()
        a.kvfmt, a.xfmt, a.rotate = H.KV_I4 if st["i4"] else H.KV_ACT, fmt[st["x"]], 1
        x, width = st["qkv"], st["qkv"].element_size()
        a.q, a.k = x.data_ptr(), x.data_ptr() + st["heads"] * st["hd"] * width
        a.v = a.k + st["kv"] * st["hd"] * width
        a.q_stride = a.k_stride = a.v_stride = x.shape[1]
        a.q_out = st["q"].data_ptr()
        if st["short"]:
            a.row_count = st["counts"].data_ptr()
    else:
        a = H.AttnKv4Args()
        a.window, a.sinks, a.q, a.out = st["window"], st["sinks"], st["q"].data_ptr(), st["out"].data_ptr()
    a.model, a.kv, a.layer, a.batch, a.rows = C.pointer(m), C.pointer(kv), 0, st["batch"], st["rows"]
    a.seq_len, a.max_ctx = st["lens"].data_ptr(), st["max_ctx"]
    return a, C.byref(a)


def _own(st):
    H, dev = _framework()
    if "args" not in st:
        st["args"] = _descriptors(st)
    if st["kind"] == "append":
        H.check(H.lib().opure_kv_append(dev.h, st["args"][1]))
        return dict(st["out"], q=st["q"])
    if st["kind"] == "attention":
        H.check(H.lib().opure_attn_kv4_paged(dev.h, st["args"][1]))
        return dict(out=st["out"])
    H.check(H.lib().opure_logprobs(dev.h, st["args"][1]))
    return {k: st[k] for k in ("logprob", "entropy", "top_tokens", "top_logprobs")}


# ---- the plain forms -----------------------------------------------------------


def _angles(positions, hd):
    """RoPE angles, in 64 bits, of pairs (2i, 2i + 1)."""
    return positions[..., None].double() * THETA ** (-2.0 * torch.arange(hd // 2, device=positions.device).double() / hd)


def _quantise(x, ng):
    """Codes, scales and bases of x [...][hd] in groups of 32 channels."""
    pad = 32 * ng - x.shape[-1]
    bad = torch.nn.functional.pad(~torch.isfinite(x), (0, pad)).unflatten(-1, (ng, 32)).any(-1)
    x = x.clamp(-MOST, MOST)
    last = x[..., -1:].expand(*x.shape[:-1], pad)                      # the last group's largest and smallest are its own channels'
    x = torch.cat([x, last], -1).unflatten(-1, (ng, 32))
    lo, hi = x.amin(-1), x.amax(-1)
    s = ((hi - lo) * (1.0 / 15.0)).half()
    b = (lo - 16.0 * s.float()).half()
    c = torch.round((x - b.float()[..., None]) / s.float()[..., None] - 16.0).clamp(0, 15)
    c = torch.where((s == 0)[..., None] | bad[..., None], 0.0, c).to(torch.int32).flatten(-2)
    if pad:
        c[..., -pad:] = 0
    return c, s.masked_fill(bad, math.nan), b.masked_fill(bad, math.nan)


def _pack(ck, cv, sk, bk, sv, bv):
    """Pages [...][160 ng] of codes [...][16][32 ng] and scales and bases [...][16][ng]."""
    ng, lead = sk.shape[-1], ck.shape[:-2]
    n, h = torch.arange(4, device=ck.device)[:, None], torch.arange(2, device=ck.device)
    k = (ck.unflatten(-1, (ng, 4, 4, 2)) << (4 * n + 16 * h).int()).sum((-1, -2)).to(torch.int32)                 # token g j
    k = k.movedim(-1, -3).reshape(*lead, 64 * ng)
    T, m = torch.arange(2, device=ck.device).reshape(2, 1, 1), torch.arange(2, device=ck.device)[:, None]
    v = cv.unflatten(-1, (ng, 2, 16)).unflatten(-4, (4, 2, 2))                                                    # j m h g T c
    d = v.dim()
    v = v.permute(*range(d - 6), d - 6, d - 1, d - 3, d - 2, d - 5, d - 4)                                        # j c g T m h
    v = (v << (8 * T + 4 * m + 16 * h).int()).sum((-1, -2, -3)).to(torch.int32).reshape(*lead, 64 * ng)
    ks = torch.stack([sk, bk], -1).reshape(*lead, 32 * ng).view(torch.int32)
    vs = torch.stack([sv, bv], -1).unflatten(-3, (4, 4)).movedim(-3, -1).reshape(*lead, 32 * ng).view(torch.int32)
    return torch.cat([k, v, ks, vs], -1)


def _unpack(pool, ng):
    """Codes [...][16][32 ng] of K and V, and scales and bases [...][16][ng] of both, of pages [...][160 ng]."""
    lead, dev = pool.shape[:-1], pool.device
    n, h = torch.arange(4, device=dev)[:, None], torch.arange(2, device=dev)
    k = pool[..., :64 * ng].reshape(*lead, 4, 16, ng).movedim(-3, -1)                                              # token g j
    ck = ((k[..., None, None] >> (4 * n + 16 * h).int()) & 15).reshape(*lead, 16, 32 * ng)
    T, m = torch.arange(2, device=dev).reshape(2, 1, 1), torch.arange(2, device=dev)[:, None]
    v = (pool[..., 64 * ng:128 * ng].reshape(*lead, 4, 16, ng)[..., None, None, None] >> (8 * T + 4 * m + 16 * h).int()) & 15   # j c g T m h
    d = v.dim()
    cv = v.permute(*range(d - 6), d - 6, d - 2, d - 1, d - 4, d - 3, d - 5).reshape(*lead, 16, 32 * ng)
    ks = pool[..., 128 * ng:144 * ng].contiguous().view(torch.float16).reshape(*lead, 16, ng, 2)
    vs = pool[..., 144 * ng:].contiguous().view(torch.float16).reshape(*lead, 4, ng, 2, 4).movedim(-1, -3).reshape(*lead, 16, ng, 2)
    return ck, cv, ks[..., 0], ks[..., 1], vs[..., 0], vs[..., 1]


def _values(c, s, b, hd):
    """What codes stand for, as 32-bit values."""
    x = s.float()[..., None] * (16 + c.unflatten(-1, (-1, 32))).float() + b.float()[..., None]
    return x.half().float().flatten(-2)[..., :hd]


def _rope(x, cos, sin):
    """x [rows][heads][hd] in 32 bits turned by its rows' angles."""
    e, o, c, s = x[..., 0::2], x[..., 1::2], cos[:, None], sin[:, None]
    return torch.stack([e * c - o * s, e * s + o * c], -1).flatten(-2)


def _append(st):
    B, R, heads, kv, hd, ng = st["batch"], st["rows"], st["heads"], st["kv"], st["hd"], st["ng"]
    j = torch.arange(R, device="cuda").expand(B, R)
    pos = st["lens"].long()[:, None] + j
    b, j = (j < st["counts"][:, None] if st["short"] else torch.ones_like(j, dtype=torch.bool)).nonzero(as_tuple=True)
    pos, row = pos[b, j], b * R + j
    x = st["qkv"][row].float().view(-1, heads + 2 * kv, hd)
    cos, sin = st["cos"][pos], st["sin"][pos]
    q, k, v = _rope(x[:, :heads], cos, sin), _rope(x[:, heads:heads + kv], cos, sin), x[:, heads + kv:]
    st["q"][row] = q.flatten(1).to(st["q"].dtype)
    page, slot = st["table"][b, pos // PAGE].long(), pos % PAGE
    if not st["i4"]:
        pool = st["pool"][0]
        pool.view(-1, 2, kv, PAGE, hd)[page, 0, :, slot] = k.to(pool.dtype)
        pool.view(-1, 2, kv, hd, PAGE)[page, 1, :, :, slot] = v.to(pool.dtype)
        return dict(st["out"], q=st["q"])
    # the touched pages unpacked, their new tokens put in, packed again
    touched, at = page.unique(return_inverse=True)
    parts = [y.clone() for y in _unpack(st["pool"][0, touched], ng)]
    new = [y for pair in zip(_quantise(k, ng), _quantise(v, ng)) for y in pair]
    for part, y in zip((parts[0], parts[1], parts[2], parts[4], parts[3], parts[5]), new):
        part[at, :, slot] = y.to(part.dtype)
    st["pool"][0, touched] = _pack(*parts)
    return dict(st["out"], q=st["q"])


def _attention(st):
    """softmax(scale q K^T) V in 32 bits over the positions that some row of a sequence sees."""
    B, R, kv, hd, ng, G = st["batch"], st["rows"], st["kv"], st["hd"], st["ng"], st["heads"] // st["kv"]
    w, sinks, n_ctx = st["window"] or 1 << 30, st["sinks"], st["max_ctx"]
    lens = st["lens"].long()[:, None]
    # the pages of the sinks and of the window
    cols = (n_ctx + PAGE - 1) // PAGE
    ns, nw = (sinks + PAGE - 1) // PAGE, (w + R + PAGE - 2) // PAGE + 1
    if ns + nw >= cols:
        col = torch.arange(cols, device="cuda").expand(B, -1)
    else:
        col = torch.cat([torch.arange(ns, device="cuda").expand(B, -1), (((lens - w + 1).clamp(min=0) // PAGE).clamp(min=ns)) + torch.arange(nw, device="cuda")], 1)
    pos = (col[..., None] * PAGE + torch.arange(PAGE, device="cuda")).flatten(1)                               # B n
    page = st["table"].long().gather(1, col.clamp(max=cols - 1)).clamp(min=0)
    ck, cv, sk, bk, sv, bv = _unpack(st["pool"][0, page], ng)                                                 # B pages kv 16 .
    there = pos < lens + R
    k = _values(ck, sk, bk, hd).permute(0, 2, 4, 1, 3).reshape(B, kv, hd, -1)                                 # B kv hd n
    v = _values(cv, sv, bv, hd).permute(0, 2, 1, 3, 4).reshape(B, kv, -1, hd)                                 # B kv n hd
    v = v.masked_fill(~there[:, None, :, None], 0.0)
    at = lens + torch.arange(R, device="cuda")                                                                # B R
    sees = there[:, None] & (pos[:, None] <= at[..., None]) & ((pos[:, None] < sinks) | (pos[:, None] > at[..., None] - w))
    q = st["q"].float().view(B, R, kv, G, hd).permute(0, 2, 1, 3, 4).reshape(B, kv, R * G, hd)
    s = torch.matmul(q * hd ** -0.5, k)
    s = s.masked_fill(~sees.repeat_interleave(G, 1)[:, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp_()
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p, v).view(B, kv, R, G, hd).permute(0, 2, 1, 3, 4)
    return dict(out=o.reshape(B * R, -1).to(st["q"].dtype))


def _logprobs(st):
    x = st["logits"]
    d = x - x.amax(-1, keepdim=True)
    e = d.exp()
    total = e.sum(-1)
    norm = total.log()
    entropy = norm - torch.where(e > 0, e * d, 0.0).sum(-1) / total
    logprob = d.gather(1, st["tokens"].long()[:, None])[:, 0] - norm
    # ties go to the lowest index: a stable order
    top = x.sort(dim=-1, descending=True, stable=True).indices[:, :st["top"]] if st["top"] > 1 else x.argmax(-1, keepdim=True)[:, :st["top"]]
    return dict(logprob=logprob, entropy=entropy, top_tokens=top.to(torch.int32), top_logprobs=d.gather(1, top) - norm[:, None])


def run(state):
    if own:
        return _own(state)
    return {"append": _append, "attention": _attention, "logprobs": _logprobs}[state["kind"]](state)


# ---- what a pass cannot do without ---------------------------------------------


def work(case):
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + case["rows"] * (12 + 8 * case["top"]), "flops": 5 * n}
    size = {"f32": 4, "f16": 2, "bf16": 2}
    hd, kv, heads = case["hd"], case["kv"], case["heads"]
    plane = 20 * ((hd + 31) // 32)                           # bytes of a token's K or V in 4 bits
    if case["kind"] == "append":
        n, eb, xb = sum(_counts(case)), size[case["a"]], size[case["x"]]
        held = 2 * kv * (plane if case["i4"] else hd * eb)
        # q, k and v read, a row's cosines and sines, q and the cache's slots written
        return {"bytes": n * ((heads + 2 * kv) * hd * xb + 4 * hd + heads * hd * eb + held), "flops": n * (3 * (heads + kv) + 6 * kv) * hd}
    lens, R = _lens(case), case["rows"]
    w, sinks, j = case["window"] or 1 << 30, case["sinks"], np.arange(R)
    read = pairs = 0
    for n in lens:
        p = n + j + 1                                        # positions up to the row's own
        near = np.minimum(p, w)
        pairs += int((near + np.minimum(sinks, p - near)).sum())
        low = max(0, n - w + 1)
        read += n + R - low + min(sinks, low)
    return {"bytes": read * kv * 2 * plane + 2 * len(lens) * R * heads * hd * size[case["a"]], "flops": 4 * pairs * heads * hd}


# ---- the definition in 64 bits -------------------------------------------------


def exact(case, seed):
    if case["kind"] == "logprobs" and case["rows"] * case["vocab"] > 1 << 28:
        return None
    st = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "logprobs": _exact_logprobs}[case["kind"]](st)


def _exact_append(st):
    heads, kv, hd, R = st["heads"], st["kv"], st["hd"], st["rows"]
    x = st["qkv"].double().view(st["batch"], R, heads + 2 * kv, hd)
    q = st["q"].double().view(st["batch"], R, heads, hd)
    pool = None if st["i4"] else st["pool"].double()
    for b, (n0, n) in enumerate(zip(st["lens"].tolist(), _counts(st))):
        turn = torch.complex(st["cos"][n0:n0 + n].double(), st["sin"][n0:n0 + n].double())[:, None]
        z = torch.view_as_complex(x[b, :n, :heads + kv].reshape(n, heads + kv, hd // 2, 2).contiguous())
        z = torch.view_as_real(z * turn).reshape(n, heads + kv, hd)
        q[b, :n] = z[:, :heads]
        if pool is not None:
            at = torch.arange(n0, n0 + n, device="cuda")
            pages, slot = st["table"][b].long()[at // PAGE], at % PAGE
            for h in range(kv):
                pool[0, :, 0, h].view(-1, PAGE, hd)[pages, slot] = z[:, heads + h]
                pool[0, :, 1, h].view(-1, hd, PAGE)[pages, :, slot] = x[b, :n, heads + kv + h]
    q = q.reshape(st["q"].shape)
    # a code is a whole number that 32-bit arithmetic decides: compared with the plain form's
    return dict(codes=None, scales=None, q=q) if st["i4"] else dict(pool=pool, q=q)


def _exact_plane(st, b, h, which, n):
    """K or V of one head's first n positions, [n][hd]: each value looked up by its word and bit."""
    hd, ng = st["hd"], st["ng"]
    t, d = torch.arange(n, device="cuda")[:, None], torch.arange(hd, device="cuda")[None]
    block = st["pool"][0, st["table"][b].long()[t[:, 0] // PAGE], h]                          # n 160 ng
    u = t % PAGE
    if which == 0:
        word, bit = (d % 32 // 8 * 16 + u) * ng + d // 32, 16 * (d % 2) + 4 * (d % 8 // 2)
        s_at = 256 * ng + (u * ng + d // 32) * 2
        b_at = s_at + 1
    else:
        word, bit = 64 * ng + (u // 4 * 16 + d % 16) * ng + d // 32, 16 * (u % 2) + 8 * (d % 32 // 16) + 4 * (u % 4 // 2)
        s_at = 288 * ng + (u // 4 * ng + d // 32) * 8 + u % 4
        b_at = s_at + 4
    code = (block.gather(1, word) >> bit) & 15
    half = block.view(torch.float16)
    return (half.gather(1, s_at).double() * (16 + code).double() + half.gather(1, b_at).double()).half().double()


def _exact_attention(st):
    R, kv, hd, G = st["rows"], st["kv"], st["hd"], st["heads"] // st["kv"]
    lens = st["lens"].tolist()
    out = torch.zeros(len(lens), R, kv, G, hd, dtype=torch.float64, device="cuda")
    q = st["q"].double().view(len(lens), R, kv, G, hd)
    for b, n in enumerate(lens):
        p, t = torch.arange(n, n + R, device="cuda")[:, None], torch.arange(n + R, device="cuda")[None]
        hidden = (t > p) | ((t >= st["sinks"]) & (t <= p - st["window"]) if st["window"] else t > p)
        for h in range(kv):
            k, v = (_exact_plane(st, b, h, i, n + R) for i in (0, 1))
            for g in range(G):
                s = (q[b, :, h, g] @ k.T.contiguous()) / math.sqrt(hd)
                out[b, :, h, g] = torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ v
    return dict(out=out.reshape(len(lens) * R, -1))


def _exact_logprobs(st):
    rows = []
    for x, token in zip(st["logits"], st["tokens"].tolist()):
        x = x.double()
        lp = x - torch.logsumexp(x, 0)
        p = lp.exp()
        best = torch.topk(lp, st["top"]).values if st["top"] else lp[:0]
        rows.append((lp[token], -(p[p > 0] * lp[p > 0]).sum(), best))
    logprob, entropy, best = (torch.stack(y) for y in zip(*rows))
    # whole numbers are compared with the plain form's
    return dict(logprob=logprob, entropy=entropy, top_tokens=None, top_logprobs=best)
