"""The operators that keep a long paged cache short, as cases to time: in plain
torch, or (`own`) through the framework's entry points.

  attention  opure_attn_window_paged: a row at position p sees the positions
             t <= p with t < sinks or t > p - window (window 0: all of them);
             with `weights`, what each position got from all rows and query
             heads of a KV head is added to that head's fp32 sums
  evict      opure_kv_evict: of every (sequence, layer, KV head) the first
             `sinks` positions stay, the last `recent` and the `heavy` others of
             the largest sums (ties: the lowest position); keys and values move
             up to the front of their pages, keys turned by RoPE to where they
             then stand

The cache is the framework's: pages of 16 tokens, K planes [16][hd], V planes
[hd][16], a page table a sequence.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
THETA = 500000.0

# head layouts of the three models that the benchmark's configurations name
M135 = dict(heads=9, kv=3, hd=64, a="f32")
ONE_B = dict(heads=32, kv=8, hd=64, a="f16")
EIGHT_B = dict(heads=32, kv=8, hd=128, a="bf16")


def listed():
    return [
        # one new token of one sequence, the window that a 1B model's chat keeps: latency alone
        dict(name="window decode 1b", kind="attention", **ONE_B, batch=1, rows=1, ctx=2000, ragged=0, window=1024,
             sinks=4, weights=False),
        # a server's batch of new tokens, contexts from 1k to 16k behind a 4k window
        dict(name="window decode 8b batch", kind="attention", **EIGHT_B, batch=32, rows=1, ctx=16384, ragged=1024,
             window=4096, sinks=4, weights=False),
        # a speculative step's rows of the smallest model, fp32 throughout, a window that ends inside a page
        dict(name="window verify 135m f32", kind="attention", **M135, batch=1, rows=5, ctx=1900, ragged=0, window=500,
             sinks=3, weights=False),
        # a batch of speculative steps, heads neither 64 nor 128 wide
        dict(name="window verify hd96 batch", kind="attention", heads=32, kv=8, hd=96, a="f16", batch=12, rows=7,
             ctx=3001, ragged=300, window=1000, sinks=5, weights=False),
        # a prompt's part behind a cache that is longer than the window
        dict(name="window prompt 8b", kind="attention", **EIGHT_B, batch=1, rows=2048, ctx=6000, ragged=0, window=4096,
             sinks=4, weights=False),
        # a new request's prompt of an odd length, a short window
        dict(name="window prompt 1b", kind="attention", **ONE_B, batch=1, rows=1437, ctx=0, ragged=0, window=512,
             sinks=4, weights=False),
        # one new token over a whole cache whose weights decide what stays
        dict(name="weights decode 1b", kind="attention", **ONE_B, batch=1, rows=1, ctx=8000, ragged=0, window=0,
             sinks=0, weights=True),
        # the same for a server's batch
        dict(name="weights decode 8b batch", kind="attention", **EIGHT_B, batch=16, rows=1, ctx=8000, ragged=2000,
             window=0, sinks=0, weights=True),
        # the first sums: a prompt's rows over themselves
        dict(name="weights prompt 1b", kind="attention", **ONE_B, batch=1, rows=1024, ctx=0, ragged=0, window=0,
             sinks=0, weights=True),
        # a batch of speculative steps that does both
        dict(name="weights verify 8b", kind="attention", **EIGHT_B, batch=4, rows=6, ctx=5000, ragged=0, window=2048,
             sinks=4, weights=True),
        # a 1B model's whole cache of one sequence, halved
        dict(name="evict 1b", kind="evict", kv=8, hd=64, a="f16", layers=16, batch=1, ctx=2048, ragged=0, sinks=4,
             recent=512, heavy=508, turn=True),
        # ragged sequences of a large model cut to one size
        dict(name="evict 8b batch", kind="evict", kv=8, hd=128, a="bf16", layers=32, batch=3, ctx=8000, ragged=3500,
             sinks=4, recent=1000, heavy=1500, turn=True),
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of lo..hi."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges: decoding, speculative rows or a
    prompt, any head size, windows and sinks of any length; evictions."""
    kind = rng.choice(["decode", "decode", "verify", "verify", "prompt", "prompt", "evict", "evict"])
    kv = rng.choice([1, 2, 3, 4, 8, 8])
    hd = rng.choice([16, 32, 48, 64, 64, 80, 96, 112, 128, 128, 160, 192, 256])
    a = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    if kind == "evict":
        layers, batch, ctx = _log(rng, 1, 32), _log(rng, 1, 8), _log(rng, 64, 8000)
        while layers * batch * ctx * kv * hd > 32 * 3 * 5000 * 8 * 128:
            layers = max(1, layers // 2)
            ctx = max(64, ctx // 2)
        keep = rng.randint(max(8, ctx // 8), max(9, 3 * ctx // 4))
        recent = rng.randint(1, keep - 5)
        return dict(kind="evict", kv=kv, hd=hd, a=a, layers=layers, batch=batch, ctx=ctx, ragged=max(8, ctx // rng.randint(1, 4)),
                    sinks=rng.randint(0, 4), recent=recent, heavy=keep - 4 - recent, turn=rng.random() < 0.8)
    heads = kv * rng.choice([1, 2, 3, 4, 4, 8])
    if kind == "prompt":
        rows, ctx, batch = _log(rng, 17, 2048), rng.choice([0, _log(rng, 16, 6000)]), 1
    else:
        rows, batch, ctx = (1 if kind == "decode" else rng.randint(2, 16)), _log(rng, 1, 32), _log(rng, 64, 16384)
        while batch * ctx * kv * hd > 16 * 8000 * 8 * 128:
            ctx //= 2
        batch = min(batch, 256 // rows)
    window = rng.choice([0, _log(rng, 16, 4096), _log(rng, 16, 4096)])
    while rows * heads * hd * min(ctx + rows, window or 1 << 30) > 2048 * 32 * 128 * 3500:
        window = max(16, (window or ctx + rows) // 2)
    return dict(kind="attention", heads=heads, kv=kv, hd=hd, a=a, batch=batch, rows=rows, ctx=ctx,
                ragged=0 if kind == "prompt" else max(8, ctx // rng.randint(1, 16)), window=window,
                sinks=rng.choice([0, rng.randint(1, 8), _log(rng, 8, 100)]) if window else 0, weights=rng.random() < 0.4)


# ---- inputs --------------------------------------------------------------------


def _gen(seed, stream):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + stream * 7919 + 17) & 0x7FFFFFFFFFFFFFFF)


def _lens(case):
    """Cached tokens of each sequence: a ragged batch spreads from ragged to ctx
    evenly over the logarithm, in no order."""
    n = case["batch"]
    if not case["ragged"] or n == 1:
        return [case["ctx"]] * n
    lens = [round(case["ragged"] * (case["ctx"] / case["ragged"]) ** (i / (n - 1))) for i in range(n)]
    return [lens[i] for i in np.random.RandomState(n).permutation(n)]


def _cache(case, seed, layers, rows):
    """A paged cache filled to the sequences' lengths and the call's rows, its pages in no order."""
    lens = _lens(case)
    need = [(n + rows + PAGE - 1) // PAGE for n in lens]
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(int(seed) + 5)).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    pool = torch.randn(layers, sum(need), 2, case["kv"], PAGE * case["hd"], generator=_gen(seed, 2), device="cuda",
                       dtype=DTYPE[case["a"]])
    return dict(case, pool=pool, table=table.cuda(), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                max_ctx=max(lens) + rows)


def _angles(positions, hd):
    """RoPE angles, in 64 bits, of pairs (2i, 2i + 1)."""
    return positions[..., None].double() * THETA ** (-2.0 * torch.arange(hd // 2, device=positions.device).double() / hd)


def prepare(case, seed):
    if case["kind"] == "evict":
        st = _cache(case, seed, case["layers"], 0)
        # sums as decoding leaves them: a few positions far above the rest
        shape = (case["batch"], case["layers"], case["kv"], st["max_ctx"])
        st["scores"] = torch.randn(*shape, generator=_gen(seed, 3), device="cuda").mul_(1.5).exp_()
        st["scores_out"] = torch.zeros_like(st["scores"])
        keep = case["sinks"] + case["recent"] + case["heavy"]
        st["kept"] = torch.full((*shape[:3], keep), -1, dtype=torch.int32, device="cuda")
        st["new_lens"] = torch.zeros_like(st["lens"])
        ang = _angles(torch.arange(st["max_ctx"], device="cuda"), case["hd"])
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        return st
    st = _cache(case, seed, 1, case["rows"])
    q = torch.randn(case["batch"] * case["rows"], case["heads"] * case["hd"], generator=_gen(seed, 3), device="cuda")
    st["q"] = q.mul_(1.5).to(DTYPE[case["a"]])
    st["out"] = torch.empty_like(st["q"])
    if case["weights"]:
        st["sums"] = torch.rand(case["batch"], case["kv"], st["max_ctx"], generator=_gen(seed, 4), device="cuda").mul_(4)
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
    m = H.Model()
    m.n_layers, m.n_kv_heads, m.head_dim = st["pool"].shape[0], st["kv"], st["hd"]
    m.n_heads = st.get("heads", st["kv"])
    m.attn_scale, m.afmt = st["hd"] ** -0.5, {"f32": H.A_F32, "f16": H.A_F16, "bf16": H.A_BF16}[st["a"]]
    kv = H.KV(st["pool"].data_ptr(), st["pool"].shape[1], PAGE, st["table"].data_ptr(), st["table"].shape[1])
    if st["kind"] == "evict":
        m.rope_cos, m.rope_sin, m.rope_max_pos = st["cos"].data_ptr(), st["sin"].data_ptr(), st["cos"].shape[0]
        a = H.EvictArgs()
        a.scores, a.scores_out, a.scores_stride = st["scores"].data_ptr(), st["scores_out"].data_ptr(), st["max_ctx"]
        a.sinks, a.recent, a.heavy, a.turn = st["sinks"], st["recent"], st["heavy"], int(st["turn"])
        a.kept, a.new_seq_len = st["kept"].data_ptr(), st["new_lens"].data_ptr()
    else:
        a = H.AttnWindowArgs()
        a.layer, a.rows, a.window, a.sinks = 0, st["rows"], st["window"], st["sinks"]
        a.q, a.out = st["q"].data_ptr(), st["out"].data_ptr()
        if st["weights"]:
            a.weights, a.weights_stride = st["sums"].data_ptr(), st["max_ctx"]
            a.weights_batch_stride = st["kv"] * st["max_ctx"]
    a.model, a.kv, a.batch = C.pointer(m), C.pointer(kv), st["batch"]
    a.seq_len, a.max_ctx = st["lens"].data_ptr(), st["max_ctx"]
    return a, C.byref(a)


def _own(st):
    H, dev = _framework()
    if "args" not in st:
        st["args"] = _descriptors(st)
    if st["kind"] == "evict":
        H.check(H.lib().opure_kv_evict(dev.h, st["args"][1]))
        return dict(pool=st["pool"], kept=st["kept"], scores=st["scores_out"], lens=st["new_lens"])
    H.check(H.lib().opure_attn_window_paged(dev.h, st["args"][1]))
    return dict(out=st["out"], sums=st["sums"]) if st["weights"] else dict(out=st["out"])


# ---- the plain forms -----------------------------------------------------------


def _attention(st):
    """softmax(scale q K^T) V in 32 bits over the positions that some row of a sequence sees."""
    B, R, kv, hd, G = st["batch"], st["rows"], st["kv"], st["hd"], st["heads"] // st["kv"]
    w, sinks, n_ctx = st["window"] or 1 << 30, st["sinks"], st["max_ctx"]
    lens = st["lens"].long()[:, None]
    if w + sinks + R >= n_ctx:
        pos = torch.arange(n_ctx, device="cuda").expand(B, -1)
    else:
        pos = torch.cat([torch.arange(sinks, device="cuda").expand(B, -1),
                         (lens - w + 1).clamp(min=sinks) + torch.arange(w + R - 1, device="cuda")], 1)
    there = pos < lens + R
    pos = torch.where(there, pos, 0)
    page = st["table"].long().gather(1, pos // PAGE)
    pool = st["pool"][0]
    k = pool.view(-1, 2, kv, PAGE, hd)[page, 0, :, pos % PAGE].float().permute(0, 2, 3, 1).contiguous()     # B kv hd n
    v = pool.view(-1, 2, kv, hd, PAGE)[page, 1, :, :, pos % PAGE].float().permute(0, 2, 1, 3).contiguous()  # B kv n hd
    at = lens + torch.arange(R, device="cuda")                                                              # B R
    sees = there[:, None] & (pos[:, None] <= at[..., None]) & ((pos[:, None] < sinks) | (pos[:, None] > at[..., None] - w))
    q = st["q"].float().view(B, R, kv, G, hd).permute(0, 2, 1, 3, 4).reshape(B, kv, R * G, hd)
    s = torch.matmul(q * hd ** -0.5, k)
    s = s.masked_fill(~sees.repeat_interleave(G, 1)[:, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp_()
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p, v).view(B, kv, R, G, hd).permute(0, 2, 1, 3, 4)
    out = o.reshape(B * R, -1).to(st["q"].dtype)
    if not st["weights"]:
        return dict(out=out)
    st["sums"].scatter_add_(2, pos[:, None].expand(-1, kv, -1), p.sum(2))
    return dict(out=out, sums=st["sums"])


def _evict(st):
    """Selection by a stable sort, then gathers, the turn in 32 bits, and scatters."""
    B, L, kv, hd, N = st["batch"], st["layers"], st["kv"], st["hd"], st["max_ctx"]
    sinks, recent, heavy = st["sinks"], st["recent"], st["heavy"]
    lens, t = st["lens"].long(), torch.arange(N, device="cuda")
    fixed = (t < sinks) | (t >= lens[:, None] - recent)                       # B N
    inside = t < lens[:, None]
    free = (inside & ~fixed)[:, None, None]
    order = torch.where(free, st["scores"], -math.inf).sort(dim=-1, descending=True, stable=True).indices[..., :heavy]
    chosen = torch.zeros_like(st["scores"], dtype=torch.bool).scatter_(-1, order, True) & free
    stay = chosen | (fixed & inside)[:, None, None]                           # B L kv N
    count = lens.clamp(max=sinks + recent + heavy)
    kept = torch.where(stay, t, N).sort(-1).values[..., :st["kept"].shape[-1]]
    kept = torch.cat([kept, kept.new_full((B, L, kv, st["kept"].shape[-1] - kept.shape[-1]), N)], -1)
    there = kept < N
    src = torch.where(there, kept, 0)
    dst = torch.arange(kept.shape[-1], device="cuda")
    table = st["table"].long()
    batch, layer, head = (torch.arange(n, device="cuda").view(s) for n, s in ((B, (-1, 1, 1, 1)), (L, (1, -1, 1, 1)), (kv, (1, 1, -1, 1))))
    page, slot = table[batch, src // PAGE], src % PAGE
    pk, pv = st["pool"].view(L, -1, 2, kv, PAGE, hd), st["pool"].view(L, -1, 2, kv, hd, PAGE)
    k, v = pk[layer, page, 0, head, slot], pv[layer, page, 1, head, :, slot]  # B L kv n hd
    if st["turn"]:
        far = torch.where(there, src - dst, 0)
        c, s = st["cos"][far], st["sin"][far]
        x, y = k[..., 0::2].float(), k[..., 1::2].float()
        turned = torch.stack([x * c + y * s, y * c - x * s], -1).flatten(-2).to(k.dtype)
        k = torch.where((far > 0)[..., None], turned, k)
    b, l, h, i = there.nonzero(as_tuple=True)
    to = table[b, i // PAGE]
    pk[l, to, 0, h, i % PAGE] = k[b, l, h, i]
    pv[l, to, 1, h, :, i % PAGE] = v[b, l, h, i]
    st["scores_out"].copy_(torch.where(inside[:, None, None], 0.0, st["scores_out"]))
    n = min(N, kept.shape[-1])
    moved = st["scores"].gather(-1, src)[..., :n]
    st["scores_out"][..., :n] = torch.where(there[..., :n], moved, st["scores_out"][..., :n])
    st["kept"].copy_(torch.where(there, kept, -1))
    st["new_lens"].copy_(count)
    return dict(pool=st["pool"], kept=st["kept"], scores=st["scores_out"], lens=st["new_lens"])


def run(state):
    if own:
        return _own(state)
    return _evict(state) if state["kind"] == "evict" else _attention(state)


# ---- what a pass cannot do without ---------------------------------------------


def work(case):
    lens, hd, kv = _lens(case), case["hd"], case["kv"]
    eb = 4 if case["a"] == "f32" else 2
    if case["kind"] == "evict":
        keep = case["sinks"] + case["recent"] + case["heavy"]
        planes = case["layers"] * kv
        moved = sum(min(n, keep) - case["sinks"] for n in lens if n > keep) * planes
        # K and V of what moves, read and written; the sums, the kept positions and sums
        return {"bytes": moved * 2 * 2 * hd * eb + sum(lens) * planes * 4 + sum(min(n, keep) for n in lens) * planes * 8,
                "flops": 4 * moved * hd}
    w, sinks, R, G = case["window"] or 1 << 30, case["sinks"], case["rows"], case["heads"] // kv
    j = np.arange(R)
    read = pairs = 0
    for n in lens:
        p = n + j + 1                                    # positions up to the row's own
        near = np.minimum(p, w)
        pairs += int((near + np.minimum(sinks, p - near)).sum())
        low = max(0, n - w + 1)
        read += n + R - low + min(sinks, low)
    b = read * kv * 2 * hd * eb + 2 * len(lens) * R * case["heads"] * hd * eb
    if case["weights"]:
        b += read * kv * 8
    return {"bytes": b, "flops": 4 * pairs * case["heads"] * hd}


# ---- the definition in 64 bits -------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_evict(st) if case["kind"] == "evict" else _exact_attention(st)


def _plane(st, layer, b, h, which, n):
    """K or V of one head's first n positions, [n][hd], as stored."""
    hd = st["hd"]
    page = st["pool"][layer, st["table"][b, :(n + PAGE - 1) // PAGE].long(), which, h]
    page = page.view(-1, PAGE, hd) if which == 0 else page.view(-1, hd, PAGE).transpose(1, 2)
    return page.reshape(-1, hd)[:n]


def _exact_attention(st):
    R, kv, hd, G = st["rows"], st["kv"], st["hd"], st["heads"] // st["kv"]
    lens = st["lens"].tolist()
    out = torch.zeros(len(lens), R, kv, G, hd, dtype=torch.float64, device="cuda")
    sums = st["sums"].double() if st["weights"] else None
    q = st["q"].double().view(len(lens), R, kv, G, hd)
    for b, n in enumerate(lens):
        p, t = torch.arange(n, n + R, device="cuda")[:, None], torch.arange(n + R, device="cuda")[None]
        hidden = (t > p) | ((t >= st["sinks"]) & (t <= p - st["window"]) if st["window"] else t > p)
        for h in range(kv):
            k, v = (_plane(st, 0, b, h, i, n + R).double() for i in (0, 1))
            for g in range(G):
                s = (q[b, :, h, g] @ k.T.contiguous()) / math.sqrt(hd)
                e = torch.softmax(s.masked_fill(hidden, -math.inf), 1)
                out[b, :, h, g] = e @ v
                if sums is not None:
                    sums[b, h, :n + R] += e.sum(0)
    out = out.reshape(len(lens) * R, -1)
    return dict(out=out, sums=sums) if st["weights"] else dict(out=out)


def _exact_evict(st):
    lens, hd = st["lens"].tolist(), st["hd"]
    keep = st["sinks"] + st["recent"] + st["heavy"]
    pool, scores = st["pool"].double(), torch.zeros_like(st["scores"], dtype=torch.float64)
    freq = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    for b, n in enumerate(lens):
        pages = st["table"][b].long()
        for layer in range(st["layers"]):
            for h in range(st["kv"]):
                s = st["scores"][b, layer, h, :n].double()
                if n > keep:
                    mid = s[st["sinks"]:n - st["recent"]]
                    best = mid.sort(descending=True, stable=True).indices[:st["heavy"]].sort().values + st["sinks"]
                    idx = torch.cat([torch.arange(st["sinks"], device="cuda"), best, torch.arange(n - st["recent"], n, device="cuda")])
                    k, v = (_plane(st, layer, b, h, i, n)[idx].double() for i in (0, 1))
                    to = torch.arange(keep, device="cuda")
                    if st["turn"]:
                        z = torch.view_as_complex(k.reshape(keep, hd // 2, 2).contiguous())
                        z = z * torch.polar(torch.ones_like(freq), (to - idx)[:, None] * freq)
                        k = torch.view_as_real(z).reshape(keep, hd)
                    pool[layer, :, 0, h].view(-1, PAGE, hd)[pages[to // PAGE], to % PAGE] = k
                    pool[layer, :, 1, h].view(-1, hd, PAGE)[pages[to // PAGE], :, to % PAGE] = v
                    s = s[idx]
                scores[b, layer, h, :len(s)] = s
    # whole numbers are compared with the plain form's
    return dict(pool=pool, kept=None, scores=scores, lens=None)
