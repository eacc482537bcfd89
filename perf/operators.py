"""The serving operators of fftsparse_amd as cases that can be timed and compared.

What a server does after the prefill, step by step: block tables and slot maps
from the requests' lengths (``plan_step``), the rotary embedding of the new
tokens with their keys and values written into a paged cache (``rope_cache``;
``rope`` alone for a prompt that is not cached in pages), attention of the new
tokens over the cache (``paged_attention``: single tokens, chunks, both at
once, with or without a sliding window and its first tokens), and that window
over a whole prompt (``window_attention``).  Head counts are those of the
benchmark configurations (32 / 8, 28 / 4, 4 / 1).

Where ``own`` is false ``run`` computes the same in elementary torch operations,
in 32 bits (angles in 64).
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEV = "cuda"


def _case(name, op, **kw):
    c = dict(op=op, B=1, Lmin=1, Lmax=1024, new=1, kind="decode", ps=64, Hq=32, Hk=8, D=128, dtype="bf16",
             window=0, sinks=0, layout="nhd", rot=128, interleaved=False, scale=1.0)
    assert set(kw) <= set(c), set(kw) - set(c)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one decoding step of a small batch: nothing but latency
        _case("plan-decode", "plan", B=48, Lmin=100, Lmax=8192, ps=64),
        # chunks of new prompts beside decoding requests, some of them finished or rolled back, in small pages
        _case("plan-mixed", "plan", B=500, Lmin=30, Lmax=30000, new=1000, kind="mixed", ps=16),
        # the new tokens of that decoding step, rotated and written to the cache
        _case("rope-cache-decode", "rope_cache", B=48, Lmin=100, Lmax=8192, ps=64),
        # a long chunk of one prompt, half of each head rotated in interleaved pairs, pages with a head's rows together
        _case("rope-cache-chunk", "rope_cache", Lmin=40000, Lmax=40000, new=8191, kind="chunk", ps=128, Hq=28, Hk=4,
              dtype="f16", rot=64, interleaved=True, layout="hnd"),
        # a whole prompt far beyond the trained length (frequencies scaled), no cache
        _case("rope-32k", "rope", Lmin=131072, Lmax=131072, new=32768, kind="chunk", scale=8.0),
        # the smallest call: one request of about a thousand tokens asks for one more
        _case("decode-1", "paged", Lmin=1000, Lmax=1000),
        # a batch of chats, every length from a few tokens on
        _case("decode-64", "paged", B=64, Lmin=64, Lmax=8192, ps=16),
        # few requests of very different, long contexts
        _case("decode-long", "paged", B=8, Lmin=5000, Lmax=131072, ps=128, Hq=28, Hk=4, dtype="f16"),
        # a chunk of a long prompt
        _case("chunk-2k", "paged", Lmin=32768, Lmax=32768, new=2048, kind="chunk", ps=64),
        # chunks and single tokens in one call, a window with the first tokens kept, head dim 64
        _case("mixed-window", "paged", B=16, Lmin=300, Lmax=6000, new=500, kind="mixed", ps=32, D=64, dtype="f16",
              window=1500, sinks=4, layout="hnd"),
        # short prompts under a window
        _case("window-1k", "window", B=2, Lmin=1000, Lmax=1000, kind="chunk", window=256, sinks=4),
        # a long prompt under a window
        _case("window-16k", "window", Lmin=16384, Lmax=16384, kind="chunk", window=2048, sinks=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rope_cache", "rope", "paged", "paged", "paged", "window"])
    Hq, Hk = rng.choice([(32, 8), (32, 8), (28, 4), (4, 1), (32, 32)])
    c = dict(Hq=Hq, Hk=Hk, dtype=rng.choice(["bf16", "bf16", "f16"]), layout=rng.choice(["nhd", "hnd"]),
             ps=rng.choice([16, 32, 64, 64, 128, 256]))
    D = rng.choice([128, 128, 64])
    if op == "plan":
        return _case(None, "plan", B=_log(rng, 1, 1000), Lmin=_log(rng, 1, 100), Lmax=_log(rng, 200, 30000),
                     kind=rng.choice(["decode", "mixed"]), new=_log(rng, 20, 1000), ps=c["ps"])
    if op in ("rope_cache", "rope"):
        if rng.random() < 0.4:
            c.update(B=_log(rng, 1, 256), Lmin=_log(rng, 2, 100), Lmax=_log(rng, 200, 8192))
        else:
            new = _log(rng, 16, 16384)
            L = new + _log(rng, 1, 100000)
            c.update(Lmin=L, Lmax=L, new=new, kind="chunk")
        return _case(None, op, **c, D=D, rot=D if rng.random() < 0.6 else D // 2, interleaved=rng.random() < 0.4,
                     scale=rng.choice([1.0, 8.0]))
    window, sinks = rng.choice([(0, 0), (0, 0), (_log(rng, 100, 4096), rng.choice([0, 4, 64]))])
    if op == "window":
        L = _log(rng, 100, 16384)
        return _case(None, "window", **dict(c, ps=64), B=2 if L < 3000 else 1, Lmin=L, Lmax=L, kind="chunk",
                     window=_log(rng, 32, 2048), sinks=rng.choice([0, 4, 16, 100]), D=D)
    kind = rng.choice(["decode", "decode", "chunk", "mixed"])
    if kind == "decode":
        B = _log(rng, 1, 64)
        L = _log(rng, 100, min(131072, 600000 // B))
        return _case(None, "paged", **c, D=D, B=B, Lmin=max(1, L // rng.choice([1, 4, 50])), Lmax=L, window=window,
                     sinks=sinks)
    if kind == "chunk":
        new = _log(rng, 2, 2048)
        L = new + _log(rng, 1, 30000)
        return _case(None, "paged", **c, D=D, Lmin=L, Lmax=L, new=new, kind="chunk", window=window, sinks=sinks)
    return _case(None, "paged", **c, D=D, B=rng.choice([8, 12, 16]), Lmin=_log(rng, 50, 500), Lmax=_log(rng, 600, 6000),
                 new=_log(rng, 20, 500), kind="mixed", window=window, sinks=sinks)


# ---- the requests of a case -----------------------------------------------------

def _requests(case):
    """(tokens in the cache, new tokens) of every request: lengths after the step
    spread evenly over the logarithm of Lmin .. Lmax, the longest first."""
    B, cached, new = case["B"], [], []
    for b in range(B):
        u = 1.0 if b == 0 else (b * 0.6180339887498949) % 1.0
        L = round(math.exp(math.log(case["Lmin"]) + u * (math.log(case["Lmax"]) - math.log(case["Lmin"]))))
        if case["kind"] == "chunk":
            n = min(L, case["new"])
        elif case["kind"] == "mixed" and b % 8 == 0:
            n = min(L, round(case["new"] * (1 - u / 2)))
        else:
            n = 1
        if B >= 16 and b % 13 == 12:                     # a place in the batch that no request holds
            L = n = 0
        if case["op"] == "plan" and case["kind"] == "mixed" and b % 7 == 3:
            cached.append(L)
            new.append(-L if b % 2 else -min(L, 3))      # finished; rejected guesses taken back
            continue
        cached.append(L - n)
        new.append(n)
    return cached, new


def _frequencies(case):
    """inv_freq [rot / 2] in float64 for a base of 500000, its slower half stretched for long contexts, and the factor
    on cos and sin."""
    half = case["rot"] // 2
    i = torch.arange(half, dtype=torch.float64)
    inv = 500000.0 ** (-i / half)
    if case["scale"] != 1.0:
        inv = torch.where(2.0 * math.pi / inv > 8192.0, inv / case["scale"], inv)
    return inv.to(DEV), 1.0 + 0.1 * math.log(case["scale"])


def _tables(case, cached, new, g):
    """block table of the requests' pages in random order, -1 past them, and a free list of the others."""
    ps, B = case["ps"], case["B"]
    have = [-(-c // ps) for c in cached]
    need = [-(-max(c + n, c) // ps) for c, n in zip(cached, new)]
    width = max(need) + 2
    total = sum(need) + 7
    perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32)
    k = torch.arange(width)[None, :] < torch.tensor(have)[:, None]
    table, k = table.to(DEV), k.to(DEV)
    table[k] = perm[:sum(have)]
    free = torch.zeros(total, dtype=torch.int32, device=DEV)
    free[:total - sum(have)] = perm[sum(have):]
    return table, free, total - sum(have), total


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt, B, Hq, Hk, D, ps = DTYPES[case["dtype"]], case["B"], case["Hq"], case["Hk"], case["D"], case["ps"]
    s = {"case": case}

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV).to(dt)

    if case["op"] == "window":
        L = case["Lmax"]
        shape = (lambda h: (B, L, h, D)) if case["layout"] == "nhd" else (lambda h: (B, h, L, D))
        q, k, v = (randn(*shape(h)) for h in (Hq, Hk, Hk))
        if case["layout"] == "nhd":                        # the projections' views
            q, k, v = (x.transpose(1, 2) for x in (q, k, v))
        k[:, :, :1] *= 3.0                                 # a first token that draws attention
        return dict(s, q=q, k=k, v=v)
    cached, new = _requests(case)
    if case["op"] == "plan":
        table, free, count, _ = _tables(case, cached, new, g)
        return dict(s, table=table, lens=_i32(cached), new=_i32(new), free=free, count=_i32([count]),
                    T=sum(max(n, 0) for n in new) + 5)     # a batch padded to a fixed size
    T = sum(new)
    if case["op"] in ("rope", "rope_cache"):
        qkv = randn(T, (Hq + 2 * Hk) * D)                  # the views of one projection
        q, k, v = (x.view(T, -1, D) for x in qkv.split([Hq * D, Hk * D, Hk * D], dim=1))
        inv, factor = _frequencies(case)
        pos = torch.cat([torch.arange(c, c + n) for c, n in zip(cached, new)]).to(torch.int32)
        s.update(q=q, k=k, v=v, inv=inv, factor=factor, pos=pos.to(DEV))
        if case["op"] == "rope":
            return s
    table, free, _, pages = _tables(case, [c + n for c, n in zip(cached, new)], [0] * B, g)
    shape = (pages, ps, Hk, D) if case["layout"] == "nhd" else (pages, Hk, ps, D)
    kc, vc = randn(*shape), randn(*shape)
    if case["layout"] == "hnd":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)    # [pages, ps, Hk, D] views
    if case["op"] == "rope_cache":
        req = torch.cat([torch.full((n,), b) for b, n in enumerate(new)]).to(DEV)
        page = table[req, (s["pos"] // ps).long()].long()
        return dict(s, kc=kc, vc=vc, slots=page * ps + s["pos"] % ps)
    first = table[:, 0][_i32([c + n for c, n in zip(cached, new)]) > 0].long()
    kc[first, 0] *= 3.0                                    # a first token that draws attention
    cu = torch.tensor([0] + new).cumsum(0)
    return dict(s, q=randn(T, Hq, D), kc=kc, vc=vc, table=table, lens=_i32([c + n for c, n in zip(cached, new)]),
                cu=cu.to(torch.int32).to(DEV), max_new=max(new), max_len=max(c + n for c, n in zip(cached, new)))


# ---- one pass -------------------------------------------------------------------

def run(s):
    return _own(s) if own else PLAIN[s["case"]["op"]](s)


def _own(s):
    import fftsparse_amd as fa
    c = s["case"]
    window = c["window"] or None
    if c["op"] == "plan":
        p = fa.plan_step(s["table"], s["lens"], s["new"], s["free"], s["count"], page_size=c["ps"], num_tokens=s["T"])
        return dict(table=s["table"], free=s["free"], cu=p.cu_lens, lens=p.seq_lens, pos=p.positions, slots=p.slots,
                    count=p.free_count, lacking=p.lacking)
    if c["op"] == "rope":
        q, k = fa.rope(s["q"], s["k"], s["pos"], s["inv"], attention_factor=s["factor"], interleaved=c["interleaved"])
        return dict(q=q, k=k)
    if c["op"] == "rope_cache":
        q = fa.rope_cache(s["q"], s["k"], s["v"], s["pos"], s["slots"], s["kc"], s["vc"], s["inv"],
                          attention_factor=s["factor"], interleaved=c["interleaved"])
        return dict(q=q, kc=s["kc"], vc=s["vc"])
    if c["op"] == "paged":
        return fa.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], max_new=s["max_new"],
                                  window=window, sinks=c["sinks"])
    return fa.window_attention(s["q"], s["k"], s["v"], window=window, sinks=c["sinks"])


def _plain_plan(s):
    ps, table, free, T = s["case"]["ps"], s["table"], s["free"], s["T"]
    B, P = table.shape
    l0, d = s["lens"].long(), s["new"].long()
    l1 = (l0 + d).clamp(min=0)
    n = d.clamp(min=0)
    p0, p1 = (l0 + ps - 1) // ps, ((l1 + ps - 1) // ps).clamp(max=P)
    grow, rel = (p1 - p0).clamp(min=0), (p0 - p1).clamp(min=0)
    gcum, rcum, cum = grow.cumsum(0), rel.cumsum(0), n.cumsum(0)
    count = s["count"].long()
    col = torch.arange(P, device=DEV)[None, :]
    # pages given back: pushed in order of request and position
    back = (col >= p1[:, None]) & (col < p0[:, None])
    to = (count + (rcum - rel)[:, None] + col - p1[:, None]).clamp(0, len(free) - 1)
    held = torch.cat([free, free[:1]])                                    # the last place takes what is no page
    held.scatter_(0, torch.where(back, to, len(free)).flatten(), table.flatten())
    free = held[:-1]
    # pages taken: from the top of the stack, in the same order
    avail = count + rcum[-1]
    take = (col >= p0[:, None]) & (col < p1[:, None])
    at = avail - 1 - (gcum - grow)[:, None] - (col - p0[:, None])
    page = torch.where(at >= 0, free[at.clamp(0, len(free) - 1)], -1)
    table = torch.where(take, page, table)
    got = torch.minimum((avail - (gcum - grow)).clamp(min=0), grow)
    lost = (l1 - torch.maximum(l0, (p0 + got) * ps)).clamp(min=0)
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), cum])
    j = torch.arange(T, device=DEV)
    b = torch.searchsorted(cum, j, right=True).clamp(max=B - 1)
    real = j < cum[-1]
    pos = l0[b] + j - cu[b]
    pg = table[b, (pos // ps).clamp(0, P - 1)].long()
    slot = torch.where(real & (pos // ps < P) & (pg >= 0), pg * ps + pos % ps, -1)
    i32 = torch.int32
    return dict(table=table, free=free, cu=cu.to(i32), lens=l1.to(i32), pos=torch.where(real, pos, -1).to(i32),
                slots=slot, count=(avail - gcum[-1]).clamp(min=0).to(i32), lacking=lost.sum().reshape(1).to(i32))


def _rotate(x, pos, inv, factor, interleaved):
    angle = pos.double()[:, None, None] * inv
    c, s = (angle.cos() * factor).float(), (angle.sin() * factor).float()
    half = inv.numel()
    x = x.float()
    r = x[..., :2 * half]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    else:
        a, b = r[..., :half], r[..., half:]
        y = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    return torch.cat([y, x[..., 2 * half:]], dim=-1)


def _plain_rope(s):
    w = (s["pos"], s["inv"], s["factor"], s["case"]["interleaved"])
    return dict(q=_rotate(s["q"], *w).to(s["q"].dtype), k=_rotate(s["k"], *w).to(s["k"].dtype))


def _plain_rope_cache(s):
    r = _plain_rope(s)
    page, off = s["slots"] // s["case"]["ps"], s["slots"] % s["case"]["ps"]
    s["kc"][page, off] = r["k"]
    s["vc"][page, off] = s["v"]
    return dict(q=r["q"], kc=s["kc"], vc=s["vc"])


def _softmax(x, seen):
    x = x.masked_fill(~seen, float("-inf"))
    m = x.amax(-1, keepdim=True).clamp(min=torch.finfo(x.dtype).min)
    e = torch.exp(x - m)
    return e / e.sum(-1, keepdim=True).clamp(min=torch.finfo(x.dtype).tiny)


def _seen(pos, key, window, sinks):
    """keys a query at pos sees"""
    ok = key <= pos
    return ok & ((key > pos - window) | (key < sinks)) if window else ok


def _plain_paged(s):
    c = s["case"]
    B, Hq, Hk, D, G = c["B"], c["Hq"], c["Hk"], c["D"], c["Hq"] // c["Hk"]
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    N, L = s["max_new"], s["max_len"]
    P = -(-L // c["ps"])
    pages = s["table"][:, :P].clamp(min=0).long()
    k = s["kc"][pages].reshape(B, P * c["ps"], Hk, D)[:, :L]
    v = s["vc"][pages].reshape(B, P * c["ps"], Hk, D)[:, :L]
    kt = k.permute(0, 2, 3, 1).float().contiguous()                       # [B, Hk, D, L]
    v = v.transpose(1, 2).float().contiguous()                            # [B, Hk, L, D]
    i = torch.arange(N, device=DEV)
    row = (s["cu"][:-1].long()[:, None] + i).clamp(max=len(s["q"]) - 1)
    q = s["q"][row].float().view(B, N, Hk, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, N * G, D)
    x = torch.matmul(q, kt).view(B, Hk, N, G, L) * D ** -0.5
    pos = (s["lens"].long() - n)[:, None] + i                             # [B, N]
    key = torch.arange(L, device=DEV)
    seen = _seen(pos[:, :, None], key, c["window"], c["sinks"]) & (key < s["lens"][:, None, None])
    p = _softmax(x, seen[:, None, :, None, :])
    o = torch.matmul(p.view(B, Hk, N * G, L), v).view(B, Hk, N, G, D).permute(0, 2, 1, 3, 4)
    j = torch.arange(len(s["q"]), device=DEV)
    b = torch.searchsorted(s["cu"][1:].long(), j, right=True)
    return o.reshape(B, N, Hq, D)[b, j - s["cu"][b].long()].to(s["q"].dtype)


def _plain_window(s):
    """Queries in blocks of the window's length: a block's keys are those of it and of the one before, and the first."""
    c = s["case"]
    W, S, B, Hq, Hk, D, L = c["window"], c["sinks"], c["B"], c["Hq"], c["Hk"], c["D"], c["Lmax"]
    G, nb = Hq // Hk, -(-L // W)
    pad = nb * W - L
    q, k, v = (torch.nn.functional.pad(s[t].float(), (0, 0, 0, pad)) for t in "qkv")
    q = q.view(B, Hk, G, nb, W, D).permute(0, 1, 3, 2, 4, 5).reshape(B, Hk, nb, G * W, D)
    at = torch.arange(nb, device=DEV)[:, None] * W + torch.arange(-W, W, device=DEV)      # [nb, 2W]
    far = torch.arange(S, device=DEV).expand(nb, S)
    key = torch.cat([far, at], -1)
    idx = key.clamp(0, nb * W - 1)
    k, v = k[:, :, idx], v[:, :, idx]                                     # [B, Hk, nb, S + 2W, D]
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(B, Hk, nb, G, W, -1) * D ** -0.5
    pos = (torch.arange(nb, device=DEV)[:, None] * W + torch.arange(W, device=DEV))[:, :, None]
    key = key[:, None, :]
    near = (key > pos - W) & (key >= 0)
    near[..., :S] = False
    first = (key < S) & (key <= pos - W)
    first[..., S:] = False
    seen = (key <= pos) & (key < L) & (near | first)
    o = torch.matmul(_softmax(x, seen[None, None, :, None]).view(B, Hk, nb, G * W, -1), v)
    o = o.view(B, Hk, nb, G, W, D).permute(0, 2, 4, 1, 3, 5).reshape(B, nb * W, Hq, D)
    return o[:, :L].to(s["q"].dtype)


PLAIN = {"plan": _plain_plan, "rope": _plain_rope, "rope_cache": _plain_rope_cache, "paged": _plain_paged,
         "window": _plain_window}


# ---- what a pass cannot do without ----------------------------------------------

def _visible(case, p):
    """keys that the token at position p sees"""
    W = case["window"]
    return p + 1 if not W or p < W else W + min(case["sinks"], p + 1 - W)


def work(case):
    e, D, Hq, Hk, ps = 4 if case["dtype"] == "f32" else 2, case["D"], case["Hq"], case["Hk"], case["ps"]
    if case["op"] == "window":
        L, B = case["Lmax"], case["B"]
        return {"bytes": 2 * B * L * (Hq + Hk) * D * e, "flops": 4 * D * Hq * B * sum(_visible(case, p) for p in range(L))}
    cached, new = _requests(case)
    T = sum(max(n, 0) for n in new)
    if case["op"] == "plan":
        moved = sum(abs(-(-(c + n) // ps) - -(-c // ps)) for c, n in zip(cached, new))
        return {"bytes": 16 * case["B"] + 12 * T + 8 * moved, "flops": 0}
    if case["op"] in ("rope", "rope_cache"):
        heads = Hq + Hk + (Hk if case["op"] == "rope_cache" else 0)
        return {"bytes": 2 * T * heads * D * e + 12 * T, "flops": 3 * T * (Hq + Hk) * case["rot"]}
    keys = pairs = 0
    for c, n in zip(cached, new):
        pairs += sum(_visible(case, p) for p in range(c, c + n))
        if n:
            start = max(0, c - case["window"] + 1) if case["window"] else 0
            keys += c + n - start + min(start, case["sinks"] if case["window"] else 0)
    return {"bytes": 2 * keys * Hk * D * e + 2 * T * Hq * D * e, "flops": 4 * D * Hq * pairs}


# ---- the definitions, in 64 bits ------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return _exact_plan(s)
    if case["op"] in ("rope", "rope_cache"):
        return _exact_rope(s)
    return _exact_window(s) if case["op"] == "window" else _exact_paged(s)


def _exact_plan(s):
    ps, T = s["case"]["ps"], s["T"]
    table, lens, new, free = (s[t].tolist() for t in ("table", "lens", "new", "free"))
    top, width = s["count"].item(), len(table[0])
    for row, a, d in zip(table, lens, new):                               # releases first
        for i in range(-(-max(a + d, 0) // ps), -(-a // ps)):
            free[top] = row[i]
            top += 1
    taken, lacking, pos, slots, cu, after = top, 0, [], [], [0], []
    for row, a, d in zip(table, lens, new):
        for i in range(-(-a // ps), min(width, -(-max(a + d, 0) // ps))):
            taken -= 1
            row[i] = free[taken] if taken >= 0 else -1
        for p in range(a, a + d):
            page = row[p // ps] if p // ps < width else -1
            pos.append(p)
            slots.append(page * ps + p % ps if page >= 0 else -1)
            lacking += page < 0
        cu.append(len(pos))
        after.append(max(a + d, 0))
    pos, slots = ((x + [-1] * T)[:T] for x in (pos, slots))
    return dict(table=_i32(table), free=_i32(free), cu=_i32(cu), lens=_i32(after), pos=_i32(pos),
                slots=torch.tensor(slots, device=DEV), count=_i32([max(taken, 0)]), lacking=_i32([lacking]))


def _exact_rope(s):
    half = s["inv"].numel()
    turn = torch.polar(torch.full((), float(s["factor"]), dtype=torch.float64, device=DEV),
                       s["pos"].double()[:, None] * s["inv"])[:, None, :]

    def rotated(x):
        x = x.double()
        y = x.clone()
        re, im = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if s["case"]["interleaved"] else \
            (slice(0, half), slice(half, 2 * half))
        z = torch.complex(x[..., re].contiguous(), x[..., im].contiguous()) * turn
        y[..., re], y[..., im] = z.real, z.imag
        return y

    q, k = rotated(s["q"]), rotated(s["k"])
    if s["case"]["op"] == "rope":
        return dict(q=q, k=k)
    kc, vc = s["kc"].double(), s["vc"].double()
    at = (s["slots"] // s["case"]["ps"], s["slots"] % s["case"]["ps"])
    kc[at], vc[at] = k, s["v"].double()
    return dict(q=q, kc=kc, vc=vc)


def _attend64(q, k, v, first, case):
    """one request: q [n, Hq, D] at positions first .., k and v [L, Hk, D] -> [n, Hq, D]"""
    G = case["Hq"] // case["Hk"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    p = first + torch.arange(len(q), device=DEV)[:, None]
    j = torch.arange(len(k), device=DEV)[None, :]
    hidden = j > p
    if case["window"]:
        hidden |= (p - j >= case["window"]) & (j >= case["sinks"])
    for h in range(case["Hq"]):
        x = q[:, h].double() @ k[:, h // G].double().t().contiguous() / math.sqrt(case["D"])
        x[hidden] = float("-inf")
        out[:, h] = torch.softmax(x, -1) @ v[:, h // G].double()
    return out


def _exact_paged(s):
    cu, lens, ps, out = s["cu"].tolist(), s["lens"].tolist(), s["case"]["ps"], []
    for b, L in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        at = s["table"][b, :-(-L // ps)].long()
        k, v = (s[t][at].reshape(-1, *s[t].shape[2:])[:L] for t in ("kc", "vc"))
        out.append(_attend64(s["q"][cu[b]:cu[b + 1]], k, v, L - n, s["case"]))
    return torch.cat(out)


def _exact_window(s):
    q, k, v = (s[t].transpose(1, 2) for t in "qkv")
    return torch.stack([_attend64(q[b], k[b], v[b], 0, s["case"]) for b in range(len(q))])
