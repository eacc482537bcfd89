"""Drafted tokens and 8-bit pages: further serving operators of fftsparse_amd as cases that can be timed and compared.

A server whose requests bring a tree of drafted tokens to a step (a node's parent is the token it follows) needs the
nodes' positions and what each sees (``plan_tree``), attention of the nodes over the paged cache
(``tree_attention``), and, once the model has chosen a token after every node, the path that is kept and the kept
tokens' rows moved to where they belong in the cache (``accept_tree``, ``move_kept``).  A cache in 8 bits (e4m3 with a
scale for each KV head) halves what a step reads: written by ``rope_cache``, read by ``paged_attention`` and
``tree_attention``.  Head counts are those of the benchmark configurations (32 / 8, 28 / 4, 4 / 1).

Where ``own`` is false ``run`` computes the same in elementary torch operations, in 32 bits (angles in 64).
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
E4M3 = torch.float8_e4m3fn
MOST = 448.0                                               # the largest e4m3 number
DEV = "cuda"


def _case(name, op, **kw):
    c = dict(op=op, B=1, Lmin=1000, Lmax=1000, Nmin=1, Nmax=1, ps=64, Hq=32, Hk=8, D=128, dtype="bf16", bits=16,
             window=0, sinks=0, layout="nhd", rot=128, interleaved=False, layers=1)
    assert set(kw) <= set(c), set(kw) - set(c)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # drafts of one step of a small batch: nothing but latency
        _case("plan-tree-small", "plan_tree", B=4, Nmin=8, Nmax=16),
        # a large batch, from a few drafted tokens to wide trees
        _case("plan-tree-large", "plan_tree", B=256, Lmin=100, Lmax=8192, Nmin=4, Nmax=250),
        # the new tokens of a decoding step of 48 requests into 8-bit pages
        _case("store8-decode", "store", B=48, Lmin=100, Lmax=8192, bits=8),
        # a long chunk of one prompt into 8-bit pages that keep a head's rows together, half of each head rotated
        _case("store8-chunk", "store", Lmin=31809, Lmax=31809, Nmin=8191, Nmax=8191, ps=128, Hq=28, Hk=4, dtype="f16",
              rot=64, interleaved=True, layout="hnd", bits=8),
        # the smallest call over an 8-bit cache: one request of about a thousand tokens asks for one more
        _case("decode8-1", "attend", bits=8),
        # a batch of chats over an 8-bit cache, every length from a few tokens on
        _case("decode8-64", "attend", B=64, Lmin=64, Lmax=8192, ps=16, bits=8),
        # a chunk of a long prompt over an 8-bit cache
        _case("chunk8-2k", "attend", Lmin=30000, Lmax=30000, Nmin=2048, Nmax=2048, bits=8),
        # one request with a small tree of drafts
        _case("tree-1", "tree", Nmin=8, Nmax=8),
        # a batch with a tree of 64 tokens each
        _case("tree-16x64", "tree", B=16, Lmin=1000, Lmax=8192, Nmin=64, Nmax=64),
        # trees of many sizes over 8-bit pages under a window with the first tokens kept, head dim 64
        _case("tree8-window", "tree", B=40, Lmin=50, Lmax=12000, Nmin=1, Nmax=60, ps=32, Hq=28, Hk=4, D=64, dtype="f16",
              bits=8, window=2000, sinks=4, layout="hnd", rot=64),
        # one request's tree against what the model chose, its kept tokens' rows moved in all layers
        _case("verify-1", "verify", Nmin=16, Nmax=16, layers=32),
        # a batch's trees, an 8-bit cache of all layers
        _case("verify-64", "verify", B=64, Lmin=30, Lmax=500, Nmin=8, Nmax=64, ps=32, bits=8, layers=32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan_tree", "store", "attend", "attend", "tree", "tree", "tree", "verify"])
    Hq, Hk, D = rng.choice([(32, 8, 128), (32, 8, 128), (28, 4, 128), (4, 1, 128), (32, 32, 128), (28, 4, 64), (4, 1, 64)])
    c = dict(Hq=Hq, Hk=Hk, D=D, dtype=rng.choice(["bf16", "bf16", "f16"]), layout=rng.choice(["nhd", "hnd"]),
             ps=rng.choice([16, 32, 64, 64, 128, 256]), bits=8)
    if op == "plan_tree":
        n = _log(rng, 2, 250)
        return _case(None, op, B=_log(rng, 1, 250), Lmin=_log(rng, 1, 100), Lmax=_log(rng, 200, 8192),
                     Nmin=max(1, n // rng.choice([1, 3, 20])), Nmax=n)
    if op == "store":
        c.update(rot=D if rng.random() < 0.6 else D // 2, interleaved=rng.random() < 0.4)
        if rng.random() < 0.4:
            return _case(None, op, **c, B=_log(rng, 1, 256), Lmin=_log(rng, 2, 100), Lmax=_log(rng, 200, 8192))
        n, L = _log(rng, 16, 16384), _log(rng, 1, 60000)
        return _case(None, op, **c, Lmin=L, Lmax=L, Nmin=n, Nmax=n)
    if op == "verify":
        n = _log(rng, 2, 64)
        return _case(None, op, **dict(c, bits=rng.choice([8, 16])), B=_log(rng, 1, 48), Lmin=_log(rng, 10, 30),
                     Lmax=_log(rng, 50, 400), Nmin=max(1, n // rng.choice([1, 4])), Nmax=n, layers=rng.choice([4, 28, 32]))
    window, sinks = rng.choice([(0, 0), (0, 0), (_log(rng, 100, 4096), rng.choice([0, 4, 64]))])
    c.update(window=window, sinks=sinks, rot=D)
    if op == "attend" and rng.random() < 0.4:
        n, L = _log(rng, 2, 2048), _log(rng, 1, 30000)
        return _case(None, op, **c, Lmin=L, Lmax=L, Nmin=n, Nmax=n)
    if op == "attend":
        B = _log(rng, 1, 64)
        L = _log(rng, 100, min(131072, 600000 // B))
        return _case(None, op, **c, B=B, Lmin=max(1, L // rng.choice([1, 4, 50])), Lmax=L)
    B, n = _log(rng, 1, 48), _log(rng, 2, 250)
    L = _log(rng, 30, 300000 // B)
    n = min(n, max(2, 6000000 // (B * L)))
    c["bits"] = rng.choice([8, 16])
    return _case(None, op, **c, B=B, Lmin=max(1, L // rng.choice([1, 4, 50])), Lmax=L, Nmin=max(1, n // rng.choice([1, 4])),
                 Nmax=n)


# ---- the requests of a case -----------------------------------------------------

def _spread(lo, hi, u):
    return round(math.exp(math.log(lo) + u * (math.log(hi) - math.log(lo))))


def _requests(case):
    """(tokens in the cache, new tokens) of every request, spread evenly over the logarithms of Lmin .. Lmax and
    Nmin .. Nmax, the largest first."""
    B, cached, new = case["B"], [], []
    for b in range(B):
        u = 1.0 if b == 0 else (b * 0.6180339887498949) % 1.0
        w = 1.0 if b == 0 else (b * 0.7548776662466927) % 1.0
        idle = B >= 16 and b % 13 == 12                    # a place in the batch that no request holds
        cached.append(0 if idle else _spread(case["Lmin"], case["Lmax"], u))
        new.append(0 if idle else _spread(case["Nmin"], case["Nmax"], w))
    return cached, new


def _trees(case):
    """Each request's new tokens as a tree: lists of the parents' indices (-1: the first token, which follows the
    context), and of the child that the model agrees with after each token (-1: with none)."""
    g = torch.Generator().manual_seed(1000 * case["B"] + case["Nmax"] + 10)
    parents, liked = [], []
    for n in _requests(case)[1]:
        i = torch.arange(n)
        p = (i * torch.rand(n, generator=g)).long().clamp(max=(i - 1).clamp(min=0)).tolist()
        if n:
            p[0] = -1
        child, like = torch.rand(n, generator=g).tolist(), [-1] * n
        for t in range(n - 1, 0, -1):                      # four in five tokens have a drafted child that is right
            if child[p[t]] < 0.8:
                like[p[t]] = t
        parents.append(p)
        liked.append(like)
    return parents, liked


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _reach(parents, B, N):
    """[B, N, N] bool: token t's ancestors and itself, from parents [B, N] (-1: none)."""
    up = (parents[:, :, None] == torch.arange(N, device=DEV)).float() + torch.eye(N, device=DEV)
    for _ in range(max(1, (N - 1).bit_length())):          # paths of twice the length each time
        up = (torch.matmul(up, up) > 0).float()
    return up > 0


def _rows_of(cu, T):
    """Request and index in it of rows 0 .. T - 1 (the last request's for rows behind it)."""
    j = torch.arange(T, device=DEV)
    b = torch.searchsorted(cu[1:].long(), j, right=True).clamp(max=len(cu) - 2)
    return b, j - cu[b].long()


def _padded(x, cu, N, fill):
    """[T] -> [B, N], fill past a request's tokens."""
    i = torch.arange(N, device=DEV)
    at = cu[:-1].long()[:, None] + i
    return torch.where(i < (cu[1:] - cu[:-1])[:, None], x[at.clamp(max=len(x) - 1)].long(), fill)


def _words(seen):
    """[..., N] bool -> [..., ceil(N / 64)] int64, bit j % 64 of word j / 64."""
    N = seen.shape[-1]
    seen = torch.nn.functional.pad(seen, (0, -N % 64)).unflatten(-1, (-1, 64))
    return (seen.long() << torch.arange(64, device=DEV)).sum(-1)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt, B, Hq, Hk, D, ps = DTYPES[case["dtype"]], case["B"], case["Hq"], case["Hk"], case["D"], case["ps"]
    cached, new = _requests(case)
    T, N = sum(new), max(new)
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(DEV)
    total = [c + n for c, n in zip(cached, new)]
    s = {"case": case, "cu": cu, "T": T, "N": N}

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32 if case["bits"] == 8 else dt)

    if case["op"] in ("plan_tree", "tree", "verify"):
        trees, liked = _trees(case)
        s["parents"] = _i32([p for t in trees for p in t])
    if case["op"] == "plan_tree":                          # a batch padded to a fixed size; contexts by the seed
        more = torch.randint(0, 500, (B,), generator=g, device=DEV, dtype=torch.int32)
        return dict(s, parents=torch.cat([s["parents"], _i32([0] * 5)]), T=T + 5, lens=_i32(total) + more)
    lens = _i32(total)
    # block tables of the requests' pages in random order, -1 past them
    need = [-(-t // ps) for t in total]
    pages = sum(need) + 7
    table = torch.full((B, max(need) + 2), -1, dtype=torch.int32)
    held = torch.arange(table.shape[1])[None, :] < torch.tensor(need)[:, None]
    table, held = table.to(DEV), held.to(DEV)
    table[held] = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)[:sum(need)]
    scale = (0.02 + 0.02 * torch.rand(2, Hk, generator=g, device=DEV)) if case["bits"] == 8 else None

    def cache(i):
        lead = (case["layers"],) if case["op"] == "verify" else ()
        x = randn(*lead, pages, *((ps, Hk) if case["layout"] == "nhd" else (Hk, ps)), D)
        x = x if case["layout"] == "nhd" else x.transpose(-2, -3)          # [pages, ps, Hk, D] views
        if i == 0 and not lead:
            x[table[:, 0][lens > 0].long(), 0] *= 3.0                      # a first token that draws attention
        return x if scale is None else (x / scale[i][:, None]).clamp(-MOST, MOST).to(E4M3)

    kc, vc = cache(0), cache(1)
    s.update(kc=kc, vc=vc, table=table, lens=lens)
    if scale is not None:
        s.update(ks=scale[0].contiguous(), vs=scale[1].contiguous())
    if case["op"] == "verify":
        # drafted tokens, and what the model chose after each of them
        tokens = torch.randint(1, 128000, (T,), generator=g, device=DEV)
        first = torch.tensor([0] + new).cumsum(0).tolist()
        like = torch.tensor([first[b] + t if t >= 0 else -1 for b, x in enumerate(liked) for t in x], device=DEV)
        return dict(s, tokens=tokens, chosen=torch.where(like >= 0, tokens[like.clamp(min=0)], 0), k_layers=list(kc),
                    v_layers=list(vc))
    if case["op"] == "store":
        qkv = randn(T, (Hq + 2 * Hk) * D).to(dt)           # the views of one projection
        q, k, v = (x.view(T, -1, D) for x in qkv.split([Hq * D, Hk * D, Hk * D], dim=1))
        b, i = _rows_of(cu, T)
        pos = torch.tensor(cached, device=DEV)[b] + i
        inv = 500000.0 ** (-torch.arange(case["rot"] // 2, dtype=torch.float64, device=DEV) / (case["rot"] // 2))
        return dict(s, q=q, k=k, v=v, pos=pos.to(torch.int32), slots=table[b, pos // ps].long() * ps + pos % ps, inv=inv)
    s["q"] = randn(T, Hq, D).to(dt)
    s["max_len"] = max(total)
    if case["op"] == "tree":
        reach = _reach(_padded(s["parents"], cu, N, -1), B, N)
        b, i = _rows_of(cu, T)
        depth = reach.sum(-1) - 1
        s.update(mask=_words(reach)[b, i].contiguous(), pos=(lens.long() - (cu[1:] - cu[:-1]))[b].add(depth[b, i]).to(torch.int32))
    return s


# ---- one pass -------------------------------------------------------------------

def run(s):
    return _own(s) if own else PLAIN[s["case"]["op"]](s)


def _own(s):
    import fftsparse_amd as fa
    c = s["case"]
    scales = dict(k_scale=s["ks"], v_scale=s["vs"]) if c["bits"] == 8 and c["op"] in ("store", "attend", "tree") else {}
    if c["op"] == "plan_tree":
        p = fa.plan_tree(s["parents"], s["cu"], s["lens"], max_new=s["N"])
        return dict(pos=p.positions, mask=p.mask)
    if c["op"] == "store":
        q = fa.rope_cache(s["q"], s["k"], s["v"], s["pos"], s["slots"], s["kc"], s["vc"], s["inv"],
                          interleaved=c["interleaved"], **scales)
        return dict(q=q, kc=s["kc"], vc=s["vc"])
    if c["op"] == "verify":
        a = fa.accept_tree(s["parents"], s["tokens"], s["chosen"], s["cu"], max_new=s["N"])
        fa.move_kept(s["k_layers"], s["v_layers"], s["table"], s["cu"], s["lens"], a.kept)
        return dict(kept=a.kept, count=a.kept_lens, dropped=a.dropped, next=a.next_tokens, kc=s["kc"], vc=s["vc"])
    w = dict(max_new=s["N"], window=c["window"] or None, sinks=c["sinks"], **scales)
    if c["op"] == "attend":
        return fa.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], **w)
    return fa.tree_attention(s["q"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], s["mask"], positions=s["pos"], **w)


def _plain_plan_tree(s):
    B, N, cu, T = s["case"]["B"], s["N"], s["cu"], s["T"]
    reach = _reach(_padded(s["parents"], cu, N, -1), B, N)
    b, i = _rows_of(cu, T)
    real = torch.arange(T, device=DEV) < cu[-1]
    i = i.clamp(max=N - 1)
    pos = (s["lens"] - (cu[1:] - cu[:-1]))[b] + reach.sum(-1)[b, i] - 1
    return dict(pos=torch.where(real, pos, -1).to(torch.int32),
                mask=torch.where(real[:, None], _words(reach)[b, i], 0))


def _plain_store(s):
    c, ps = s["case"], s["case"]["ps"]
    angle = s["pos"].double()[:, None, None] * s["inv"]
    co, si = angle.cos().float(), angle.sin().float()
    half = s["inv"].numel()

    def rotated(x):
        x = x.float()
        r = x[..., :2 * half]
        if c["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            y = torch.stack([a * co - b * si, b * co + a * si], dim=-1).flatten(-2)
        else:
            a, b = r[..., :half], r[..., half:]
            y = torch.cat([a * co - b * si, b * co + a * si], dim=-1)
        return torch.cat([y, x[..., 2 * half:]], dim=-1)

    def in8(x, scale):
        return (x.float() / scale[:, None]).clamp(-MOST, MOST).to(E4M3)

    page, off = s["slots"] // ps, s["slots"] % ps
    s["kc"][page, off] = in8(rotated(s["k"]), s["ks"])
    s["vc"][page, off] = in8(s["v"], s["vs"])
    return dict(q=rotated(s["q"]).to(s["q"].dtype), kc=s["kc"], vc=s["vc"])


def _softmax(x, seen):
    x = x.masked_fill(~seen, float("-inf"))
    m = x.amax(-1, keepdim=True).clamp(min=torch.finfo(x.dtype).min)
    e = torch.exp(x - m)
    return e / e.sum(-1, keepdim=True).clamp(min=torch.finfo(x.dtype).tiny)


def _plain_attend(s):
    c = s["case"]
    B, Hq, Hk, D, G = c["B"], c["Hq"], c["Hk"], c["D"], c["Hq"] // c["Hk"]
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    N, L = s["N"], s["max_len"]
    P = -(-L // c["ps"])
    pages = s["table"][:, :P].clamp(min=0).long()
    k, v = (s[t][pages].reshape(B, P * c["ps"], Hk, D)[:, :L].float() for t in ("kc", "vc"))
    if c["bits"] == 8:
        k, v = k * s["ks"][:, None], v * s["vs"][:, None]
    kt, v = k.permute(0, 2, 3, 1).contiguous(), v.transpose(1, 2).contiguous()
    i = torch.arange(N, device=DEV)
    row = (s["cu"][:-1].long()[:, None] + i).clamp(max=len(s["q"]) - 1)     # [B, N]
    q = s["q"][row].float().view(B, N, Hk, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, N * G, D)
    x = torch.matmul(q, kt).view(B, Hk, N, G, L) * D ** -0.5
    base = (s["lens"].long() - n)[:, None, None]
    key = torch.arange(L, device=DEV)
    if c["op"] == "tree":
        pos, own_key = s["pos"].long()[row][:, :, None], key - base
        word = s["mask"][row].gather(2, (own_key // 64).clamp(0, s["mask"].shape[1] - 1).expand(B, N, L))
        drafted = (own_key >= 0) & (own_key < n[:, None, None]) & (word >> (own_key % 64) & 1 != 0)
        seen = key < base
    else:
        pos, drafted = base + i[:, None], False
        seen = (key <= pos) & (key < s["lens"][:, None, None])
    if c["window"]:
        seen = seen & ((key > pos - c["window"]) | (key < c["sinks"]))
    p = _softmax(x, (seen | drafted)[:, None, :, None, :])
    o = torch.matmul(p.view(B, Hk, N * G, L), v).view(B, Hk, N, G, D).permute(0, 2, 1, 3, 4).reshape(B, N, Hq, D)
    return o[_rows_of(s["cu"], len(s["q"]))].to(s["q"].dtype)


def _plain_verify(s):
    B, N, cu, ps = s["case"]["B"], s["N"], s["cu"], s["case"]["ps"]
    n = (cu[1:] - cu[:-1]).long()
    parents = _padded(s["parents"], cu, N, -1)
    tokens, chosen = _padded(s["tokens"], cu, N, -1), _padded(s["chosen"], cu, N, -1)
    i = torch.arange(N, device=DEV)
    there, p = i < n[:, None], parents.clamp(min=0)
    right = there & (parents >= 0) & (tokens == chosen.gather(1, p))
    lowest = torch.full((B, N), N, device=DEV).scatter_reduce(1, p, torch.where(right, i, N), "amin")
    on = there & ((i == 0) | right & (lowest.gather(1, p) == i))
    kept = there & ((_reach(parents, B, N) & ~on[:, None, :]).sum(-1) == 0)
    count = kept.sum(-1)
    rank = torch.where(kept, kept.long().cumsum(-1) - 1, N)
    place = torch.full((B, N + 1), -1, device=DEV).scatter(1, rank, i.expand(B, N))[:, :N]
    last = place.amax(-1)
    after = torch.where(count > 0, chosen.gather(1, last.clamp(min=0)[:, None])[:, 0], -1)
    # the i-th kept token's rows go to the i-th place behind the context
    b, j = ((place >= 0) & (place != i)).nonzero(as_tuple=True)
    base = s["lens"].long() - n
    src, dst = base[b] + place[b, j], base[b] + j
    for t in ("kc", "vc"):
        rows = s[t][:, s["table"][b, src // ps].long(), src % ps]
        s[t][:, s["table"][b, dst // ps].long(), dst % ps] = rows
    return dict(kept=place[_rows_of(cu, s["T"])].to(torch.int32), count=count.to(torch.int32),
                dropped=(count - n).to(torch.int32), next=after, kc=s["kc"], vc=s["vc"])


PLAIN = {"plan_tree": _plain_plan_tree, "store": _plain_store, "attend": _plain_attend, "tree": _plain_attend,
         "verify": _plain_verify}


# ---- what a pass cannot do without ----------------------------------------------

def _kept(parents, liked):
    """Indices of the kept path of one request."""
    path, t = [], 0 if parents else -1
    while t >= 0:
        path.append(t)
        t = liked[t]
    return path


def work(case):
    D, Hq, Hk, B, W = case["D"], case["Hq"], case["Hk"], case["B"], case["window"]
    e, cached, new = case["bits"] // 8, *_requests(case)
    T, words = sum(new), -(-max(new) // 64)
    if case["op"] == "plan_tree":
        return {"bytes": 8 * B + T * (8 + 8 * words), "flops": 0}
    if case["op"] == "store":
        return {"bytes": T * D * (2 * (2 * Hq + 2 * Hk) + 2 * Hk * e) + 12 * T, "flops": 3 * T * (Hq + Hk) * case["rot"]}
    if case["op"] == "verify":
        moved = sum(t != i for p, k in zip(*_trees(case)) for i, t in enumerate(_kept(p, k)))
        return {"bytes": 24 * T + 20 * B + moved * 4 * Hk * D * e * case["layers"], "flops": 0}
    keys = pairs = 0
    for c, n in zip(cached, new):
        # a token sees its context (or what the window leaves of it), and at least itself of the new ones
        start = max(0, c - W + 1) if W else 0
        first = min(start, case["sinks"]) if W else 0
        keys += c + n - start + first if n else 0
        if case["op"] == "tree":
            pairs += n * (c - start + first + 1)
        else:
            pairs += sum(p + 1 if not W or p < W else W + min(case["sinks"], p + 1 - W) for p in range(c, c + n))
    drafts = T * (8 * words + 4) if case["op"] == "tree" else 0
    return {"bytes": 2 * keys * Hk * D * e + 4 * T * Hq * D + drafts, "flops": 4 * D * Hq * pairs}


# ---- the definitions, in 64 bits ------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return EXACT[case["op"]](s)


def _lines(parent):
    """Ancestors of each token and itself, nearest first."""
    lines = []
    for t, p in enumerate(parent):
        lines.append([t] + (lines[p] if p >= 0 else []))
    return lines


def _exact_plan_tree(s):
    cu, lens, words = s["cu"].tolist(), s["lens"].tolist(), -(-s["N"] // 64)
    parents, pos, mask = s["parents"].tolist(), [-1] * s["T"], [[0] * words for _ in range(s["T"])]
    for b, L in enumerate(lens):
        n = cu[b + 1] - cu[b]
        for t, line in enumerate(_lines(parents[cu[b]:cu[b + 1]])):
            pos[cu[b] + t] = L - n + len(line) - 1
            bits = sum(1 << u for u in line)
            for w in range(words):
                x = bits >> 64 * w & (1 << 64) - 1
                mask[cu[b] + t][w] = x - (1 << 64) if x >> 63 else x
    return dict(pos=_i32(pos), mask=torch.tensor(mask, dtype=torch.int64, device=DEV))


def _exact_store(s):
    half, ps = s["inv"].numel(), s["case"]["ps"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), s["pos"].double()[:, None] * s["inv"])[:, None, :]

    def rotated(x):
        y = x.double().clone()
        re, im = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if s["case"]["interleaved"] else \
            (slice(0, half), slice(half, 2 * half))
        z = torch.complex(y[..., re].contiguous(), y[..., im].contiguous()) * turn
        y[..., re], y[..., im] = z.real, z.imag
        return y

    kc, vc = s["kc"].double(), s["vc"].double()
    at = (s["slots"] // ps, s["slots"] % ps)
    kc[at] = (rotated(s["k"]) / s["ks"].double()[:, None]).clamp(-MOST, MOST)
    vc[at] = (s["v"].double() / s["vs"].double()[:, None]).clamp(-MOST, MOST)
    return dict(q=rotated(s["q"]), kc=kc, vc=vc)


def _exact_attend(s):
    c = s["case"]
    cu, lens, ps, G, out = s["cu"].tolist(), s["lens"].tolist(), c["ps"], c["Hq"] // c["Hk"], []
    parents = s["parents"].tolist() if c["op"] == "tree" else []
    for b, L in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        base, key = L - n, torch.arange(L, device=DEV)
        at = s["table"][b, :-(-L // ps)].long()
        k, v = (s[t][at].reshape(-1, c["Hk"], c["D"])[:L] for t in ("kc", "vc"))
        if c["op"] == "tree":
            lines = _lines(parents[cu[b]:cu[b + 1]])
            p = torch.tensor([base + len(x) - 1 for x in lines], device=DEV)[:, None]
            sees = torch.zeros(n, n, dtype=torch.bool)
            for t, line in enumerate(lines):
                sees[t, line] = True
            hidden = (key >= base).repeat(n, 1)
            hidden[:, base:] = ~sees.to(DEV)
        else:
            p = base + torch.arange(n, device=DEV)[:, None]
            hidden = key > p
        if c["window"]:
            hidden |= (p - key >= c["window"]) & (key >= c["sinks"]) & ((key < base) | (c["op"] != "tree"))
        o = torch.empty(n, c["Hq"], c["D"], dtype=torch.float64, device=DEV)
        for h in range(c["Hq"]):
            ki, vi = k[:, h // G].double(), v[:, h // G].double()
            if c["bits"] == 8:
                ki, vi = ki * s["ks"][h // G].double(), vi * s["vs"][h // G].double()
            x = s["q"][cu[b]:cu[b + 1], h].double() @ ki.t().contiguous() / math.sqrt(c["D"])
            o[:, h] = torch.softmax(x.masked_fill(hidden, float("-inf")), -1) @ vi
        out.append(o)
    return torch.cat(out)


def _exact_verify(s):
    cu, lens, ps = s["cu"].tolist(), s["lens"].tolist(), s["case"]["ps"]
    parents, tokens, chosen, table = (s[t].tolist() for t in ("parents", "tokens", "chosen", "table"))
    kept, count, after = [-1] * s["T"], [], []
    kc, vc = s["kc"].clone(), s["vc"].clone()
    for b, L in enumerate(lens):
        n, path = cu[b + 1] - cu[b], []
        p, x, y = (z[cu[b]:cu[b + 1]] for z in (parents, tokens, chosen))
        t = 0 if n else None
        while t is not None:
            path.append(t)
            t = next((u for u in range(t + 1, n) if p[u] == t and x[u] == y[t]), None)
        place = lambda i: (table[b][(L - n + i) // ps], (L - n + i) % ps)   # noqa: E731
        for i, t in enumerate(path):
            kept[cu[b] + i] = t
            for old, cache in ((s["kc"], kc), (s["vc"], vc)):
                cache[:, place(i)[0], place(i)[1]] = old[:, place(t)[0], place(t)[1]]
        count.append(len(path))
        after.append(y[path[-1]] if path else -1)
    dropped = [c - (cu[b + 1] - cu[b]) for b, c in enumerate(count)]
    return dict(kept=_i32(kept), count=_i32(count), dropped=_i32(dropped), next=torch.tensor(after, device=DEV),
                kc=kc.double(), vc=vc.double())


EXACT = {"plan_tree": _exact_plan_tree, "store": _exact_store, "attend": _exact_attend, "tree": _exact_attend,
         "verify": _exact_verify}
