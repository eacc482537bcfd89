"""Trees and 8-bit pages where it can go wrong beside the sizes: keys that are cut into pieces (as each call's workspace
shows), the bytes behind workspaces, caches past 32 bits, replayed graphs, streams at once, the largest trees.

Queries are three times normal numbers where keys are cut, so a few keys of each row hold most of its weight and a piece lost,
joined twice or with a wrong maximum shows.  Tolerance as in ``test_gpu_serving_split``: 3 u of the weighted |v| (weights
rounded, their sum of the rounded ones, the result rounded once) and 2 d of it, d = (D + 8) 2^-23 max sum |q k| scale for a
score in 32 bits; sums over the keys 2^-24 each, the scales' products 2^-22; f16: weights 2^7 times as large in steps of
2^-24, keys 2^-32 max |v|, and results in steps of 2^-24."""
from __future__ import annotations

import pytest
import torch

import fftsparse_amd as fa
from oracle import tree as ref
from tests.test_gpu_pages8 import Chain
from tests.test_gpu_serving_split import cuts  # noqa: F401
from tests.test_gpu_tree import BF, DEV, E4M3, F16, I32, Batch, _i32

pytestmark = pytest.mark.gpu


def _check(b, got, window=None, sinks=0, rows=None):
    """Rows of a batch (all, or those of some requests) against 64 bits."""
    u, D = torch.finfo(b.dtype).eps / 2, b.q.shape[2]
    for r, (c, n) in enumerate(b.lens):
        if not n or (rows is not None and r not in rows):
            continue
        x = slice(b.cu[r], b.cu[r + 1])
        sees = torch.ones(n, n).tril().bool() if isinstance(b, Chain) else b.sees(r)
        pos = list(range(c, c + n)) if isinstance(b, Chain) else b.pos[x]
        if isinstance(b, Chain) and window:                # among the new tokens the window holds too
            i = torch.arange(n)
            sees = sees & ((i[None] > i[:, None] - window) | (c + i[None] < sinks))
        want, mag = ref.attend(b.q[x], b.k[r], b.v[r], n, sees, window, sinks, pos=pos)
        heads = torch.arange(b.q.shape[1]) // (b.q.shape[1] // b.k[r].shape[1])
        top = (b.q[x].double().abs().amax((0, 1))[None] * b.k[r].double().abs().amax(1)).sum(-1).max() * D ** -0.5
        assert len(heads) == b.q.shape[1]
        d = (D + 8) * 2.0 ** -23 * float(top)
        tol = (3 * u + 2 * d + (c + n) * 2.0 ** -24 + 2.0 ** -22) * mag + 1e-30
        if b.dtype is F16:
            tol = tol + (c + n) * 2.0 ** -32 * float(b.v[r].abs().max()) + 2.0 ** -24
        y = got[x].double().cpu()
        assert bool(torch.isfinite(y).all()), r
        err = (y - want).abs()
        assert bool((err <= tol).all()), (r, window, float((err / tol).max()), float(err.max()))


LENS = [(6000, 40), (77, 1), (0, 5), (700, 33)]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (7, 1), (6, 2)])
@pytest.mark.parametrize("ps", [16, 48])
def test_trees_whose_keys_are_cut(cuts, dtype, D, Hq, Hk, ps, bits):  # noqa: F811
    b = Batch(LENS, Hq=Hq, Hk=Hk, D=D, ps=ps, dtype=dtype, bits=bits, hnd=ps == 48, seed=ps + Hq, pad=3)
    b.q *= 3
    for window, sinks in ((None, 0), (2000, 5)):
        out = torch.full(b.q.shape, 7.0, dtype=dtype, device=DEV)
        b.gpu(window=window, sinks=sinks, out=out)
        assert cuts.pop() > 0
        _check(b, out, window, sinks)
        assert bool((out[b.T:] == 7.0).all())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk", [(8, 1), (6, 2)])
@pytest.mark.parametrize("ps", [16, 256])
def test_chunks_over_8_bit_pages_whose_keys_are_cut(cuts, D, Hq, Hk, ps):  # noqa: F811
    b = Chain(LENS, Hq=Hq, Hk=Hk, D=D, ps=ps, seed=ps + Hq)
    b.q *= 3
    for window, sinks in ((None, 0), (2000, 5)):
        got = b.gpu(window=window, sinks=sinks)
        assert cuts.pop() > 0
        _check(b, got, window, sinks)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (7, 1), (8, 2), (28, 4), (33, 1), (64, 64), (6, 6)])
def test_few_rows_whose_keys_are_cut(cuts, D, Hq, Hk):  # noqa: F811
    """Single tokens and small trees over long contexts in workspaces of the size asked for: ranges that end inside requests, long
    rows of pieces."""
    n = max(1, min(4, 32 * Hk // Hq))
    lens = [(30000 if Hq < 28 else 5000, n), (900, 1), (0, 0), (0, n), *((37 * i, 1) for i in range(40 if Hq < 28 else 9)), (2000, n)]
    for b in (Chain(lens, Hq=Hq, Hk=Hk, D=D, ps=64, seed=7), Batch(lens, Hq=Hq, Hk=Hk, D=D, ps=64, bits=8, seed=8),
              Batch(lens, Hq=Hq, Hk=Hk, D=D, ps=64, seed=9)):
        b.q *= 3
        _check(b, b.gpu(max_new=n))


@pytest.mark.parametrize("bits", [16, 8])
def test_caches_past_32_bits(bits):
    """Pages whose offsets, in elements and in bytes, pass 2^32: written, read and moved."""
    ps, Hk, Hq, D = 64, 8, 16, 128
    pages = 90_000                                         # 5.9e9 elements
    store = E4M3 if bits == 8 else BF
    kc, vc = (torch.empty(pages, ps, Hk, D, dtype=torch.uint8 if bits == 8 else BF, device=DEV) for _ in range(2))
    far = [89_999, 70_000, 3]
    for c in (kc, vc):
        c[far] = 0
    kc, vc = (c.view(store) for c in (kc, vc))
    s = torch.full((Hk,), 0.02, device=DEV)
    sc = dict(k_scale=s, v_scale=s) if bits == 8 else {}
    g = torch.Generator().manual_seed(5)
    L, n = 150, 6
    q, k, v = (torch.randn(L, h, D, generator=g).to(BF) for h in (Hq, Hk, Hk))
    table = _i32([far])
    pos = torch.arange(L, dtype=I32, device=DEV)
    slots = table[0].long()[pos.long() // ps] * ps + pos % ps
    inv = torch.zeros(1, dtype=torch.float64, device=DEV)  # no turn: keys as they are
    fa.rope_cache(q.to(DEV), k.to(DEV), v.to(DEV), pos, slots, kc, vc, inv, **sc)
    if bits == 8:
        k8, v8 = ((x.float() / 0.02).clamp(-448, 448).to(E4M3).double() * float(s[0]) for x in (k, v))
    else:
        k8, v8 = k, v
    at = (slots // ps, slots % ps)
    assert torch.equal(vc[at].float().cpu(), (v.float() / 0.02).clamp(-448, 448).to(E4M3).float() if bits == 8 else v.float())
    parents = [-1, 0, 0, 1, 3, 2]
    sees = torch.zeros(n, n, dtype=torch.bool)
    for t, line in enumerate(ref.lines(parents)):
        sees[t, line] = True
    plan = fa.plan_tree(_i32(parents), _i32([0, n]), _i32([L]), max_new=n)
    for max_new in (None, 1000):
        got = fa.tree_attention(q[-n:].to(DEV), kc, vc, table, _i32([0, n]), _i32([L]), plan.mask, max_new=max_new, **sc)
        want, mag = ref.attend(q[-n:], k8, v8, n, sees)
        assert bool(((got.double().cpu() - want).abs() <= (3 * torch.finfo(BF).eps / 2 + 2e-4) * mag).all())
    got = fa.paged_attention(q[-n:].to(DEV), kc, vc, table, _i32([0, n]), _i32([L]), **sc)
    want, mag = ref.attend(q[-n:], k8, v8, n, torch.ones(n, n).tril().bool())
    assert bool(((got.double().cpu() - want).abs() <= (3 * torch.finfo(BF).eps / 2 + 2e-4) * mag).all())
    before = [c.view(torch.uint8)[at].clone() for c in (kc, vc)]
    fa.move_kept(kc, vc, table, _i32([0, n]), _i32([L]), _i32([0, 1, 3, 4, -1, -1]))
    for c, x in zip((kc, vc), before):
        x[L - n + 2], x[L - n + 3] = x[L - n + 3].clone(), x[L - n + 4].clone()
        assert torch.equal(c.view(torch.uint8)[at], x)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("n", [5, 40])
def test_a_captured_tree_step_replays(n, bits):
    """Plan, attention and acceptance in one graph; trees, queries and lengths change between the replays, with eager calls of
    the same in between."""
    b = Batch([(300, n), (0, n), (70, 3), (1500, 1)], bits=bits, ps=32, seed=3)
    (kc, vc), table, cu = b.dev_caches(), b.table.to(DEV), _i32(b.cu)
    lens, q = _i32(b.total), b.q.to(DEV)
    g = torch.Generator().manual_seed(1)
    tree = _i32([p for t in b.trees for p in t])
    tokens, chosen = (torch.randint(0, 2, (b.T,), generator=g).to(DEV) for _ in range(2))
    sc = dict(k_scale=b.ks.to(DEV), v_scale=b.vs.to(DEV)) if bits == 8 else {}

    def run():
        p = fa.plan_tree(tree, cu, lens, max_new=n)
        o = fa.tree_attention(q, kc, vc, table, cu, lens, p.mask, positions=p.positions, max_new=n, window=200, sinks=3, **sc)
        a = fa.accept_tree(tree, tokens, chosen, cu, max_new=n)
        return p.positions, p.mask, o, a.kept, a.kept_lens, a.dropped, a.next_tokens

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(4):
        q.mul_(0.8)
        lens.copy_(_i32([t - i * 7 % 5 for t in b.total]))
        tokens.copy_(torch.randint(0, 2, (b.T,), generator=g))
        tree.copy_(_i32([max(p - (i if p > 2 else 0), -1) for t in b.trees for p in t]))
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y)


def test_two_streams_at_once():
    """Calls that overlap, each with the workspace of its own stream."""
    batches = [Batch([(9000, 8), (30, 3)], seed=1), Chain([(12000, 1), (500, 1)], seed=2), Batch([(4000, 60)], bits=8, seed=3)]
    alone = [b.gpu(max_new=max(b.ns)) for b in batches]
    args = []
    for b in batches:
        kw = dict(k_scale=b.ks.to(DEV), v_scale=b.vs.to(DEV)) if b.bits == 8 else {}
        args.append((b.q.to(DEV), *b.dev_caches(), b.table.to(DEV), _i32(b.cu), _i32(b.total), b.mask.to(DEV), kw))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    got = [[] for _ in batches]
    for _ in range(5):
        for i, (s, b, a) in enumerate(zip(streams, batches, args)):
            with torch.cuda.stream(s):
                if isinstance(b, Chain):
                    got[i].append(fa.paged_attention(*a[:6], max_new=1, **a[7]))
                else:
                    got[i].append(fa.tree_attention(*a[:7], max_new=max(b.ns), **a[7]))
    torch.cuda.synchronize()
    for x, ys in zip(alone, got):
        assert all(torch.equal(x, y) for y in ys)


@pytest.mark.parametrize("bits", [16, 8])
def test_the_largest_trees(bits):
    """1024 tokens in one request, all in one line and in any other: plan, attention, acceptance and move."""
    b = Batch([(100, 1024), (0, 700)], kind="chain", Hq=2, Hk=1, D=64, bits=bits, seed=4)
    cu, lens = _i32(b.cu), _i32(b.total)
    parents = [p for t in b.trees for p in t]
    p = fa.plan_tree(_i32(parents), cu, lens, max_new=1024)
    assert torch.equal(p.mask.cpu(), b.mask) and p.positions.tolist() == b.pos
    _check(b, b.gpu(max_new=1024))
    _check(b, b.gpu(max_new=1024, window=50, sinks=4), 50, 4)
    tokens = torch.arange(b.T, device=DEV)
    a = fa.accept_tree(_i32(parents), tokens, tokens + 1, cu, max_new=1024)
    assert a.kept_lens.tolist() == [1024, 700] and a.kept.tolist() == [*range(1024), *range(700)]


@pytest.mark.parametrize("last", [2 ** 31 - 1, -(2 ** 31)])
def test_row_numbers_at_the_ends_of_their_range(last):
    """A last row number far out of range is taken as the number of rows, or as 0, and nothing outside the outputs is written."""
    T, B = 70, 1
    parents = torch.arange(-1, T - 1, dtype=I32, device=DEV)
    cu = torch.tensor([0, last], dtype=I32, device=DEV)
    n = T if last > 0 else 0
    held = torch.full((3 * T,), 7, dtype=I32, device=DEV)
    masks = torch.full((3 * T, 2), 7, dtype=torch.int64, device=DEV)
    fa.plan_tree(parents, cu, _i32([n]), max_new=128, out=fa.TreePlan(held[T:2 * T], masks[T:2 * T]))
    torch.cuda.synchronize()
    assert held[T:2 * T].tolist() == (list(range(T)) if n else [-1] * T)
    want = [[(1 << min(t + 1, 63)) - 1 | (-(1 << 63) if t > 62 else 0), (1 << max(t - 63, 0)) - 1] for t in range(T)]
    assert masks[T:2 * T].tolist() == (want if n else [[0, 0]] * T)
    tokens = torch.ones(T, dtype=I32, device=DEV)
    kept = torch.full((3 * T,), 7, dtype=I32, device=DEV)
    small = torch.zeros(2, B, dtype=I32, device=DEV)
    acc = fa.accept_tree(parents, tokens, tokens, cu, max_new=128,
                         out=fa.Accepted(kept[T:2 * T], small[0], small[1], tokens.new_empty(B)))
    assert kept[T:2 * T].tolist() == (list(range(T)) if n else [-1] * T)
    assert acc.kept_lens.tolist() == [n] and acc.dropped.tolist() == [0]
    for x in (held, kept, masks):
        assert bool((x[:T] == 7).all()) and bool((x[2 * T:] == 7).all())
