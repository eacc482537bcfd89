"""Trees under a window on the GPU: the window holds among the new tokens too, so every token gets what decoding its line
token by token would give it, however deep the tree is.

Tolerance: each result is within (3 u + 2e-4) times the softmax average of |v| of the exact one, as ``test_gpu_tree``
derives it (u: half a step of the type), so two of them are within twice that of each other; f16 adds the weights' absolute
error as there."""
from __future__ import annotations

import pytest
import torch

import fftsparse_amd as fa
from oracle import paged, tree as ref
from tests.test_gpu_tree import BF, DEV, F16, I32, SMALL, WIDE, Batch, Model, _cu, _i32, _tree, _words

pytestmark = pytest.mark.gpu

WINDOWS = [(1, 0), (1, 3), (2, 0), (7, 4), (16, 70), (40, 0), (64, 5), (130, 200), (1023, 1), (2 ** 31 - 1, 2 ** 31 - 1)]


def _planned(b, window, sinks):
    """The batch with the mask that plan_tree forms under the window."""
    tree = [p for t in b.trees for p in t] + [0] * (len(b.q) - b.T)
    p = fa.plan_tree(_i32(tree), _i32(b.cu), _i32(b.total), max_new=max(b.ns), window=window, sinks=sinks)
    assert p.positions.tolist()[:b.T] == b.pos
    b.mask = p.mask.cpu()
    return b


@pytest.mark.parametrize("kind", ["chain", "star", "roots", "random"])
@pytest.mark.parametrize("ns,max_new", [([0, 3, 0, 64, 65, 1, 63, 0], 65), ([200, 7, 128, 129], 200), ([1024, 1, 1000], 1024),
                                        ([300, 20], 100), ([18] * 300, 18)])
def test_plan_tree_windows(kind, ns, max_new):
    g = torch.Generator().manual_seed(len(ns) + max_new)
    parents = [p for n in ns for p in _tree(n, kind, g)] + [0] * 7
    cu, words = _cu(ns), -(-max_new // 64)
    lens = [n - 1 if b == 2 and n else n + 11 * (b % 30) for b, n in enumerate(ns)]     # one with less room than new tokens
    for window, sinks in WINDOWS:
        got = fa.plan_tree(_i32(parents), _i32(cu), _i32(lens), max_new=max_new, window=window, sinks=sinks)
        pos, mask = ref.plan(parents, cu, lens, words, window, sinks)
        assert got.positions.tolist() == pos
        assert torch.equal(got.mask.cpu(), _words(mask)), (window, sinks)
    none = fa.plan_tree(_i32(parents), _i32(cu), _i32(lens), max_new=max_new, sinks=5)     # without a window they say nothing
    assert torch.equal(none.mask.cpu(), _words(ref.plan(parents, cu, lens, words)[1]))


def _tol(b, mag, keys):
    u = torch.finfo(b.dtype).eps / 2
    tol = (3 * u + 2e-4) * mag + 1e-30
    return tol + keys * 2.0 ** -25 * 8.0 + 2.0 ** -25 if b.dtype is F16 else tol


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("window,sinks", [(None, 0), *WINDOWS[:-2]])
@pytest.mark.parametrize("lens", [SMALL, WIDE], ids=["small", "wide"])
def test_a_chain_of_tree_attention_is_paged_attention(lens, window, sinks, bits, dtype):
    """The same tokens through both calls, windows shorter than the chains among them."""
    b = _planned(Batch(lens, kind="chain", bits=bits, dtype=dtype, ps=32, seed=15), window, sinks)
    sc = dict(k_scale=b.ks.to(DEV), v_scale=b.vs.to(DEV)) if bits == 8 else {}
    for max_new in (None, max(b.ns)):
        x = b.gpu(window=window, sinks=sinks, max_new=max_new).double().cpu()
        y = fa.paged_attention(b.q.to(DEV), *b.dev_caches(), b.table.to(DEV), _i32(b.cu), _i32(b.total), window=window,
                               sinks=sinks, max_new=max_new, **sc).double().cpu()
        for r, (c, n) in enumerate(b.lens):
            rows = slice(b.cu[r], b.cu[r + 1])
            want, mag = paged.attend(b.q[rows], b.k[r], b.v[r], c, window, sinks)
            tol = _tol(b, mag, c + n)
            assert bool(((x[rows] - want).abs() <= tol).all()) and bool(((y[rows] - want).abs() <= tol).all()), r
            assert bool(((x[rows] - y[rows]).abs() <= 2 * tol).all())


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 2), (6, 0), (20, 40)])
@pytest.mark.parametrize("kind", ["random", "roots"])
def test_every_token_sees_what_decoding_its_line_shows_it(kind, window, sinks, D, bits):
    """A token's row against a sequence of its context and its ancestors, under the window by positions."""
    lens = [(0, 30), (11, 8), (50, 70), (2, 1), (0, 0), (100, 33)]
    b = _planned(Batch(lens, kind=kind, D=D, bits=bits, seed=window), window, sinks)
    got = b.gpu(window=window, sinks=sinks, max_new=70).double().cpu()
    deep = 0
    for r, (c, n) in enumerate(lens):
        for t, line in enumerate(ref.lines(b.trees[r])):
            at = [*range(c), *(c + j for j in reversed(line))]
            deep = max(deep, len(line))
            row = b.cu[r] + t
            want, mag = paged.attend(b.q[row:row + 1], b.k[r][at], b.v[r][at], len(at) - 1, window, sinks)
            assert bool(((got[row:row + 1] - want).abs() <= _tol(b, mag, len(at))).all()), (r, t)
    assert deep > 5


def test_a_long_line_under_a_window():
    """1024 new tokens in a line, whose keys are cut into pieces, under windows of 50 and 700."""
    for window, sinks in ((50, 4), (700, 0)):
        b = _planned(Batch([(100, 1024), (0, 700)], kind="chain", Hq=2, Hk=1, D=64, seed=4), window, sinks)
        x = b.gpu(window=window, sinks=sinks, max_new=1024).double().cpu()
        for r, (c, n) in enumerate(b.lens):
            rows = slice(b.cu[r], b.cu[r + 1])
            want, mag = paged.attend(b.q[rows], b.k[r], b.v[r], c, window, sinks)
            assert bool(((x[rows] - want).abs() <= _tol(b, mag, c + n)).all())


def test_a_captured_plan_under_a_window_replays():
    """Parents and lengths change between the replays, with eager calls in between."""
    g = torch.Generator().manual_seed(2)
    ns, cu = [40, 0, 130, 7], _i32(_cu([40, 0, 130, 7]))
    parents, lens = _i32([p for n in ns for p in _tree(n, "chain", g)]), _i32([60, 5, 131, 9])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fa.plan_tree(parents, cu, lens, max_new=130, window=9, sinks=4)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fa.plan_tree(parents, cu, lens, max_new=130, window=9, sinks=4)
    for i in range(4):
        tree = [p for n in ns for p in _tree(n, ("chain", "random")[i % 2], g)]
        parents.copy_(torch.tensor(tree, dtype=I32))
        lens.add_(i)
        graph.replay()
        eager = fa.plan_tree(parents, cu, lens, max_new=130, window=9, sinks=4)
        torch.cuda.synchronize()
        pos, mask = ref.plan(tree, cu.tolist(), lens.tolist(), 3, 9, 4)
        assert out.positions.tolist() == eager.positions.tolist() == pos
        assert torch.equal(out.mask, eager.mask) and torch.equal(out.mask.cpu(), _words(mask))


@pytest.mark.parametrize("window,sinks", [(4, 0), (5, 2)])
def test_drafts_under_a_short_window_equal_token_by_token(window, sinks):
    """A serving loop whose trees are deeper than the window: the kept tokens and their outputs are those of decoding one token
    after the other.  |v| is up to 5; both outputs are within the tolerance above."""
    B, N, Hq, Hk, D, ps, steps = 3, 12, 4, 2, 64, 16, 6
    m, inv = Model(97, Hq, Hk, D, 3), fa.rope_frequencies(D, device=DEV)[0]

    def fresh():
        kc, vc = (torch.zeros(32, ps, Hk, D, dtype=BF, device=DEV) for _ in range(2))
        return dict(kc=kc, vc=vc, table=torch.zeros(B, 8, dtype=I32, device=DEV), lens=torch.zeros(B, dtype=I32, device=DEV),
                    free=torch.arange(32, dtype=I32, device=DEV), count=_i32([32]))

    first, a = torch.tensor([3, 50, 11], device=DEV), fresh()
    tokens, line, outs = first, [[] for _ in range(B)], [[] for _ in range(B)]
    for _ in range(N * steps):
        plan = fa.plan_step(a["table"], a["lens"], _i32([1] * B), a["free"], a["count"], page_size=ps, num_tokens=B)
        q = fa.rope_cache(m.q[tokens], m.k[tokens], m.v[tokens], plan.positions, plan.slots, a["kc"], a["vc"], inv)
        o = fa.paged_attention(q, a["kc"], a["vc"], a["table"], plan.cu_lens, plan.seq_lens, max_new=1, window=window, sinks=sinks)
        for b, t in enumerate(tokens.tolist()):
            line[b].append(t)
            outs[b].append(o[b])
        tokens = m.next(tokens, plan.positions)
        a["lens"], a["count"] = plan.seq_lens, plan.free_count
    s, at, deepest = fresh(), [0] * B, 0
    g = torch.Generator().manual_seed(9)
    for _ in range(steps):
        parents, toks = [], []
        for b in range(B):                                 # the right line as far as a chance goes, wrong tokens beside it
            p, right = [-1], [0]
            for t in range(1, N):
                p.append(right[-1] if torch.rand((), generator=g) < 0.85 else int(torch.randint(0, t, (), generator=g)))
                good = p[t] == right[-1] and torch.rand((), generator=g) < 0.95
                right += [t] if good else []
            depth = [len(x) - 1 for x in ref.lines(p)]
            toks += [line[b][at[b] + depth[t]] if t in right else 96 - line[b][at[b] + depth[t]] for t in range(N)]
            parents += p
        par, tokens = _i32(parents), torch.tensor(toks, device=DEV)
        plan = fa.plan_step(s["table"], s["lens"], _i32([N] * B), s["free"], s["count"], page_size=ps, num_tokens=B * N)
        tree = fa.plan_tree(par, plan.cu_lens, plan.seq_lens, max_new=N, window=window, sinks=sinks)
        q = fa.rope_cache(m.q[tokens], m.k[tokens], m.v[tokens], tree.positions, plan.slots, s["kc"], s["vc"], inv)
        o = fa.tree_attention(q, s["kc"], s["vc"], s["table"], plan.cu_lens, plan.seq_lens, tree.mask, positions=tree.positions,
                              max_new=N, window=window, sinks=sinks)
        acc = fa.accept_tree(par, tokens, m.next(tokens, tree.positions), plan.cu_lens, max_new=N)
        fa.move_kept(s["kc"], s["vc"], s["table"], plan.cu_lens, plan.seq_lens, acc.kept)
        back = fa.plan_step(s["table"], plan.seq_lens, acc.dropped, s["free"], plan.free_count, page_size=ps, num_tokens=0)
        s["lens"], s["count"] = back.seq_lens, back.free_count
        kept, lens = acc.kept.tolist(), acc.kept_lens.tolist()
        for b in range(B):
            for i, t in enumerate(kept[b * N:b * N + lens[b]]):
                assert toks[b * N + t] == line[b][at[b] + i]
                err = (o[b * N + t].double() - outs[b][at[b] + i].double()).abs().max().item()
                assert err <= 2 * (3 * torch.finfo(BF).eps / 2 + 2e-4) * 5.0, (b, i, err)
            at[b] += lens[b]
            deepest = max(deepest, lens[b])
            assert int(acc.next_tokens[b]) == line[b][at[b]]
    assert s["lens"].tolist() == at and deepest > window
