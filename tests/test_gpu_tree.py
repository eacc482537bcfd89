"""Trees of drafted tokens on the GPU against plain forms (``oracle.tree``): plans, attention, acceptance, moves, and
a serving loop of them.

Tolerance of the attention, as in ``test_gpu_serving``: the weights are rounded to the input type before the product
with v, the row sum is of the rounded ones, the result is rounded once: 3 u times the softmax average of |v| (u = half
a step of the type); scores of these inputs are off by less than 1e-4 (2e-4 of the result); in f16 a weight below 2^-14 of
the running maximum has the absolute error 2^-25.  An e4m3 number is one of bf16 and of f16, so 8-bit caches add
nothing; their scales are applied in 32 bits (2^-23).
"""
from __future__ import annotations

import pytest
import torch

import fftsparse_amd as fa
from oracle import tree as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3 = torch.float8_e4m3fn
I32 = torch.int32


def _i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


def _cu(ns):
    return torch.tensor([0] + list(ns)).cumsum(0).tolist()


def _tree(n, kind, g):
    """Parents of one tree of n tokens."""
    i = torch.arange(n)
    if kind == "chain":
        p = i - 1
    elif kind == "star":
        p = torch.zeros_like(i)
    elif kind == "roots":                                  # some tokens follow the context, not each other
        p = torch.where(torch.rand(n, generator=g) < 0.3, -1, (i * torch.rand(n, generator=g)).long())
    else:
        p = torch.minimum((i * torch.rand(n, generator=g)).long(), i - 1)
    p = p.tolist()
    if n:
        p[0] = -1
    return p


def _signed(x):
    return x - (1 << 64) if x >> 63 else x


def _words(rows):
    return torch.tensor([[_signed(x) for x in r] for r in rows], dtype=torch.int64)


# ---- plans -------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["chain", "star", "roots", "random"])
@pytest.mark.parametrize("ns,max_new", [([1], 1), ([5], 5), ([0, 3, 0, 64, 65, 1, 63, 0], 65), ([200, 7, 128, 129], 200),
                                        ([1024, 1, 1000], 1024), ([300, 20], 100), ([70, 64], 64)])
def test_plan_tree(kind, ns, max_new):
    g = torch.Generator().manual_seed(len(ns) + max_new)
    parents = [p for n in ns for p in _tree(n, kind, g)] + [0] * 7
    cu, words = _cu(ns), -(-max_new // 64)
    lens = [n + 11 * b for b, n in enumerate(ns)]
    got = fa.plan_tree(_i32(parents), _i32(cu), _i32(lens), max_new=max_new)
    pos, mask = ref.plan(parents, cu, lens, words)
    assert got.positions.tolist() == pos
    assert torch.equal(got.mask.cpu(), _words(mask))


def test_plan_tree_many_requests_and_out():
    g = torch.Generator().manual_seed(3)
    ns = [(7 * b) % 19 for b in range(3000)]
    parents = [p for n in ns for p in _tree(n, "random", g)]
    cu, lens = _cu(ns), [n + b % 50 for b, n in enumerate(ns)]
    out = fa.TreePlan(torch.empty(len(parents), dtype=I32, device=DEV), torch.empty(len(parents), 1, dtype=torch.int64, device=DEV))
    got = fa.plan_tree(_i32(parents), _i32(cu), _i32(lens), max_new=18, out=out)
    pos, mask = ref.plan(parents, cu, lens, 1)
    assert got is out and out.positions.tolist() == pos and torch.equal(out.mask.cpu(), _words(mask))


def test_plan_tree_parents_that_are_none():
    """Numbers that name no earlier token: the token follows the context."""
    parents = [5, 1, 1, -9, 2 ** 31 - 1, -2 ** 31, 4, 3]
    got = fa.plan_tree(_i32(parents), _i32([0, 8]), _i32([20]), max_new=8)
    pos, mask = ref.plan(parents, [0, 8], [20], 1)
    assert pos == [12, 12, 13, 12, 12, 12, 13, 13]
    assert got.positions.tolist() == pos and torch.equal(got.mask.cpu(), _words(mask))


def test_plan_tree_without_rows():
    assert fa.plan_tree(_i32([]), _i32([0, 0]), _i32([4]), max_new=1).mask.shape == (0, 1)
    got = fa.plan_tree(_i32([0, 0]), _i32([0, 0]), _i32([4]), max_new=1)
    assert got.positions.tolist() == [-1, -1] and got.mask.tolist() == [[0], [0]]


# ---- attention -----------------------------------------------------------------------

class Batch:
    """Requests (context, new tokens) in a paged cache on the CPU: pages in random order, NaN in every slot without a
    token, numbers outside the cache in table entries that are not used."""

    def __init__(self, lens, *, kind="random", Hq=4, Hk=2, D=128, ps=16, dtype=BF, bits=16, hnd=False, pad=0, seed=0):
        g = torch.Generator().manual_seed(seed)
        total = [c + n for c, n in lens]
        need = [-(-t // ps) for t in total]
        P, pages = max(need) + 2, sum(need) + 3
        perm = torch.randperm(pages, generator=g).tolist()
        table = torch.full((len(lens), P), 2 ** 31 - 1, dtype=I32)
        table[::2] = -7
        self.store = E4M3 if bits == 8 else dtype
        self.ks, self.vs = (0.005 + 0.02 * torch.rand(Hk, generator=g) for _ in range(2))
        shape = (pages, Hk, ps, D) if hnd else (pages, ps, Hk, D)
        kc, vc = (torch.full(shape, float("nan")).to(self.store) for _ in range(2))
        self.kc, self.vc = (x.transpose(1, 2) if hnd else x for x in (kc, vc))
        self.k, self.v = [], []
        for b, t in enumerate(total):
            k, v = (torch.randn(t, Hk, D, generator=g) for _ in range(2))
            if t:
                k[0] *= 3
            if bits == 8:
                k, v = ((x / s[:, None]).clamp(-448.0, 448.0).to(E4M3) for x, s in ((k, self.ks), (v, self.vs)))
            else:
                k, v = k.to(dtype), v.to(dtype)
            for i in range(need[b]):
                table[b, i] = pg = perm.pop()
                m = min(ps, t - i * ps)
                self.kc[pg, :m], self.vc[pg, :m] = k[i * ps:i * ps + m], v[i * ps:i * ps + m]
            if bits == 8:
                k, v = k.double() * self.ks.double()[:, None], v.double() * self.vs.double()[:, None]
            self.k.append(k)
            self.v.append(v)
        self.ns = [n for _, n in lens]
        self.cu, self.T, self.total, self.lens, self.dtype, self.bits = _cu(self.ns), sum(self.ns), total, lens, dtype, bits
        self.trees = [_tree(n, kind, g) for n in self.ns]
        self.q = torch.randn(self.T + pad, Hq, D, generator=g).to(dtype)
        self.table, self.words = table, -(-max(max(self.ns), 1) // 64)
        self.pos, rows = ref.plan([p for t in self.trees for p in t], self.cu, total, self.words)
        self.mask = torch.cat([_words(rows), torch.full((pad, self.words), -1, dtype=torch.int64)]) if self.T else \
            torch.zeros(pad, self.words, dtype=torch.int64)

    def sees(self, b):
        m = self.mask[self.cu[b]:self.cu[b + 1]]
        j = torch.arange(self.ns[b])
        ok = torch.zeros(self.ns[b], self.ns[b], dtype=torch.bool)
        inside = j[j < 64 * m.shape[1]]
        ok[:, inside] = (m[:, inside // 64] >> (inside % 64) & 1).bool()
        return ok

    def dev_caches(self):
        def dev(x):
            y = x.view(torch.uint8) if x.dtype == E4M3 else x
            y = y.to(DEV) if y.is_contiguous() else y.transpose(1, 2).to(DEV).transpose(1, 2)
            return y.view(E4M3) if x.dtype == E4M3 else y
        return dev(self.kc), dev(self.vc)

    def gpu(self, **kw):
        if self.bits == 8:
            kw.update(k_scale=self.ks.to(DEV), v_scale=self.vs.to(DEV))
        if kw.get("window") is not None and "positions" not in kw:
            kw["positions"] = _i32(self.pos + [0] * (len(self.q) - self.T))
        return fa.tree_attention(kw.pop("q", self.q.to(DEV)), *self.dev_caches(), self.table.to(DEV), _i32(self.cu),
                                 _i32(self.total), self.mask.to(DEV), **kw)

    def check(self, got, window=None, sinks=0, scale=None, present=None, pos=None, note=""):
        u = torch.finfo(self.dtype).eps / 2
        pos = self.pos if pos is None else pos
        for b, (c, n) in enumerate(self.lens):
            if not n:
                continue
            rows = slice(self.cu[b], self.cu[b + 1])
            want, mag = ref.attend(self.q[rows], self.k[b], self.v[b], n, self.sees(b), window, sinks, scale,
                                   None if present is None else present[b], pos[rows])
            tol = (3 * u + 2e-4) * mag + 1e-30
            if self.dtype is F16:
                tol = tol + (c + n) * 2.0 ** -25 * 8.0 + 2.0 ** -25
            x = got[rows].double().cpu()
            err = (x - want).abs()
            assert bool(torch.isfinite(x).all()), (b, note)
            assert bool((err <= tol).all()), (b, note, (err / tol).max().item(), err.max().item())


SMALL = [(0, 1), (5, 8), (62, 3), (0, 5), (64, 1), (999, 8), (0, 0), (129, 2), (30, 0)]       # few rows
WIDE = [(0, 1), (0, 17), (100, 33), (1000, 130), (0, 0), (3, 250), (64, 64), (40, 65), (17, 3)]
WINDOWS = [(None, 0), (1, 0), (1, 3), (16, 4), (100, 0), (64, 70), (130, 200), (5000, 3)]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("kind", ["chain", "star", "roots", "random"])
@pytest.mark.parametrize("lens", [SMALL, WIDE], ids=["small", "wide"])
def test_tree_attention(lens, kind, bits):
    b = Batch(lens, kind=kind, bits=bits, seed=1)
    b.check(b.gpu())
    b.check(b.gpu(max_new=max(b.ns)))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("lens", [SMALL, WIDE], ids=["small", "wide"])
def test_tree_attention_windows(lens, window, sinks, bits):
    b = Batch(lens, bits=bits, ps=32, seed=2)
    b.check(b.gpu(window=window, sinks=sinks, max_new=max(b.ns)), window, sinks)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (8, 1), (7, 1), (6, 2), (28, 4), (33, 1)])
@pytest.mark.parametrize("ps", [16, 48, 64, 256])
def test_tree_attention_heads_pages_types(dtype, D, Hq, Hk, ps, bits):
    b = Batch([(0, 1), (77, 4), (0, 5), (300, 40), (450, 1), (20, 70)], Hq=Hq, Hk=Hk, D=D, ps=ps, dtype=dtype, bits=bits,
              hnd=ps == 48, seed=ps)
    b.check(b.gpu())
    b.check(b.gpu(window=50, sinks=2), 50, 2)


@pytest.mark.parametrize("max_new", [None, 1, 2, 40, 1000])
@pytest.mark.parametrize("lens", [SMALL, WIDE], ids=["small", "wide"])
def test_tree_attention_is_right_for_any_max_new(lens, max_new):
    for window in (None, 60):
        b = Batch(lens, seed=5)
        b.check(b.gpu(max_new=max_new, window=window), window)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("lens,max_new", [([(20000, 8)], 8), ([(9000, 20)], None), ([(6000, 100), (40, 1)], None),
                                          ([(2500, 16), (900, 3), (5000, 7)], 16)])
def test_tree_attention_long(lens, max_new, bits):
    """Long contexts, whose keys are split over workgroups and joined."""
    b = Batch(lens, ps=64, bits=bits, seed=3)
    b.check(b.gpu(max_new=max_new))
    b.check(b.gpu(max_new=max_new, window=4000, sinks=10), 4000, 10)


@pytest.mark.parametrize("max_new", [None, 6])
def test_tree_attention_many_requests(max_new):
    lens = [((7 * i) % 45, i % 7) for i in range(700)] + [(3000, 5)]
    b = Batch(lens, Hq=4, Hk=1, D=64, seed=2)
    b.check(b.gpu(max_new=max_new))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("lens", [SMALL, WIDE, [(3000, 1000), (0, 1024)]], ids=["small", "wide", "most"])
def test_masks_of_any_kind(lens, bits):
    """Bits at random: tokens that see later ones, rows that see no new token, and none at all where there is no context."""
    b = Batch(lens, Hq=2, Hk=1, D=64, bits=bits, seed=9)
    g = torch.Generator().manual_seed(10)
    b.mask = torch.randint(-2 ** 63, 2 ** 63 - 1, b.mask.shape, generator=g)
    b.mask[::3] = 0
    b.mask[1::5] = -1
    got = b.gpu()
    b.check(got)
    empty = [b.cu[r] for r, (c, n) in enumerate(lens) if c == 0 and n and not b.sees(r)[0].any()]
    for t in empty:
        assert bool((got[t] == 0).all())
    b.check(b.gpu(max_new=max(b.ns), window=20, sinks=1), 20, 1)


def test_a_row_that_sees_nothing_is_0():
    b = Batch([(0, 3), (0, 40)], seed=12)
    b.mask.zero_()
    for max_new in (None, 3):
        assert bool((b.gpu(max_new=max_new) == 0).all())


@pytest.mark.parametrize("words", [1, 2])
def test_tokens_past_the_masks_words_are_seen_by_none(words):
    b = Batch([(50, 200), (10, 130), (7, 3)], seed=13)
    b.mask = b.mask[:, :words].contiguous()
    b.check(b.gpu())


def test_positions_are_held_to_those_of_the_new_tokens():
    b = Batch(SMALL, seed=14)
    far = _i32([(-2 ** 31, 2 ** 31 - 1, 0)[t % 3] for t in range(b.T)])
    pos = [0] * b.T
    for r, (c, n) in enumerate(b.lens):
        for t in range(b.cu[r], b.cu[r + 1]):
            pos[t] = min(max(int(far[t]), c), c + n - 1)
    b.check(b.gpu(window=30, sinks=2, positions=far), 30, 2, pos=pos)


def test_a_chain_is_paged_attention():
    for lens in (SMALL, WIDE):
        b = Batch(lens, kind="chain", seed=15)
        b.check(fa.paged_attention(b.q.to(DEV), *b.dev_caches(), b.table.to(DEV), _i32(b.cu), _i32(b.total)))


@pytest.mark.parametrize("bits", [16, 8])
def test_rows_behind_the_last_request_stay(bits):
    for lens in (SMALL, WIDE):
        b = Batch(lens, pad=37, bits=bits, seed=6)
        out = torch.full(b.q.shape, 7.0, dtype=BF, device=DEV)
        got = b.gpu(out=out, max_new=max(b.ns))
        assert got.data_ptr() == out.data_ptr()
        b.check(got)
        assert bool((got[b.T:] == 7.0).all())


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("lens", [SMALL, WIDE], ids=["small", "wide"])
def test_pages_that_are_none(lens, bits):
    """Table entries outside the cache, in the context and among the new tokens: their tokens are not there."""
    b = Batch(lens, ps=16, bits=bits, seed=16)
    present = [torch.ones(t, dtype=torch.bool) for t in b.total]
    for r, t in enumerate(b.total):
        for i in range(-(-t // 16)):
            if (i + r) % 3 == 0:
                b.table[r, i] = (-1, 10 ** 9, len(b.kc))[i % 3]
                present[r][16 * i:16 * i + 16] = False
    b.check(b.gpu(), present=present)
    b.check(b.gpu(max_new=max(b.ns), window=100, sinks=3), 100, 3, present=present)


def test_more_new_tokens_than_tokens():
    """seq_lens below the new tokens: the first of them have no place and are not there."""
    b = Batch([(0, 40), (0, 6)], seed=17)
    b.total = [30, 4]
    for r, t in enumerate(b.total):
        b.k[r], b.v[r] = b.k[r][:t], b.v[r][:t]
    for max_new in (None, 40):
        b.check(b.gpu(max_new=max_new))


def test_repeats_and_streams():
    for lens, bits in ((SMALL, 16), (WIDE, 8), ([(20000, 8)], 8)):
        b = Batch(lens, bits=bits, seed=18)
        x = b.gpu(max_new=max(b.ns))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            y = b.gpu(max_new=max(b.ns))
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(x, y)


def test_output_in_the_queries_place_and_strides():
    for lens in (SMALL, WIDE):
        b = Batch(lens, seed=19)
        wide = torch.zeros(b.T, 12, 128, dtype=BF, device=DEV)
        wide[:, 4:8] = b.q.to(DEV)
        q = wide[:, 4:8]
        got = b.gpu(q=q, out=q)
        b.check(got)
        assert bool((wide[:, :4] == 0).all()) and bool((wide[:, 8:] == 0).all())


# ---- acceptance ------------------------------------------------------------------------

def _accept_case(ns, g, vocab, given=0.0, kind="random"):
    parents = [p for n in ns for p in _tree(n, kind, g)]
    T = len(parents)
    tokens = torch.randint(0, vocab, (T,), generator=g)
    tokens[torch.rand(T, generator=g) < given] = -1
    return parents, tokens.tolist(), torch.randint(0, vocab, (T,), generator=g).tolist()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("vocab,given", [(2, 0.0), (3, 0.2), (50000, 0.0), (1, 0.0), (50000, 1.0)])
@pytest.mark.parametrize("ns,max_new", [([1], 1), ([9], 9), ([0, 3, 0, 64, 65, 1, 40, 0], 65), ([1024, 700], 1024),
                                        ([300, 20, 100], 100)])
def test_accept_tree(ns, max_new, vocab, given, dtype):
    g = torch.Generator().manual_seed(vocab + max_new)
    for kind in ("random", "chain", "roots"):
        parents, tokens, chosen = _accept_case(ns, g, vocab, given, kind)
        pad = [0] * 5
        args = [torch.tensor(x + pad, dtype=d, device=DEV) for x, d in ((parents, I32), (tokens, dtype), (chosen, dtype))]
        got = fa.accept_tree(*args, _i32(_cu(ns)), max_new=max_new)
        kept, lens, dropped, after = ref.accept(parents, tokens, chosen, _cu(ns), max_new)
        assert got.kept.tolist() == kept + [-1] * 5
        assert (got.kept_lens.tolist(), got.dropped.tolist(), got.next_tokens.tolist()) == (lens, dropped, after)
        assert got.next_tokens.dtype == dtype


def test_accept_tree_large_tokens_and_out():
    """64-bit tokens that agree in their low halves only; a former result written again."""
    big = 1 << 40
    parents, tokens, chosen = [-1, 0, 0, 1], [7, 5, big + 5, 9], [big + 5, 9, 9, 3]
    t64 = [torch.tensor(x, dtype=torch.int64, device=DEV) for x in (tokens, chosen)]
    got = fa.accept_tree(_i32(parents), *t64, _i32([0, 4]), max_new=4)
    assert got.kept.tolist() == [0, 2, -1, -1] and got.next_tokens.tolist() == [9]
    again = fa.accept_tree(_i32(parents), t64[0], torch.tensor([5, 9, 9, 3], device=DEV), _i32([0, 4]), max_new=4, out=got)
    assert again is got and got.kept.tolist() == [0, 1, 3, -1] and got.next_tokens.tolist() == [3]


def test_accept_tree_without_rows():
    e = _i32([])
    got = fa.accept_tree(e, e, e, _i32([0, 0, 0]), max_new=1)
    assert got.kept_lens.tolist() == [0, 0] and got.dropped.tolist() == [0, 0] and got.next_tokens.tolist() == [-1, -1]


def test_accept_tree_many_requests():
    g = torch.Generator().manual_seed(8)
    ns = [(5 * b) % 23 for b in range(2500)]
    parents, tokens, chosen = _accept_case(ns, g, 2)
    got = fa.accept_tree(_i32(parents), _i32(tokens), _i32(chosen), _i32(_cu(ns)), max_new=22)
    kept, lens, dropped, after = ref.accept(parents, tokens, chosen, _cu(ns), 22)
    assert (got.kept.tolist(), got.kept_lens.tolist(), got.dropped.tolist(), got.next_tokens.tolist()) == \
        (kept, lens, dropped, after)


# ---- moves -----------------------------------------------------------------------------

def _moved(cache, table, cu, lens, kept, ps):
    """The same on the CPU, on a copy: cache [layers, pages, ps, Hk, D] of bytes."""
    out = cache.clone()
    for b, L in enumerate(lens):
        n = cu[b + 1] - cu[b]
        for i in range(n):
            j = kept[cu[b] + i]
            if not i < j < n:
                continue
            s, d = L - n + j, L - n + i
            ps_, pd = int(table[b, s // ps]), int(table[b, d // ps])
            if 0 <= ps_ < cache.shape[1] and 0 <= pd < cache.shape[1]:
                out[:, pd, d % ps] = cache[:, ps_, s % ps]
    return out


@pytest.mark.parametrize("dtype,Hk,D", [(BF, 8, 128), (F16, 3, 64), (E4M3, 4, 128), (E4M3, 1, 16), (F32, 2, 40), (F32, 64, 128),
                                        (BF, 96, 128)])
@pytest.mark.parametrize("layers,form", [(1, "one"), (3, "tensor"), (3, "list"), (70, "list"), (2, "hnd")])
def test_move_kept(dtype, Hk, D, layers, form):
    if layers == 70 and Hk > 8:
        layers = 3
    g = torch.Generator().manual_seed(Hk + D)
    ps, ns = 16, [0, 1, 12, 40, 7, 0, 100, 3]
    lens = [n + c for n, c in zip(ns, (4, 0, 30, 9, 15, 0, 61, 16))]
    cu = _cu(ns)
    need = [-(-t // ps) for t in lens]
    pages = sum(need) + 2
    perm = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(ns), max(need) + 1), -1, dtype=I32)
    for b, m in enumerate(need):
        for i in range(m):
            table[b, i] = perm.pop()
    kept = [-1] * cu[-1]
    for b, n in enumerate(ns):
        if n:
            path = [0] + (torch.randperm(n - 1, generator=g)[:(n + 1) // 2] + 1).sort().values.tolist()
            kept[cu[b]:cu[b] + len(path)] = path
    es = torch.empty(0, dtype=dtype).element_size()
    raw = [torch.randint(0, 256, (layers, pages, ps, Hk, D * es), generator=g, dtype=torch.uint8) for _ in range(2)]
    if form == "hnd":
        dev = [r.transpose(2, 3).contiguous().to(DEV).view(dtype).transpose(2, 3) for r in raw]
    else:
        dev = [r.to(DEV).view(dtype) for r in raw]
    given = {"one": lambda x: x[0], "list": list}.get(form, lambda x: x)
    fa.move_kept(given(dev[0]), given(dev[1]), table.to(DEV), _i32(cu), _i32(lens), _i32(kept + [-1] * 4))
    for r, x in zip(raw, dev):
        x = x.transpose(2, 3).contiguous().view(torch.uint8).transpose(2, 3) if form == "hnd" else x.view(torch.uint8)
        assert torch.equal(x.cpu(), _moved(r, table, cu, lens, kept, ps))


def test_move_kept_bad_pages_and_lengths():
    """Tokens without a page stay, nothing else is touched; lengths past the table and below the new tokens too."""
    g = torch.Generator().manual_seed(1)
    raw = torch.randint(0, 256, (1, 6, 16, 2, 256), generator=g, dtype=torch.uint8)
    dev = raw.to(DEV).view(BF)
    table = torch.tensor([[0, -1, 10 ** 9, 1], [2, 3, 6, 4], [5, 5, 5, 5]], dtype=I32)
    cu, kept = [0, 40, 50, 60], [0] + list(range(3, 30)) + [-1] * 12 + [0, 5] + [-1] * 8 + [0, 4, 5, 6, 9] + [-1] * 5
    lens = [40, 40, 7]
    fa.move_kept(dev, dev.clone(), table.to(DEV), _i32(cu), _i32(lens), _i32(kept))
    want = raw.clone()
    for b in range(2):
        want = _moved(want, table[b:b + 1], [0, cu[b + 1] - cu[b]], [lens[b]], kept[cu[b]:cu[b + 1]], 16)
    for i, j in ((1, 4), (2, 5), (3, 6), (4, 9)):          # its new token i stands at i - 3
        if i >= 3:
            want[0, 5, i - 3] = raw[0, 5, j - 3]
    assert torch.equal(dev.view(torch.uint8).cpu(), want)
    before = dev.clone()
    fa.move_kept(dev, dev.clone(), table.to(DEV), _i32([0, 2, 2, 2]), _i32([2 ** 31 - 1, 0, 0]), _i32([1, -1]))
    fa.move_kept(dev, dev.clone(), table.to(DEV), _i32([0, 2, 2, 2]), _i32([-2 ** 31, 0, 0]), _i32([1, -1]))
    assert torch.equal(dev.view(torch.uint8), before.view(torch.uint8))


# ---- a serving loop ----------------------------------------------------------------------

class Model:
    """A toy model: a token's q, k and v by its number; what it takes next is a function of the token and its position."""

    def __init__(self, vocab, Hq, Hk, D, seed):
        g = torch.Generator().manual_seed(seed)
        self.q, self.k, self.v = (torch.randn(vocab, h, D, generator=g).to(BF).to(DEV) for h in (Hq, Hk, Hk))
        self.vocab = vocab

    def next(self, tokens, positions):
        return (tokens * 7 + positions.long() * 3 + 1) % self.vocab


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("captured", [False, True])
def test_speculative_serving_equals_token_by_token(bits, captured):
    """Steps of drafted trees leave the tokens, lengths, pages' contents and the kept tokens' outputs that decoding one token
    after the other does.  Captured: the whole step as one graph, replayed with eager work between the replays."""
    B, Hq, Hk, D, ps, vocab, N, steps = 5, 4, 2, 64, 16, 97, 12, 9
    m = Model(vocab, Hq, Hk, D, 3)
    inv, _ = fa.rope_frequencies(D, device=DEV)
    store = E4M3 if bits == 8 else BF
    scales = dict(k_scale=torch.tensor([0.02, 0.03], device=DEV), v_scale=torch.tensor([0.01, 0.025], device=DEV)) if bits == 8 else {}
    pages = 64

    def fresh():
        kc, vc = (torch.zeros(2, pages, ps, Hk, D, device=DEV).to(store) for _ in range(2))     # two layers
        return dict(kc=kc, vc=vc, table=torch.zeros(B, 12, dtype=I32, device=DEV), lens=torch.zeros(B, dtype=I32, device=DEV),
                    free=torch.arange(pages, dtype=I32, device=DEV), count=_i32([pages]))

    def layers(s, tokens, positions, slots, plan, attend):
        outs = []
        for l in range(2):
            q = fa.rope_cache(m.q[tokens] * (l + 1), m.k[tokens], m.v[tokens], positions, slots, s["kc"][l], s["vc"][l], inv,
                              **scales)
            outs.append(attend(q, s["kc"][l], s["vc"][l], s["table"], plan.cu_lens, plan.seq_lens))
        return torch.stack(outs, 1)

    # token by token
    first = torch.tensor([3, 50, 11, 96, 0], device=DEV)
    a = fresh()
    tokens, line, outs = first.clone(), [[] for _ in range(B)], [[] for _ in range(B)]
    for step in range(N * steps):
        plan = fa.plan_step(a["table"], a["lens"], _i32([1] * B), a["free"], a["count"], page_size=ps, num_tokens=B)
        o = layers(a, tokens, plan.positions, plan.slots, plan,
                   lambda *x: fa.paged_attention(*x, max_new=1, window=40, sinks=2, **scales))
        for b in range(B):
            line[b].append(int(tokens[b]))
            outs[b].append(o[b])
        tokens = m.next(tokens, plan.positions)
        a["lens"], a["count"] = plan.seq_lens, plan.free_count
        if min(plan.seq_lens.tolist()) >= 12 * ps - N:
            break

    # trees: request b drafts trees of 1 + (N - 1) tokens, some of whose paths are right
    s = fresh()
    g = torch.Generator().manual_seed(4)
    T = B * N
    new = _i32([N, N, 5, N, 1])
    buf = dict(parents=torch.zeros(T, dtype=I32, device=DEV), tokens=torch.zeros(T, dtype=torch.int64, device=DEV))
    res = {}

    def step():
        plan = fa.plan_step(s["table"], s["lens"], new, s["free"], s["count"], page_size=ps, num_tokens=T)
        tree = fa.plan_tree(buf["parents"], plan.cu_lens, plan.seq_lens, max_new=N)
        res["out"] = layers(s, buf["tokens"], tree.positions, plan.slots, plan,
                            lambda *x: fa.tree_attention(*x, tree.mask, positions=tree.positions, max_new=N, window=40, sinks=2,
                                                         **scales))
        chosen = m.next(buf["tokens"], tree.positions)
        acc = fa.accept_tree(buf["parents"], buf["tokens"], chosen, plan.cu_lens, max_new=N)
        fa.move_kept(s["kc"], s["vc"], s["table"], plan.cu_lens, plan.seq_lens, acc.kept)
        back = fa.plan_step(s["table"], plan.seq_lens, acc.dropped, s["free"], plan.free_count, page_size=ps, num_tokens=0)
        s["lens"].copy_(back.seq_lens)
        s["count"].copy_(back.free_count)
        res["acc"], res["cu"], res["lacking"] = acc, plan.cu_lens, plan.lacking

    def drafts(at, last):
        """A tree per request: its guesses continue the right line with some chance, at random places."""
        parents, toks = [], []
        for b, n in enumerate(new.tolist()):
            p = _tree(n, "random", g)
            depth = [len(x) - 1 for x in ref.lines(p)]
            for t in range(n):
                right = line[b][at[b] + depth[t]] if at[b] + depth[t] < len(line[b]) else 0
                toks.append(last[b] if t == 0 else right if torch.rand((), generator=g) < 0.6 else int(
                    torch.randint(0, vocab, (), generator=g)))
            parents += p
        pad = T - len(parents)
        buf["parents"].copy_(_i32(parents + [0] * pad))
        buf["tokens"].copy_(torch.tensor(toks + [0] * pad, device=DEV))

    graph = None
    if captured:
        drafts([0] * B, first.tolist())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()                                         # everything is allocated and loaded once
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for name, x in fresh().items():
            s[name].copy_(x) if s[name].dtype != E4M3 else s[name].view(torch.uint8).copy_(x.view(torch.uint8))
    at, last = [0] * B, first.tolist()
    u = torch.finfo(BF).eps / 2
    for _ in range(steps):
        drafts(at, last)
        graph.replay() if graph is not None else step()
        acc = res["acc"]
        kept, lens, cu = acc.kept.tolist(), acc.kept_lens.tolist(), res["cu"].tolist()
        assert res["lacking"].item() == 0
        for b in range(B):
            path = kept[cu[b]:cu[b] + lens[b]]
            for i, t in enumerate(path):
                assert int(buf["tokens"][cu[b] + t]) == line[b][at[b] + i]
                # both are off by 3 u of the weighted |v| at most, and scores by 1e-4: |v| up to 5
                err = (res["out"][cu[b] + t].double() - outs[b][at[b] + i].double()).abs().max().item()
                assert err <= 2 * (3 * u + 2e-4) * 5.0, (b, i, err)
            at[b] += lens[b]
            last[b] = int(acc.next_tokens[b])
            assert last[b] == line[b][at[b]]
        assert s["lens"].tolist() == at
    assert sum(at) > 2 * steps * B                         # drafts were kept
    # the cache holds what token by token wrote, pages may differ
    for c in ("kc", "vc"):
        x, y = (z[c].view(torch.uint8) if bits == 8 else z[c] for z in (s, a))
        for b in range(B):
            p = torch.arange(at[b], device=DEV)
            assert torch.equal(x[:, s["table"][b, p // ps].long(), p % ps], y[:, a["table"][b, p // ps].long(), p % ps])
    assert s["count"].item() == pages - sum(-(-n // ps) for n in at)
