"""The serving operators on the GPU against plain 64-bit forms (``oracle.paged``).

Tolerances.  A rounding is off by at most u = eps / 2 relative.  Attention: the
weights are rounded to the input type before the product with v (the row sum is
taken from the rounded ones, which doubles the bound) and the result is rounded
once: 3 u times the softmax average of |v|.  Scores are sums of D products in 32
bits: for these inputs (|q|, |k| about 1 to 3 per element) off by less than 1e-4.
In f16 a weight below 2^-14 of the running maximum has the absolute error 2^-25.
Rotations: one rounding of the result, and in 32 bits the cosine and sine (the
angle's rest is rounded to 2^-25 of a turn; 2 units in the last place), two
products and a sum: 2^-20 times the pair's magnitude.
"""
from __future__ import annotations

import pytest
import torch

import fftsparse_amd as fa
from oracle import paged as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
I32 = torch.int32


def _i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _check_attn(got, want, mag, keys, dtype, note=""):
    u = _half_step(dtype)
    tol = (3 * u + 2e-4) * mag + 1e-30
    if dtype is F16:
        tol = tol + keys * 2.0 ** -25 * 8.0 + 2.0 ** -25
    err = (got.double().cpu() - want).abs()
    assert bool(torch.isfinite(got).all()), note
    assert bool((err <= tol).all()), (note, (err / tol).max().item(), err.max().item())


class Batch:
    """A paged cache on the CPU and the GPU with requests of given lengths (cached, new): pages in random order, NaN in
    every slot that holds no token, numbers outside the cache in every table entry that is not used."""

    def __init__(self, lens, *, Hq=4, Hk=2, D=128, ps=16, dtype=BF, hnd=False, pad=0, seed=0, spare=3):
        g = torch.Generator().manual_seed(seed)
        B = len(lens)
        total = [c + n for c, n in lens]
        need = [-(-t // ps) for t in total]
        P = max(need) + 2
        pages = sum(need) + spare
        perm = torch.randperm(pages, generator=g).tolist()
        table = torch.full((B, P), 2 ** 31 - 1, dtype=I32)
        table[::2] = -7
        shape = (pages, Hk, ps, D) if hnd else (pages, ps, Hk, D)
        kc, vc = (torch.full(shape, float("nan"), dtype=dtype) for _ in range(2))
        self.kc, self.vc = (x.transpose(1, 2) if hnd else x for x in (kc, vc))
        self.k, self.v = [], []
        for b, t in enumerate(total):
            k, v = (torch.randn(t, Hk, D, generator=g).to(dtype) for _ in range(2))
            if t:
                k[0] *= 3
            for i in range(need[b]):
                pg = perm.pop()
                table[b, i] = pg
                n = min(ps, t - i * ps)
                self.kc[pg, :n], self.vc[pg, :n] = k[i * ps:i * ps + n], v[i * ps:i * ps + n]
            self.k.append(k)
            self.v.append(v)
        cu = torch.tensor([0] + [n for _, n in lens]).cumsum(0)
        self.T = int(cu[-1])
        self.q = torch.randn(self.T + pad, Hq, D, generator=g).to(dtype)
        self.lens, self.table, self.cu, self.total, self.dtype = lens, table, cu.to(I32), total, dtype

    def gpu(self, **kw):
        dev = {n: getattr(self, n).to(DEV) for n in ("q", "table", "cu")}
        kc, vc = (x.transpose(1, 2).to(DEV).transpose(1, 2) if not x.is_contiguous() else x.to(DEV)
                  for x in (self.kc, self.vc))
        return fa.paged_attention(kw.pop("q", dev["q"]), kc, vc, dev["table"], dev["cu"], _i32(self.total), **kw)

    def want(self, window=None, sinks=0, scale=None):
        r = [ref.attend(self.q[self.cu[b]:self.cu[b + 1]], self.k[b], self.v[b], c, window, sinks, scale)
             for b, (c, n) in enumerate(self.lens) if n]
        return torch.cat([o for o, _ in r]), torch.cat([m for _, m in r])

    def check(self, got, window=None, sinks=0, scale=None, note=""):
        want, mag = self.want(window, sinks, scale)
        _check_attn(got[:self.T], want, mag, max(self.total), self.dtype, note)


DECODE = [(0, 1), (5, 1), (62, 1), (63, 1), (64, 1), (999, 1), (0, 0), (129, 1), (30, 0)]
CHUNKS = [(0, 1), (0, 17), (100, 33), (1000, 130), (0, 0), (3, 257), (64, 64)]
FEW = [(2500, 3), (900, 8)]
WINDOWS = [(None, 0), (1, 0), (1, 3), (16, 4), (100, 0), (64, 70), (130, 200), (5000, 3)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("lens", [DECODE, CHUNKS, FEW], ids=["decode", "chunks", "few"])
def test_paged_attention_windows(lens, window, sinks):
    b = Batch(lens, ps=16, seed=1)
    b.check(b.gpu(window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (8, 1), (7, 1), (6, 2), (28, 4), (33, 1)])
@pytest.mark.parametrize("ps", [16, 48, 64, 256])
def test_paged_attention_heads_pages_types(dtype, D, Hq, Hk, ps):
    b = Batch([(0, 1), (77, 1), (0, 5), (300, 40), (450, 1)], Hq=Hq, Hk=Hk, D=D, ps=ps, dtype=dtype, hnd=ps == 48, seed=ps)
    b.check(b.gpu())
    b.check(b.gpu(window=50, sinks=2), 50, 2)


@pytest.mark.parametrize("max_new", [None, 1, 2, 40, 1000])
@pytest.mark.parametrize("lens", [DECODE, CHUNKS], ids=["decode", "chunks"])
def test_paged_attention_is_right_for_any_max_new(lens, max_new):
    b = Batch(lens, seed=5)
    b.check(b.gpu(max_new=max_new))


@pytest.mark.parametrize("max_new", [None, 1])
def test_paged_attention_many_requests(max_new):
    """More requests than a workgroup has threads, most of them short."""
    lens = [((7 * i) % 45, 1 if i % 5 else 0) for i in range(700)] + [(3000, 1)]
    b = Batch(lens, Hq=4, Hk=1, D=64, seed=2)
    b.check(b.gpu(max_new=max_new))


@pytest.mark.parametrize("max_new", [None, 1])
def test_paged_attention_most_requests(max_new):
    lens = [((7 * i) % 37, 1 if i % 3 else 0) for i in range(4094)] + [(2000, 1), (50, 1)]
    b = Batch(lens, Hq=2, Hk=1, D=64, seed=27)
    b.check(b.gpu(max_new=max_new))


@pytest.mark.parametrize("window,sinks", [(500, 5), (None, 0)])
def test_paged_attention_many_row_tiles(window, sinks):
    """A prompt of more row tiles than the plan of pieces holds in LDS; some of its rows against the oracle."""
    n, ps = 264_000, 256
    pages = -(-n // ps)
    g = torch.Generator().manual_seed(28)
    q, k, v = (torch.randn(n, h, 64, generator=g).to(BF) for h in (4, 1, 1))
    table = torch.randperm(pages, generator=g).to(I32)
    kc, vc = (torch.zeros(pages, ps, 1, 64, dtype=BF) for _ in range(2))
    for x, c in ((k, kc), (v, vc)):
        c[table.long()] = torch.cat([x, x.new_zeros(pages * ps - n, 1, 64)]).view(pages, ps, 1, 64)
    got = fa.paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), table[None].to(DEV), _i32([0, n]), _i32([n]), window=window,
                             sinks=sinks).cpu()
    for i in (0, 1, 31, 32, 1023, 4999, 131_071, 262_143, 262_144, n - 1) if window else (0, 77, n - 1):
        want, mag = ref.attend(q[i:i + 1], k[:i + 1], v[:i + 1], i, window, sinks)
        _check_attn(got[i:i + 1], want, mag, i + 1, BF, i)


@pytest.mark.parametrize("lens,max_new", [([(20000, 1)], 1), ([(9000, 20)], None), ([(6000, 100), (40, 1)], None)])
def test_paged_attention_long(lens, max_new):
    """Long contexts, whose keys are split over workgroups and joined."""
    b = Batch(lens, Hq=4, Hk=2, ps=64, seed=3)
    b.check(b.gpu(max_new=max_new))
    b.check(b.gpu(max_new=max_new, window=4000, sinks=10), 4000, 10)


def test_paged_attention_scale_and_repeat():
    b = Batch(CHUNKS, seed=4)
    x = b.gpu(softmax_scale=0.2)
    b.check(x, scale=0.2)
    assert torch.equal(x, b.gpu(softmax_scale=0.2))


@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-4])
@pytest.mark.parametrize("lens", [DECODE, CHUNKS], ids=["decode", "chunks"])
def test_scales_of_zero_and_near(lens, scale):
    b = Batch(lens, seed=24)
    b.check(b.gpu(softmax_scale=scale), scale=scale)
    b.check(b.gpu(softmax_scale=scale, window=30, sinks=20), 30, 20, scale)


def test_rows_behind_the_last_request_stay():
    for lens in (DECODE, CHUNKS):
        b = Batch(lens, pad=37, seed=6)
        out = torch.full(b.q.shape, 7.0, dtype=BF, device=DEV)
        got = b.gpu(out=out, max_new=1 if lens is DECODE else None)
        assert got.data_ptr() == out.data_ptr()
        b.check(got)
        assert bool((got[b.T:] == 7.0).all())


def test_no_request_has_tokens():
    b = Batch([(5, 0), (0, 0)], pad=4)
    out = torch.full(b.q.shape, 7.0, dtype=BF, device=DEV)
    assert bool((b.gpu(out=out) == 7.0).all())
    assert b.gpu(q=torch.empty(0, 4, 128, dtype=BF, device=DEV)).shape == (0, 4, 128)


def test_strided_queries_and_output():
    b = Batch(CHUNKS, seed=8)
    T = b.T
    wide = torch.zeros(T, 3, 4, 128, dtype=BF, device=DEV)
    wide[:, 1] = b.q.to(DEV)
    heads_first = torch.zeros(4, T, 128, dtype=BF, device=DEV)
    got = b.gpu(q=wide[:, 1], out=heads_first.transpose(0, 1))
    b.check(got)
    odd = torch.zeros(T, 4, 130, dtype=BF, device=DEV)                    # rows that are not aligned: copied
    odd[..., 1:129] = b.q.to(DEV)
    b.check(b.gpu(q=odd[..., 1:129]))


@pytest.mark.parametrize("lens", [DECODE, CHUNKS], ids=["decode", "chunks"])
def test_output_in_the_queries_place_and_a_wide_table(lens):
    b = Batch(lens, ps=48, seed=22)
    want = b.gpu()
    q = b.q.to(DEV)
    wide = torch.full((b.table.shape[0], b.table.shape[1] + 9), 5, dtype=I32, device=DEV)
    wide[:, 4:-5] = b.table.to(DEV)
    got = fa.paged_attention(q, b.kc.to(DEV), b.vc.to(DEV), wide[:, 4:-5], b.cu.to(DEV), _i32(b.total), out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
    x = torch.randn(1, 4, 700, 128, generator=torch.Generator().manual_seed(2)).to(BF).to(DEV)
    k = torch.randn(1, 2, 700, 128, generator=torch.Generator().manual_seed(3)).to(BF).to(DEV)
    want = fa.window_attention(x, k, k, window=90, sinks=4)
    assert torch.equal(fa.window_attention(x, k, k, window=90, sinks=4, out=x.transpose(1, 2)), want)


@pytest.mark.parametrize("max_new", [None, 1])
def test_fewer_tokens_than_rows(max_new):
    """A length below the number of new tokens: the first rows stand before the first token and are 0."""
    b = Batch([(0, 9), (0, 70), (0, 1)], seed=25)
    for take in ((4, 21, 0), (0, 69, 1)):
        got = fa.paged_attention(b.q.to(DEV), b.kc.to(DEV), b.vc.to(DEV), b.table.to(DEV), b.cu.to(DEV), _i32(list(take)),
                                 max_new=max_new)
        for i, (L, (_, n)) in enumerate(zip(take, b.lens)):
            want, mag = ref.attend(b.q[b.cu[i]:b.cu[i + 1]], b.k[i][:L], b.v[i][:L], L - n)
            _check_attn(got[b.cu[i]:b.cu[i + 1]], want, mag, 100, BF, (take, i))
            assert bool((got[b.cu[i]:b.cu[i] + n - L] == 0).all())


@pytest.mark.parametrize("max_new", [None, 1])
def test_more_heads_to_a_group_than_rows_to_a_tile(max_new):
    b = Batch([(0, 1), (200, 1), (70, 3)], Hq=300, Hk=1, D=64, seed=26)
    b.check(b.gpu(max_new=max_new))
    b.check(b.gpu(max_new=max_new, window=20, sinks=17), 20, 17)


def test_row_numbers_that_fall_write_nothing():
    b = Batch([(100, 1), (60, 40), (3, 1)], seed=23)
    for cu in ([0, 5, 2, 42], [0, 1, -7, 42], [40, 0, 41, 42]):
        for max_new in (None, 1):
            out = torch.full(b.q.shape, 7.0, dtype=BF, device=DEV)
            fa.paged_attention(b.q.to(DEV), b.kc.to(DEV), b.vc.to(DEV), b.table.to(DEV), _i32(cu), _i32(b.total), max_new=max_new,
                               out=out)
            assert bool((out == 7.0).all())


@pytest.mark.parametrize("max_new", [None, 1])
def test_pages_outside_the_cache_hold_no_token(max_new):
    lens = [(700, 1), (10, 1), (200, 30), (100, 1)]
    b = Batch(lens, seed=9)
    b.table[0, 3], b.table[0, 20] = -1, 2 ** 31 - 1
    b.table[1] = 10 ** 9                                                   # none left: a row of zeros
    b.table[2, 13] = -2 ** 31
    got = b.gpu(max_new=max_new)
    row = 0
    for r, (c, n) in enumerate(lens):
        present = torch.ones(c + n, dtype=torch.bool)
        for i in range(-(-(c + n) // 16)):
            if not 0 <= int(b.table[r, i]) < b.kc.shape[0]:
                present[16 * i:16 * i + 16] = False
        want, mag = ref.attend(b.q[row:row + n], b.k[r], b.v[r], c, present=present)
        _check_attn(got[row:row + n], want, mag, c + n, BF, r)
        row += n
    assert bool((got[1] == 0).all())


def test_lengths_the_table_cannot_hold_are_cut():
    """Lengths and row numbers from the device that do not fit: read and written within bounds."""
    b = Batch([(100, 1), (60, 1)], seed=10)
    b.table = b.table[:, :4].contiguous()                                  # 64 tokens per request
    kc, vc, q, t, cu = (x.to(DEV) for x in (b.kc, b.vc, b.q, b.table, b.cu))
    got = fa.paged_attention(q, kc, vc, t, cu, _i32([2 ** 31 - 1, 61]))
    want, mag = ref.attend(b.q[:1], b.k[0][:64], b.v[0][:64], 63)
    _check_attn(got[:1], want, mag, 64, BF)
    want, mag = ref.attend(b.q[1:2], b.k[1], b.v[1], 60)
    _check_attn(got[1:], want, mag, 64, BF)
    out = torch.full((2, 4, 128), 7.0, dtype=BF, device=DEV)
    fa.paged_attention(q, kc, vc, t, _i32([0, 0, 0]), _i32([-5, 0]), out=out)
    assert bool((out == 7.0).all())
    # fewer tokens in the cache than new ones: the first rows are before it and see nothing
    got = fa.paged_attention(q, kc, vc, t, _i32([0, 2, 2]), _i32([1, 0]))
    assert bool((got[0] == 0).all()) and torch.equal(got[1], b.v[0][0].to(DEV).repeat_interleave(2, 0))
    # more rows announced than there are
    got = fa.paged_attention(q, kc, vc, t, _i32([0, 1, 50]), _i32([64, 61]))
    assert bool(torch.isfinite(got).all())


def test_other_requests_may_hold_anything():
    b = Batch([(300, 1), (300, 40), (200, 1)], seed=11)
    want = b.gpu()
    for x in (b.kc, b.vc):
        for pg in b.table[1, :22].tolist():
            x[pg] = float("inf")
    got = b.gpu()
    assert torch.equal(got[0], want[0]) and torch.equal(got[41:], want[41:])


def test_tokens_outside_the_window_may_hold_anything():
    """Pages wholly outside every row's window may have gone to others: NaN there, or numbers outside the cache."""
    lens = [(999, 1), (700, 20)]
    b = Batch(lens, seed=12)
    want = b.gpu(window=100, sinks=4)
    for r, (c, n) in enumerate(lens):
        first = (c - 100 + 1) // 16                                        # the first page that a row sees
        for i in range(1, first):
            b.kc[b.table[r, i]] = b.vc[b.table[r, i]] = float("nan")
            if i % 2:
                b.table[r, i] = -1
    assert torch.equal(b.gpu(window=100, sinks=4), want)


def test_scores_that_rise_and_large_values():
    b = Batch([(600, 1), (600, 50)], seed=13)
    u = torch.nn.functional.normalize(torch.randn(128, generator=torch.Generator().manual_seed(1)), dim=0)
    b.q[:] = (8 * u).to(BF)
    for r, k in enumerate(b.k):
        k[:] = (torch.arange(len(k))[:, None, None] / len(k) * 50 * u).to(BF)
        b.v[r] *= 2.0 ** 100
        for i in range(-(-len(k) // 16)):
            n = min(16, len(k) - 16 * i)
            b.kc[b.table[r, i], :n], b.vc[b.table[r, i], :n] = k[16 * i:16 * i + n], b.v[r][16 * i:16 * i + n]
    got = b.gpu()
    want, mag = b.want()
    # scores of about 35 from products of magnitude 400 / 11.3: off by 128 * 2^-24 * 35 in 32 bits
    err = (got.double().cpu() - want).abs()
    assert bool((err <= (3 * 2.0 ** -8 + 128 * 2.0 ** -24 * 70) * mag).all())


def test_far_pages_and_wide_strides():
    """A cache past 2^31 elements, read at its end, and pages of one slab for keys and values."""
    ps, Hk, D, pages = 64, 8, 128, 40000
    b = Batch([(500, 1), (100, 30)], Hq=8, Hk=Hk, ps=ps, seed=14)
    both = torch.empty(pages, 2, ps, Hk, D, dtype=BF, device=DEV)          # 5.2e9 elements
    near = b.kc.shape[0]
    both[pages - near:, 0], both[pages - near:, 1] = b.kc.to(DEV), b.vc.to(DEV)
    table = torch.where((b.table >= 0) & (b.table < near), b.table + pages - near, -1).to(DEV)
    args = (table, b.cu.to(DEV), _i32(b.total))
    b.check(fa.paged_attention(b.q.to(DEV), both[:, 0], both[:, 1], *args))
    b.check(fa.paged_attention(b.q.to(DEV), both[:, 0], both[:, 1], *args, window=77, sinks=5), 77, 5)
    slots = torch.tensor([(pages - 1) * ps + 5, 3, -1, pages * ps], device=DEV)
    k = torch.randn(4, Hk, D, device=DEV).to(BF)
    inv, _ = fa.rope_frequencies(D)
    before = both[pages - 1, :, 6].view(torch.int16).clone()               # NaN among it
    fa.rope_cache(k, k, k, _i32([0, 0, 0, 0]), slots, both[:, 0], both[:, 1], inv)
    assert torch.equal(both[pages - 1, 1, 5], k[0]) and torch.equal(both[0, 0, 3], k[1])
    assert torch.equal(both[pages - 1, :, 6].view(torch.int16), before)


# ---- sliding window on contiguous tensors ---------------------------------------

@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (7, 2), (64, 0), (100, 130), (300, 16)])
@pytest.mark.parametrize("Lq,Lk", [(1, 1), (1, 700), (33, 33), (257, 257), (40, 300), (300, 40), (520, 520)])
def test_window_attention(Lq, Lk, window, sinks):
    g = torch.Generator().manual_seed(Lq + Lk)
    for D, dtype, Hq, Hk in ((128, BF, 4, 1), (64, F16, 6, 2)):
        B = 2
        q, k, v = (torch.randn(B, n, h, D, generator=g).to(dtype) for n, h in ((Lq, Hq), (Lk, Hk), (Lk, Hk)))
        got = fa.window_attention(*(x.to(DEV).transpose(1, 2) for x in (q, k, v)), window=window, sinks=sinks)
        for b in range(B):
            want, mag = ref.attend(q[b], k[b], v[b], Lk - Lq, window, sinks)
            _check_attn(got[b], want, mag, Lk, dtype, (D, b))
        if Lq > Lk:
            assert bool((got[:, :Lq - Lk] == 0).all())


def test_window_attention_layouts_and_dense():
    q, k, v = (torch.randn(2, h, 900, 128, generator=torch.Generator().manual_seed(h)).to(BF).to(DEV) for h in (8, 2, 2))
    a = fa.window_attention(q, k, v, window=200, sinks=3)
    t = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    assert torch.equal(fa.window_attention(*t, window=200, sinks=3), a)
    out = torch.empty(2, 8, 900, 128, dtype=BF, device=DEV).transpose(1, 2)
    assert torch.equal(fa.window_attention(q, k, v, window=200, sinks=3, out=out), a)
    # repeated KV heads, as a broadcast view
    r = [x[:, :, None].expand(-1, -1, 4, -1, -1).reshape(2, 8, 900, 128) for x in (k, v)]
    wide = fa.window_attention(q, *r, window=200, sinks=3)
    assert (wide.float() - a.float()).abs().max() < 2.0 ** -6
    # no window: the causal attention of block_sparse_attention
    dense = fa.block_sparse_attention(q, k, v)
    assert (fa.window_attention(q, k, v, window=None).float() - dense.float()).abs().max() < 2.0 ** -6


# ---- rotary positions -------------------------------------------------------------

def _check_rot(got, x, pos, inv, factor, inter, dtype):
    want = ref.rotate(x, pos, inv, factor, inter)
    half = len(inv)
    big = x.double().abs().amax(-1, keepdim=True) * 2 * factor
    tol = _half_step(dtype) * want.abs() + 2.0 ** -20 * big + (2.0 ** -25 if dtype is F16 else 0.0)
    tol[..., 2 * half:] = 0
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), (err - tol).max().item()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (64, 64), (128, 32), (128, 34), (64, 2), (256, 256), (80, 40),
                                   (8, 6), (512, 256)])
@pytest.mark.parametrize("inter", [False, True])
def test_rope(dtype, D, rot, inter):
    g = torch.Generator().manual_seed(rot)
    T = 37
    q, k = (torch.randn(T, h, D, generator=g).to(dtype) for h in (5, 2))
    pos = torch.randint(0, 2 ** 20, (T,), generator=g)
    pos[:3] = torch.tensor([0, 1, 2 ** 31 - 1])
    inv, factor = fa.rope_frequencies(rot, base=500000.0, attention_factor=1.25, device="cpu")
    for p in (pos, pos.to(I32)):
        gq, gk = fa.rope(q.to(DEV), k.to(DEV), p.to(DEV), inv.to(DEV), attention_factor=factor, interleaved=inter)
        _check_rot(gq, q, pos, inv, factor, inter, dtype)
        _check_rot(gk, k, pos, inv, factor, inter, dtype)


@pytest.mark.parametrize("T", [1, 2047, 2048, 5001])
def test_rope_lengths_in_place_and_strided(T):
    g = torch.Generator().manual_seed(T)
    qkv = torch.randn(T, 7 * 128, generator=g).to(BF)
    pos = torch.arange(T) + 100000
    inv, _ = fa.rope_frequencies(128, device="cpu")
    dev = qkv.to(DEV)
    q, k = dev[:, :512].view(T, 4, 128), dev[:, 512:640].view(T, 1, 128)
    rq, rk = fa.rope(q, k, pos.to(DEV), inv.to(DEV))
    _check_rot(rq, qkv[:, :512].view(T, 4, 128), pos, inv, 1.0, False, BF)
    assert torch.equal(dev.cpu(), qkv)
    fa.rope(q, k, pos.to(DEV), inv.to(DEV), q_out=q, k_out=k)              # in place
    assert torch.equal(q, rq) and torch.equal(k, rk)
    assert torch.equal(dev[:, 640:].cpu(), qkv[:, 640:])


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("hnd", [False, True])
@pytest.mark.parametrize("inter", [False, True])
def test_rope_cache(dtype, hnd, inter):
    g = torch.Generator().manual_seed(3)
    T, Hq, Hk, D, pages, ps = 45, 4, 2, 128, 9, 16
    q, k, v = (torch.randn(T, h, D, generator=g).to(dtype) for h in (Hq, Hk, Hk))
    pos = torch.randint(0, 300000, (T,), generator=g).to(I32)
    slots = torch.randperm(pages * ps, generator=g)[:T]
    pos[7] = -1                                                            # a row behind the last request
    slots[9], slots[11], slots[12] = -1, pages * ps, 2 ** 40               # no place
    inv, f = fa.rope_frequencies(64, base=1e6, scaling="yarn", factor=4.0, original_length=4096, device="cpu")
    kc, vc = (torch.randn(*((pages, Hk, ps, D) if hnd else (pages, ps, Hk, D)), generator=g).to(dtype) for _ in range(2))
    gk, gv = (x.to(DEV).transpose(1, 2) if hnd else x.to(DEV) for x in (kc, vc))
    kc, vc = (x.transpose(1, 2).clone() if hnd else x.clone() for x in (kc, vc))
    q_out = torch.full((T, Hq, D), 7.0, dtype=dtype, device=DEV)
    got = fa.rope_cache(q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), slots.to(DEV), gk, gv, inv.to(DEV),
                        attention_factor=f, interleaved=inter, q_out=q_out)
    rows = torch.arange(T) != 7
    _check_rot(got[rows.to(DEV)], q[rows], pos[rows], inv, f, inter, dtype)
    assert bool((got[7] == 7.0).all())
    placed = rows & (slots >= 0) & (slots < pages * ps)
    at = (slots[placed] // ps, slots[placed] % ps)
    _check_rot(gk.cpu()[at], k[placed], pos[placed], inv, f, inter, dtype)
    vc[at] = v[placed]
    assert torch.equal(gv.cpu(), vc)
    kc[at] = gk.cpu()[at]
    assert torch.equal(gk.cpu(), kc)                                       # no other slot is touched


# ---- block tables and slot maps -----------------------------------------------------

def _plan_case(B, P, F, ps, seed, grow=40, lack=False):
    """Random requests over a cache of F pages: some grow, shrink, finish or stand still."""
    g = torch.Generator().manual_seed(seed)
    rnd = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))     # noqa: E731
    perm = torch.randperm(F, generator=g).tolist()
    table, lens, new = [], [], []
    for b in range(B):
        want = rnd(0, max(2, min(P, 1 + len(perm) // 2) * ps)) if rnd(0, 4) else 0
        n = min(-(-want // ps), len(perm))
        want = min(want, n * ps)
        table.append([perm.pop() for _ in range(n)] + [-1] * (P - n))
        lens.append(want)
        kind = rnd(0, 5)
        new.append([rnd(0, grow), 1, 0, -rnd(0, want + 1), -want][kind])
    free = perm + [0] * (F - len(perm))
    return table, lens, new, free, (len(perm) // 8 if lack else len(perm))


def _check_plan(case, ps, T, wide=False):
    table, lens, new, free, count = case
    want = ref.plan(table, lens, new, free, count, ps, T)
    t = _i32(table)
    if wide:                                                               # rows of a wider table
        w = torch.full((len(table), len(table[0]) + 5), -9, dtype=I32, device=DEV)
        w[:, 2:2 + len(table[0])] = t
        t = w[:, 2:2 + len(table[0])]
    f, lens_d, count_d = _i32(free), _i32(lens), _i32([count])
    p = None
    for _ in range(2):                                                     # repeated: the same result
        p = fa.plan_step(t, lens_d, _i32(new), f, count_d, page_size=ps, num_tokens=T, out=p)
        got = dict(block_table=t, free_pages=f, cu_lens=p.cu_lens, seq_lens=p.seq_lens, positions=p.positions,
                   slots=p.slots, free_count=p.free_count, lacking=p.lacking)
        for name, w in want.items():
            assert got[name].tolist() == w, name
    assert lens_d.tolist() == lens and count_d.tolist() == [count]
    return p


@pytest.mark.parametrize("B,P,F,ps", [(1, 4, 8, 16), (7, 9, 60, 16), (64, 20, 900, 1), (513, 6, 2000, 64), (4096, 5, 9000, 3)])
@pytest.mark.parametrize("seed", [0, 1])
def test_plan_step(B, P, F, ps, seed):
    case = _plan_case(B, P, F, ps, seed)
    total = sum(max(n, 0) for n in case[2])
    _check_plan(case, ps, total + 13, wide=bool(seed))
    _check_plan(case, ps, max(total - 5, 0))                               # fewer rows than tokens: the first ones


@pytest.mark.parametrize("seed", [0, 1, 2])
def test_plan_step_without_enough_pages(seed):
    case = _plan_case(40, 6, 100, 16, seed, grow=90, lack=True)
    p = _check_plan(case, 16, sum(max(n, 0) for n in case[2]))
    assert int(p.lacking) > 0


def test_plan_step_many_tokens_and_releases():
    P, ps = 700, 16
    table = [list(range(b * P, b * P + P)) for b in range(4)] + [[-1] * P for _ in range(3)]
    lens, new = [P * ps] * 4 + [0, 0, 0], [-P * ps, -1, -17, 0, 9000, 8999, 1]
    free = [0] * (4 * P)
    _check_plan((table, lens, new, free, 0), ps, 18005)


def test_plan_step_takes_lengths_at_the_border():
    _check_plan(([[0, 1], [2, -1]], [1000, -5], [7, 3], [3, 4, 5, 6], 99), 16, 12)
    _check_plan(([[0, 1], [2, -1]], [20, 3], [5, -2 ** 31], [3, 4, 5, 6], -1), 16, 9)


def test_plan_step_refuses_outputs_that_are_inputs():
    t, lens, new, free, count = _i32([[0, 1]]), _i32([3]), _i32([1]), _i32([1, 0]), _i32([1])
    p = fa.plan_step(t, lens, new, free, count, page_size=16, num_tokens=1)
    for bad in (dict(seq_lens=lens), dict(free_count=count)):
        o = fa.StepPlan(**{**vars(p), **bad})
        with pytest.raises(ValueError, match="shares storage"):
            fa.plan_step(t, lens, new, free, count, page_size=16, num_tokens=1, out=o)


# ---- together ---------------------------------------------------------------------------

class Server:
    """A small serving loop: what it holds on the GPU, and the same requests' keys and values on the CPU."""

    def __init__(self, B=5, Hq=8, Hk=2, D=128, ps=16, pages=80, dtype=BF, seed=0):
        self.Hq, self.Hk, self.D, self.ps, self.dtype = Hq, Hk, D, ps, dtype
        self.g = torch.Generator().manual_seed(seed)
        self.table = torch.full((B, 24), -1, dtype=I32, device=DEV)
        self.lens, self.count = _i32([0] * B), _i32([pages])
        self.free = torch.arange(pages, dtype=I32, device=DEV)
        self.kc, self.vc = (torch.full((pages, ps, Hk, D), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
        self.inv, self.factor = fa.rope_frequencies(D, base=500000.0, scaling="llama3", factor=8.0, original_length=64)
        self.k = [torch.zeros(0, Hk, D, dtype=torch.float64) for _ in range(B)]
        self.v = [torch.zeros(0, Hk, D, dtype=torch.float64) for _ in range(B)]

    def tokens(self, T):
        return [torch.randn(T, h, self.D, generator=self.g).to(self.dtype) for h in (self.Hq, self.Hk, self.Hk)]

    def launch(self, new, q, k, v, window, sinks, plan=None, out=None, q_out=None):
        plan = fa.plan_step(self.table, self.lens, new, self.free, self.count, page_size=self.ps, num_tokens=len(q), out=plan)
        r = fa.rope_cache(q, k, v, plan.positions, plan.slots, self.kc, self.vc, self.inv,
                          attention_factor=self.factor, q_out=q_out)
        out = fa.paged_attention(r, self.kc, self.vc, self.table, plan.cu_lens, plan.seq_lens, window=window,
                                 sinks=sinks, out=out)
        return plan, out

    def expect(self, new, q, k, v, window, sinks):
        row, want = 0, []
        for b, n in enumerate(new):
            if n <= 0:
                keep = max(len(self.k[b]) + n, 0)
                self.k[b], self.v[b] = self.k[b][:keep], self.v[b][:keep]
                continue
            first = len(self.k[b])
            pos = torch.arange(first, first + n)
            x = slice(row, row + n)
            rot = lambda t: ref.rotate(t[x], pos, self.inv.cpu(), self.factor).to(self.dtype)   # noqa: E731
            self.k[b] = torch.cat([self.k[b], rot(k).double()])
            self.v[b] = torch.cat([self.v[b], v[x].double()])
            want.append(ref.attend(rot(q), self.k[b], self.v[b], first, window, sinks))
            row += n
        return torch.cat([w for w, _ in want]), torch.cat([m for _, m in want]), row

    def check(self, got, want, mag, rows):
        # q and k are rounded to bf16 from 32-bit rotations that may fall on the other side of a tie: one more step of
        # 2^-7 of a few elements, which moves a score by up to 2^-7 * |q| |k| / sqrt(D) of single products (about 0.02)
        u = _half_step(self.dtype)
        err = (got[:rows].double().cpu() - want).abs()
        assert bool((err <= (3 * u + 0.02) * mag).all()), (err / mag).max().item()


STEPS = [[17, 0, 40, 1, 0], [1, 1, 1, 1, 1], [30, 5, 1, -1, 64], [1, -6, 1, -100, 1], [0, 8, -20, 33, 1], [1, 1, 1, 1, 1]]


@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 3)])
def test_a_serving_loop(window, sinks):
    s = Server()
    for new in STEPS:
        q, k, v = s.tokens(sum(max(n, 0) for n in new) + 3)
        plan, got = s.launch(_i32(new), *(x.to(DEV) for x in (q, k, v)), window, sinks)
        s.check(got, *s.expect(new, q, k, v, window, sinks))
        assert int(plan.lacking) == 0
        s.lens, s.count = plan.seq_lens, plan.free_count
        assert s.lens.tolist() == [len(x) for x in s.k]
        assert int(s.count) == 80 - sum(-(-len(x) // s.ps) for x in s.k)


def test_a_captured_step():
    """One step captured with its buffers, replayed with other lengths, eager work and synchronizations between."""
    s = Server(seed=1)
    T = 110
    q, k, v = (torch.zeros(T, h, s.D, dtype=BF, device=DEV) for h in (s.Hq, s.Hk, s.Hk))
    new, out, q_out = _i32([0] * 5), torch.zeros(T, s.Hq, s.D, dtype=BF, device=DEV), torch.zeros(T, s.Hq, s.D, dtype=BF, device=DEV)
    plan, _ = s.launch(new, q, k, v, 30, 2, out=out, q_out=q_out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.launch(new, q, k, v, 30, 2, plan, out, q_out)
        s.lens.copy_(plan.seq_lens)
        s.count.copy_(plan.free_count)
    for step in STEPS:
        n = sum(max(x, 0) for x in step)
        cq, ck, cv = s.tokens(n)
        q[:n], k[:n], v[:n] = cq.to(DEV), ck.to(DEV), cv.to(DEV)
        new.copy_(torch.tensor(step, dtype=I32))
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.full_like(out, 7.0)
        fa.paged_attention(q_out, s.kc, s.vc, s.table, plan.cu_lens, plan.seq_lens, window=30, sinks=2, out=eager)
        assert torch.equal(out, eager)
        s.check(out, *s.expect(step, cq, ck, cv, 30, 2))
        assert bool((out[n:] == 7.0).all())


def test_two_calls_at_once_on_streams():
    """Each call has its own workspace: two streams at once give what one gives."""
    b = [Batch([(3000, 1), (500, 1)], ps=64, seed=20), Batch([(200, 150), (10, 3)], seed=21)]
    want = [x.gpu() for x in b]
    streams = [torch.cuda.Stream() for _ in b]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (x, st) in enumerate(zip(b, streams)):
            with torch.cuda.stream(st):
                got[i].append(x.gpu())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
