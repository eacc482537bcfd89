"""Pages in 8 bits (e4m3, a scale for each KV head) on the GPU: written by rope_cache, read by paged_attention.

Tolerances.  Written: one rounding to e4m3, at most half a step there; before it, in 32 bits, the angle's cosine and sine
(2 units in the last place), two products, a sum, the scale's reciprocal and a product: 2^-20 of the pair's
magnitude, which also decides which way a value next to a border is rounded.  Read: an e4m3 number is one of bf16 and of
f16, so nothing is added to what ``test_gpu_serving`` counts for 16-bit caches but the scales' products in 32 bits.
"""
from __future__ import annotations

import pytest
import torch

import fftsparse_amd as fa
from oracle import paged as ref
from oracle import tree as ref8
from tests.test_gpu_tree import BF, DEV, E4M3, F16, F32, I32, Batch, _i32

pytestmark = pytest.mark.gpu

DECODE = [(0, 1), (5, 1), (62, 1), (63, 1), (64, 1), (999, 1), (0, 0), (129, 1), (30, 0)]
CHUNKS = [(0, 1), (0, 17), (100, 33), (1000, 130), (0, 0), (3, 257), (64, 64)]
FEW = [(2500, 3), (900, 8)]
WINDOWS = [(None, 0), (1, 0), (1, 3), (16, 4), (100, 0), (64, 70), (130, 200), (5000, 3)]


class Chain(Batch):
    """Chains of new tokens over 8-bit pages."""

    def __init__(self, lens, **kw):
        super().__init__(lens, kind="chain", bits=8, **kw)

    def gpu(self, **kw):
        return fa.paged_attention(kw.pop("q", self.q.to(DEV)), *self.dev_caches(), self.table.to(DEV), _i32(self.cu),
                                  _i32(self.total), k_scale=self.ks.to(DEV), v_scale=self.vs.to(DEV), **kw)

    def check(self, got, window=None, sinks=0, scale=None, note=""):
        u = torch.finfo(self.dtype).eps / 2
        for b, (c, n) in enumerate(self.lens):
            if not n:
                continue
            rows = slice(self.cu[b], self.cu[b + 1])
            want, mag = ref.attend(self.q[rows], self.k[b], self.v[b], c, window, sinks, scale)
            tol = (3 * u + 2e-4) * mag + 1e-30
            if self.dtype is F16:
                tol = tol + (c + n) * 2.0 ** -25 * 8.0 + 2.0 ** -25
            x = got[rows].double().cpu()
            err = (x - want).abs()
            assert bool(torch.isfinite(x).all()), (b, note)
            assert bool((err <= tol).all()), (b, note, (err / tol).max().item(), err.max().item())


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("lens", [DECODE, CHUNKS, FEW], ids=["decode", "chunks", "few"])
def test_attention_windows(lens, window, sinks):
    b = Chain(lens, ps=16, seed=1)
    b.check(b.gpu(window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (8, 1), (7, 1), (6, 2), (28, 4), (33, 1)])
@pytest.mark.parametrize("ps", [16, 48, 64, 256])
def test_attention_heads_pages_types(dtype, D, Hq, Hk, ps):
    b = Chain([(0, 1), (77, 1), (0, 5), (300, 40), (450, 1)], Hq=Hq, Hk=Hk, D=D, ps=ps, dtype=dtype, hnd=ps == 48, seed=ps)
    b.check(b.gpu())
    b.check(b.gpu(window=50, sinks=2), 50, 2)


@pytest.mark.parametrize("max_new", [None, 1, 2, 40, 1000])
@pytest.mark.parametrize("lens", [DECODE, CHUNKS], ids=["decode", "chunks"])
def test_attention_is_right_for_any_max_new(lens, max_new):
    b = Chain(lens, seed=5)
    b.check(b.gpu(max_new=max_new))


@pytest.mark.parametrize("max_new", [None, 1])
def test_attention_many_requests(max_new):
    lens = [((7 * i) % 45, 1 if i % 5 else 0) for i in range(700)] + [(3000, 1)]
    b = Chain(lens, Hq=4, Hk=1, D=64, seed=2)
    b.check(b.gpu(max_new=max_new))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,max_new", [([(20000, 1)], 1), ([(9000, 20)], None), ([(6000, 100), (40, 1)], None)])
def test_attention_long(lens, max_new, D):
    b = Chain(lens, ps=64, D=D, seed=3)
    b.check(b.gpu(max_new=max_new))
    b.check(b.gpu(max_new=max_new, window=4000, sinks=10), 4000, 10)


@pytest.mark.parametrize("scale", [0.0, 1e-4, 0.3])
def test_attention_scales_of_zero_and_near(scale):
    for lens in (DECODE, CHUNKS):
        b = Chain(lens, seed=24)
        b.check(b.gpu(softmax_scale=scale), scale=scale)


@pytest.mark.parametrize("lens", [DECODE, CHUNKS], ids=["decode", "chunks"])
def test_attention_is_that_of_the_numbers_the_pages_stand_for(lens):
    """Scales that are powers of two: a 16-bit cache of the same numbers gives the result within the rounding's bound (both
    within 3 u of the weighted |v|), scales from 2^-20 to 2^20 on values included."""
    for shift in (-20, 0, 20):
        b = Chain(lens, seed=25)
        b.ks.fill_(2.0 ** -6)
        b.vs.fill_(2.0 ** shift)
        x = b.gpu()
        kc, vc = b.dev_caches()
        y = fa.paged_attention(b.q.to(DEV), (kc.float() * 2.0 ** -6).to(BF), (vc.float() * 2.0 ** shift).to(BF),
                               b.table.to(DEV), _i32(b.cu), _i32(b.total))
        rows = x[:b.T].double() - y[:b.T].double()
        u = torch.finfo(BF).eps / 2
        assert bool((rows.abs() <= 2 * (3 * u + 2e-4) * 448 * 2.0 ** shift).all())
        assert (rows.norm() / y[:b.T].double().norm()).item() <= 2 * (3 * u + 2e-4)


def test_attention_all_numbers():
    """Every finite e4m3 number as a key's and a value's element: one request that sees one token returns it, over the scale's
    product, rounded once."""
    codes = torch.tensor([c for c in range(256) if c & 127 != 127], dtype=torch.uint8)
    for dtype in (BF, F16):
        kc = torch.zeros(2, 16, 1, 128, dtype=torch.uint8)
        kc[0, 0, 0], kc[1, 0, 0] = codes[:128], torch.cat([codes[128:], codes[:2]])
        vc = kc.clone()
        s = torch.tensor([0.37], device=DEV)
        got = fa.paged_attention(torch.zeros(2, 1, 128, dtype=dtype, device=DEV), kc.to(DEV).view(E4M3), vc.to(DEV).view(E4M3),
                                 _i32([[0], [1]]), _i32([0, 1, 2]), _i32([1, 1]), k_scale=s, v_scale=s)
        want = vc.view(E4M3)[:, 0].double() * s.double().cpu()
        assert bool(((got.double().cpu() - want).abs() <= want.abs() * (torch.finfo(dtype).eps / 2 + 2.0 ** -22) + 2.0 ** -25).all())


def test_rows_behind_the_last_request_stay():
    for lens in (DECODE, CHUNKS):
        b = Chain(lens, pad=37, seed=6)
        out = torch.full(b.q.shape, 7.0, dtype=BF, device=DEV)
        got = b.gpu(out=out, max_new=1 if lens is DECODE else None)
        b.check(got)
        assert bool((got[b.T:] == 7.0).all())


def test_a_captured_step_replays():
    for lens in (DECODE, CHUNKS):
        b = Chain(lens, seed=26)
        q, (kc, vc), table, cu, total = b.q.to(DEV), b.dev_caches(), b.table.to(DEV), _i32(b.cu), _i32(b.total)
        ks, vs = b.ks.to(DEV), b.vs.to(DEV)
        run = lambda: fa.paged_attention(q, kc, vc, table, cu, total, k_scale=ks, v_scale=vs)   # noqa: E731
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x = run()
        for i in range(4):
            vs.mul_(0.5 + i)
            q.mul_(0.9)
            g.replay()
            want = run()
            torch.cuda.synchronize()
            assert torch.equal(x[:b.T], want[:b.T])


# ---- writing -------------------------------------------------------------------------------

def _write(T, Hq, Hk, D, rot, inter, dtype, ps=16, hnd=False, seed=0, scales=None, scale_in=None):
    """rope_cache into 8-bit pages and what it has to leave: (cache numbers, exact x / scale, rows written, q, q exact)."""
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(T, h, D, generator=g).to(dtype) for h in (Hq, Hk, Hk))
    if scale_in is not None:
        k, v = (x * scale_in for x in (k, v))
    pages = -(-T // ps) + 4
    slots = torch.randperm(pages * ps, generator=g)[:T].to(torch.int64)
    pos = torch.randint(0, 100000, (T,), generator=g).to(I32)
    inv, _ = fa.rope_frequencies(rot, base=500000.0, device="cpu")
    ks, vs = (0.005 + 0.02 * torch.rand(Hk, generator=g) for _ in range(2)) if scales is None else scales
    shape = (pages, Hk, ps, D) if hnd else (pages, ps, Hk, D)
    caches = [torch.full(shape, 0x2a, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2)]
    if hnd:
        caches = [c.transpose(1, 2) for c in caches]
    qo = fa.rope_cache(q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), slots.to(DEV), *caches, inv.to(DEV), interleaved=inter,
                       k_scale=ks.to(DEV), v_scale=vs.to(DEV))
    return dict(q=q, k=k, v=v, pos=pos, inv=inv, slots=slots, caches=caches, ks=ks, vs=vs, qo=qo, ps=ps, pages=pages)


def _rotated(x, w, inter):
    """Exact rotation of x, and the magnitude of the pair that each element comes from."""
    half, pair = len(w["inv"]), x.double().abs()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if inter else (slice(0, half), slice(half, 2 * half))
    m = torch.hypot(pair[..., a], pair[..., b])
    pair[..., a], pair[..., b] = m, m
    return ref.rotate(x, w["pos"], w["inv"], 1.0, inter), pair


def _check_written(w, inter):
    for cache, x, s, turned in ((w["caches"][0], w["k"], w["ks"], True), (w["caches"][1], w["v"], w["vs"], False)):
        y, pair = _rotated(x, w, inter) if turned else (x.double(), x.double().abs())
        y, pair = (z / s.double()[:, None] for z in (y, pair))
        got = cache.float().cpu().double()
        rows = got[w["slots"] // w["ps"], w["slots"] % w["ps"]]
        c = y.clamp(-448.0, 448.0)
        tol = ref8.e4m3_half_step(c) + pair * 2.0 ** -20
        assert bool(((rows - c).abs() <= tol).all()), ((rows - c).abs() / tol).max().item()
        flat = cache.contiguous().view(torch.uint8).cpu().reshape(w["pages"] * w["ps"], -1)
        other = torch.ones(len(flat), dtype=torch.bool)
        other[w["slots"]] = False
        assert bool((flat[other] == 0x2a).all())


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (64, 64), (64, 34), (80, 20), (16, 2), (256, 256)])
@pytest.mark.parametrize("T", [1, 7, 1500])
def test_rope_cache_into_8_bits(T, D, rot, dtype, inter):
    w = _write(T, 3, 2, D, rot, inter, dtype, hnd=T == 7, seed=T + D)
    _check_written(w, inter)
    # q as from rope, but not bit for bit: f16 results are rounded from the sum itself there and from its 32 bits here.  Both are
    # within half a step of the type, and 2^-20 of the pair's magnitude, of the exact value.
    y, pair = _rotated(w["q"], w, inter)
    tol = y.abs() * (torch.finfo(dtype).eps / 2) + pair * 2.0 ** -20 + (2.0 ** -25 if dtype is F16 else 0.0)
    assert bool(((w["qo"].double().cpu() - y).abs() <= tol).all())


def test_values_past_the_range_are_held_to_it():
    w = _write(40, 2, 2, 64, 64, False, BF, scale_in=200.0, seed=3)
    _check_written(w, False)
    assert w["caches"][1].float().abs().max().item() == 448.0


def test_small_values_and_nan_and_infinities():
    w = _write(40, 2, 2, 64, 64, False, F32, scale_in=2.0 ** -14, seed=4)
    _check_written(w, False)
    inf = float("inf")
    v = torch.tensor([float("nan"), inf, -inf, 0.0, -0.0, 448.0, 449.0, 464.0, 1e-9, -1e-9] + [1.0] * 6).view(1, 1, 16)
    kc, vc = (torch.zeros(1, 16, 1, 16, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2))
    one = torch.ones(1, device=DEV)
    fa.rope_cache(torch.zeros(1, 1, 16, device=DEV), torch.zeros(1, 1, 16, device=DEV), v.to(DEV), _i32([0]),
                  torch.zeros(1, dtype=torch.int64, device=DEV), kc, vc, torch.ones(8, dtype=torch.float64, device=DEV),
                  k_scale=one, v_scale=one)
    got = vc.float().cpu()[0, 0, 0]
    assert bool(got[0].isnan())
    assert got[1:].tolist() == [448.0, -448.0, 0.0, 0.0, 448.0, 448.0, 448.0, 0.0, 0.0] + [1.0] * 6


def test_ties_go_to_even():
    """Halfway between two e4m3 numbers, scale 1."""
    x = torch.tensor([1.0625, 1.1875, 1.3125, -1.0625, 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10, 5 * 2.0 ** -10, 432.0, 0.0, 0.0,
                      0.0, 0.0, 0.0, 0.0])
    kc, vc = (torch.zeros(1, 16, 1, 16, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2))
    one = torch.ones(1, device=DEV)
    z = torch.zeros(1, 1, 16, device=DEV)
    fa.rope_cache(z, z, x.view(1, 1, 16).to(DEV), _i32([0]), torch.zeros(1, dtype=torch.int64, device=DEV), kc, vc,
                  torch.ones(8, dtype=torch.float64, device=DEV), k_scale=one, v_scale=one)
    assert vc.float().cpu()[0, 0, 0].tolist() == [1.0, 1.25, 1.25, -1.0, 16.0, 20.0, 0.0, 2.0 ** -8, 2.0 ** -8,
                                                  448.0] + [0.0] * 6


def test_rows_without_a_place():
    """Slots outside the cache and rows with a negative position are not written."""
    T, D = 9, 64
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(T, h, D, generator=g).to(BF).to(DEV) for h in (2, 1, 1))
    slots = torch.tensor([0, -1, 32, 5, 10 ** 12, 31, 7, -(2 ** 62), 8], device=DEV)
    pos = _i32([1, 2, 3, -1, 5, 6, -7, 8, 9])
    kc, vc = (torch.full((2, 16, 1, D), 0x2a, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2))
    one = torch.full((1,), 0.01, device=DEV)
    fa.rope_cache(q, k, v, pos, slots, kc, vc, torch.ones(32, dtype=torch.float64, device=DEV), k_scale=one, v_scale=one)
    for c in (kc, vc):
        rows = c.view(torch.uint8).view(32, D).cpu()
        written = (rows != 0x2a).any(-1).nonzero()[:, 0].tolist()
        assert written == [0, 8, 31]


def test_writing_then_reading():
    """What one step writes the next reads, against attention over the unrounded keys and values: e4m3's half step, 2^-4, on
    values (averaged over the tokens) and on scores."""
    T, Hq, Hk, D, ps = 300, 8, 2, 128, 16
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(T, h, D, generator=g).to(BF).to(DEV) for h in (Hq, Hk, Hk))
    inv, _ = fa.rope_frequencies(D, device=DEV)
    pos = torch.arange(T, dtype=I32, device=DEV)
    pages = -(-T // ps)
    table = torch.randperm(pages, generator=g).to(I32).to(DEV)
    slots = table[(pos // ps).long()].long() * ps + pos % ps
    s = torch.full((Hk,), 0.02, device=DEV)
    c8 = [torch.zeros(pages, ps, Hk, D, device=DEV).to(E4M3) for _ in range(2)]
    c16 = [torch.zeros(pages, ps, Hk, D, dtype=BF, device=DEV) for _ in range(2)]
    q8 = fa.rope_cache(q, k, v, pos, slots, *c8, inv, k_scale=s, v_scale=s)
    q16 = fa.rope_cache(q, k, v, pos, slots, *c16, inv)
    assert bool(((q8.double() - q16.double()).abs() <= q16.double().abs() * torch.finfo(BF).eps + 1e-5).all())
    args = table[None].contiguous(), _i32([0, T]), _i32([T])
    x = fa.paged_attention(q8, *c8, *args, k_scale=s, v_scale=s).double()
    y = fa.paged_attention(q16, *c16, *args).double()
    assert ((x - y).norm() / y.norm()).item() <= 2.0 ** -4 * 1.5
