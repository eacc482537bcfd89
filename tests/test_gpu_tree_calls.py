"""Calls of the tree operators on the GPU that the documentation allows beside the usual ones, and some that it refuses."""
from __future__ import annotations

import pytest
import torch

import fftsparse_amd as fa
from oracle import tree as ref
from tests.test_gpu_tree import BF, DEV, E4M3, I32, Batch, _i32, _moved

pytestmark = pytest.mark.gpu

LAYERS, PAGES, PS, HK, D = 3, 5, 16, 2, 64
TABLE = [[3, 0, -1], [4, 1, 2]]
CU, LENS, KEPT = [0, 12, 32], [30, 40], [0, 2, 3, 7, 11, *[-1] * 7, 0, 1, 4, 9, 10, 18, 19, *[-1] * 13]


def _views(form, dtype):
    """One storage and the layers' keys and values in it, [PAGES, PS, HK, D] each."""
    n = 2 * LAYERS * PAGES * PS * HK * D * torch.empty(0, dtype=dtype).element_size()
    raw = torch.randint(0, 256, (n,), generator=torch.Generator().manual_seed(1), dtype=torch.uint8).to(DEV)
    x = raw.view(dtype)
    if form == "pages hold all layers":
        x = x.view(PAGES, LAYERS, 2, PS, HK, D)
        return raw, [x[:, i, 0] for i in range(LAYERS)], [x[:, i, 1] for i in range(LAYERS)]
    if form == "tokens hold all layers":
        x = x.view(PAGES, PS, LAYERS, 2, HK, D)
        return raw, [x[:, :, i, 0] for i in range(LAYERS)], [x[:, :, i, 1] for i in range(LAYERS)]
    if form == "pages hold all layers, tokens keys and values":
        x = x.view(PAGES, LAYERS, PS, 2, HK, D)
        return raw, [x[:, i, :, 0] for i in range(LAYERS)], [x[:, i, :, 1] for i in range(LAYERS)]
    if form == "tokens hold keys and values":
        x = x.view(LAYERS, PAGES, PS, 2, HK, D)
        return raw, x[:, :, :, 0], x[:, :, :, 1]
    if form == "heads hold keys and values":
        x = x.view(LAYERS, PAGES, PS, HK, 2, D)
        return raw, [*x[..., 0, :]], [*x[..., 1, :]]
    if form == "values by heads":                          # of each page, behind the keys by tokens
        x = x.view(LAYERS, PAGES, 2, PS * HK * D)
        return (raw, [*x[:, :, 0].view(LAYERS, PAGES, PS, HK, D)],
                [*x[:, :, 1].view(LAYERS, PAGES, HK, PS, D).transpose(2, 3)])
    x = x.view(2 * LAYERS, PAGES, PS, HK, D)               # keys and values in turn
    return raw, [*x[::2]], [*x[1::2]]


@pytest.mark.parametrize("dtype", [BF, E4M3])
@pytest.mark.parametrize("form", ["pages hold all layers", "tokens hold keys and values", "heads hold keys and values",
                                  "values by heads", "in turn", "tokens hold all layers",
                                  "pages hold all layers, tokens keys and values"])
def test_move_kept_in_caches_of_one_storage(form, dtype):
    """Caches that lie between each other's rows are apart: each is moved as if it were alone."""
    raw, k, v = _views(form, dtype)
    before = [[t.view(torch.uint8).cpu()[None] if t.is_contiguous() else t.contiguous().view(torch.uint8).cpu()[None] for t in c]
              for c in (k, v)]
    table = torch.tensor(TABLE, dtype=I32)
    fa.move_kept(k, v, table.to(DEV), _i32(CU), _i32(LENS), _i32(KEPT))
    for c, old in zip((k, v), before):
        for t, x in zip(c, old):
            assert torch.equal(t.contiguous().view(torch.uint8).cpu()[None], _moved(x, table, CU, LENS, KEPT, PS))


def test_move_kept_refuses_caches_that_share_storage():
    """A cache that is named twice, in whatever form: refused, and nothing is moved."""
    table = torch.tensor(TABLE, dtype=I32).to(DEV)
    raw, k, v = _views("in turn", BF)
    before = raw.clone()
    whole = raw.view(BF).view(2 * LAYERS, PAGES, PS, HK, D)
    for a, b in [([k[0], k[0]], v[:2]), (k[:2], [v[1], v[1]]), ([k[0], k[1], k[0]], [v[0], v[1], v[0]]), (k, k), (k[0], k[0]),
                 (whole[:3], whole[2:5]), (whole[:3], whole[:3]), (whole[0], whole.view(-1, PS, HK, D)[2:7]),
                 ([k[0]], [k[0].view(PAGES, HK, PS, D).transpose(1, 2)])]:
        with pytest.raises(ValueError, match="share storage"):
            fa.move_kept(a, b, table, _i32(CU), _i32(LENS), _i32(KEPT))
    torch.cuda.synchronize()
    assert torch.equal(raw, before)


@pytest.mark.parametrize("first,last", [(0, 6), (2, 6), (3, 5), (5, 6), (0, 1)])
def test_requests_of_the_middle_of_a_batch(first, last):
    """Row numbers that begin behind the first rows and end before the last ones: rows of no request have position -1, no bit
    and nothing kept, and attention leaves them as they were."""
    b = Batch([(5, 8), (62, 3), (0, 70), (64, 1), (99, 8), (30, 4)], kind="random", seed=3)
    parents = [p for t in b.trees for p in t]
    cu, lens = _i32(b.cu)[first:last + 1], _i32(b.total)[first:last]
    rows = slice(b.cu[first], b.cu[last])
    out = fa.TreePlan(torch.full((b.T,), 7, dtype=I32, device=DEV), torch.full((b.T, 2), 7, dtype=torch.int64, device=DEV))
    fa.plan_tree(_i32(parents), cu, lens, max_new=70, out=out)
    pos, mask = [-1] * b.T, torch.zeros(b.T, 2, dtype=torch.int64)
    pos[rows], mask[rows] = b.pos[rows], b.mask[rows]
    assert out.positions.tolist() == pos and torch.equal(out.mask.cpu(), mask)
    tokens = torch.ones(b.T, dtype=I32, device=DEV)
    want = ref.accept(parents, [1] * b.T, [1] * b.T, b.cu, 70)
    acc = fa.Accepted(torch.full((b.T,), 7, dtype=I32, device=DEV), *(torch.full((last - first,), 7, dtype=I32, device=DEV) for _ in range(3)))
    fa.accept_tree(_i32(parents), tokens, tokens, cu, max_new=70, out=acc)
    kept = [-1] * b.T
    kept[rows] = want[0][rows]
    assert acc.kept.tolist() == kept and acc.kept_lens.tolist() == want[1][first:last]
    got = torch.full(b.q.shape, 7.0, dtype=BF, device=DEV)
    fa.tree_attention(b.q.to(DEV), *b.dev_caches(), b.table.to(DEV)[first:last], cu, lens, out.mask, out=got)
    assert bool((got[:rows.start] == 7.0).all()) and bool((got[rows.stop:] == 7.0).all())
    got[:rows.start], got[rows.stop:] = (b.gpu()[x] for x in (slice(0, rows.start), slice(rows.stop, None)))
    b.check(got)


@pytest.mark.parametrize("scale", [2.0 ** -126, 1.5 * 2.0 ** -126, 2.0 ** -60, 2.0 ** 60, 1.75 * 2.0 ** 125, 2.0 ** 126])
def test_scales_at_the_ends_of_their_range(scale):
    """x / scale in e4m3, exact where the scale is a power of two, else within half a step and the quotient's 2^-22; attention
    reads the numbers times the scale (results below 2^-126 in steps of 2^-133)."""
    T, D = 20, 64
    g = torch.Generator().manual_seed(6)
    v = (torch.randn(T, 1, D, generator=g).double() * 1.9 * scale).float().clamp(-3e38, 3e38)
    kc, vc = (torch.zeros(2, 16, 1, D, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2))
    one, s = torch.ones(1, device=DEV), torch.tensor([scale], device=DEV)
    pos, zero = torch.arange(T, dtype=I32, device=DEV), torch.zeros(T, 1, D, device=DEV)
    fa.rope_cache(zero, zero, v.to(DEV), pos, pos.long(), kc, vc, torch.ones(32, dtype=torch.float64, device=DEV),
                  k_scale=one, v_scale=s)
    y, got = v[:, 0].double() / scale, vc.view(32, D)[:T].cpu().float().double()
    assert bool(((got - y).abs() <= ref.e4m3_half_step(y) + y.abs() * 2.0 ** -22).all())
    if scale == 2.0 ** torch.tensor(scale).log2().round().item():
        assert torch.equal(got, y.float().to(E4M3).double())
    if scale > 2.0 ** 84:                                  # attention takes values up to 2^93
        return
    # every key alike: the mean of the values up to each token, in 32 bits but for the weights and the result (bf16)
    q = torch.ones(T, 1, D, dtype=BF, device=DEV)
    out = fa.paged_attention(q, kc, vc, _i32([[0, 1]]), _i32([0, T]), _i32([T]), k_scale=one, v_scale=s).double().cpu()[:, 0]
    want = (got.cumsum(0) / torch.arange(1, T + 1)[:, None]) * scale
    mag = (got.abs().cumsum(0) / torch.arange(1, T + 1)[:, None]) * scale
    assert bool(((out - want).abs() <= 3 * 2.0 ** -8 * mag + 2.0 ** -133).all())
