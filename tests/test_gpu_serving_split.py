"""Attention whose keys are cut into pieces that are joined afterwards, on the GPU against 64 bits.

Whether a call cuts its keys follows from a cost rule in the library, so each test reads from the call's own workspace
that it did: its first four integers are the pieces of a KV head, the row tiles that were cut, the key tiles of a
piece and the pieces of cut row tiles.  The workspace has the size that is asked for, and what stands behind it has to stay.

Inputs.  Queries are three times normal numbers, so a few keys of each row, in any of its pieces, hold most of its weight
and the result is as large as the values: a piece lost, joined twice or with a wrong maximum shows.

Tolerance, u = eps / 2 of the type.  Weights are rounded to the type (u, and again u through the row sum, which adds
the rounded ones) and the result once: 3 u times the softmax average of |v|.  A score is D products added in 32 bits, each
addition off by at most 2^-23 of the sum of their magnitudes, then scaled, and its exponential taken (a few 2^-23 more):
d = (D + 8) 2^-23 max sum |q k| scale changes numerator and denominator by d each.  Sums over the keys in 32 bits: keys
2^-24.  f16 holds weights, 2^7 times as large, down to steps of 2^-24: keys 2^-32 max |v|, and results in steps of 2^-24."""
from __future__ import annotations

import ctypes

import pytest
import torch

import fftsparse_amd as fa
from fftsparse_amd import _lib
from tests.test_gpu_serving import Batch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, F16 = torch.bfloat16, torch.float16


@pytest.fixture
def cuts(monkeypatch):
    """Row tiles that each attention call cut (-1: the call made no plan of pieces)."""
    seen, launch = [], _lib.call

    def call(name, args, device=None):
        if name not in ("fs_paged_attn", "fs_window_attn"):
            return launch(name, args, device)
        n = getattr(_lib.load(), name + "_work_bytes")(ctypes.byref(args))
        work = torch.full((n + 65536,), 0xA5, dtype=torch.uint8, device=DEV)
        args.work = work.data_ptr()
        launch(name, args, device)
        head = work[:16].view(torch.int32).tolist()
        seen.append(-1 if head == [-0x5A5A5A5B] * 4 else head[1])
        assert bool((work[n:] == 0xA5).all()), "written behind the workspace"

    monkeypatch.setattr(_lib, "call", call)
    return seen


def attend64(q, k, v, first, window, sinks):
    """q [n, Hq, D] at positions first .., k and v [L, Hk, D] -> the result and its tolerance, both [n, Hq, D] float64"""
    n, Hq, D = q.shape
    L, G = len(k), Hq // k.shape[1]
    p, s = first + torch.arange(n)[:, None], torch.arange(L)[None, :]
    seen = (s <= p) & ((s > p - window) | (s < sinks)) if window else s <= p
    u = torch.finfo(q.dtype).eps / 2
    out, tol = (torch.zeros(n, Hq, D, dtype=torch.float64) for _ in range(2))
    for h in range(Hq):
        qh, kh, vh = q[:, h].double(), k[:, h // G].double(), v[:, h // G].double()
        w = torch.softmax((qh @ kh.t() * D ** -0.5).masked_fill(~seen, float("-inf")), -1).nan_to_num(0.0)
        d = (D + 8) * 2.0 ** -23 * float((qh.abs() @ kh.abs().t()).max()) * D ** -0.5
        out[:, h] = w @ vh
        tol[:, h] = (3 * u + 2 * d + L * 2.0 ** -24) * (w @ vh.abs())
        if q.dtype is F16:
            tol[:, h] += L * 2.0 ** -32 * float(vh.abs().max()) + 2.0 ** -24
    return out, tol + 1e-30


def check(got, q, k, v, first, window, sinks, note):
    want, tol = attend64(q, k, v, first, window or 0, sinks)
    err = (got.double().cpu() - want).abs()
    assert bool(torch.isfinite(got).all()), note
    assert bool((err <= tol).all()), (note, float((err / tol).max()), float(err.max()))


LENS = [(6000, 40), (77, 1), (0, 5), (700, 33)]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (8, 1), (7, 1), (6, 2), (28, 4), (33, 1)])
@pytest.mark.parametrize("ps", [16, 48, 256])
def test_paged_attention_cut(cuts, dtype, D, Hq, Hk, ps):
    b = Batch(LENS, Hq=Hq, Hk=Hk, D=D, ps=ps, dtype=dtype, hnd=ps == 48, seed=ps + Hq, pad=3)
    b.q *= 3
    for window, sinks in ((None, 0), (2000, 5)):
        out = torch.full(b.q.shape, 7.0, dtype=dtype, device=DEV)
        b.gpu(window=window, sinks=sinks, out=out)
        assert cuts.pop() > 0
        for r, (c, n) in enumerate(b.lens):
            x = slice(int(b.cu[r]), int(b.cu[r + 1]))
            check(out[x], b.q[x], b.k[r], b.v[r], c, window, sinks, (r, window))
        assert bool((out[b.T:] == 7.0).all())


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk", [(4, 1), (7, 1), (6, 3)])
@pytest.mark.parametrize("Lq,Lk,window,sinks", [(1800, 1800, None, 0), (40, 6000, None, 0), (500, 5000, 1500, 20),
                                                (2111, 2111, 1900, 3), (300, 2500, None, 0)])
def test_window_attention_cut(cuts, dtype, D, Hq, Hk, Lq, Lk, window, sinks):
    """Few enough row tiles that the keys are cut; the queries as a part of one projection's rows, keys and values by
    heads, the output by heads."""
    B = 1 if Hq == 7 else 2
    g = torch.Generator().manual_seed(Lq + Hq)
    q = torch.zeros(B, Lq, Hq + 1, D, dtype=dtype)
    q[:, :, :Hq] = 3 * torch.randn(B, Lq, Hq, D, generator=g)
    k, v = (torch.randn(B, Hk, Lk, D, generator=g).to(dtype) for _ in range(2))
    out = torch.full((B, Hq, Lq, D), 7.0, dtype=dtype, device=DEV).transpose(1, 2)
    fa.window_attention(q.to(DEV)[:, :, :Hq].transpose(1, 2), k.to(DEV), v.to(DEV), window=window, sinks=sinks, out=out)
    assert cuts.pop() > 0
    for b in range(B):
        for i in {0, Lq // 2, Lq - 40}:
            check(out[b, i:i + 40], q[b, i:i + 40, :Hq], k[b].transpose(0, 1), v[b].transpose(0, 1), Lk - Lq + i, window,
                  sinks, (b, i))


def test_window_attention_cut_before_the_first_key(cuts):
    """More queries than keys: the first stand before any key and are 0, also where row tiles are cut."""
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(1, h, n, 128, generator=g).to(BF) for h, n in ((4, 2300), (1, 2100), (1, 2100)))
    got = fa.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), window=None)
    assert cuts.pop() > 0
    assert bool((got[0, :200] == 0).all())
    for i in (200, 1500, 2260):
        check(got[0, i:i + 40], q[0, :, i:i + 40].transpose(0, 1), k[0].transpose(0, 1), v[0].transpose(0, 1), i - 200,
              None, 0, i)


@pytest.mark.parametrize("max_new", [1, None])
@pytest.mark.parametrize("Hq,Hk,D", [(4, 1, 128), (28, 4, 64), (64, 64, 128)])
def test_workspaces_hold_what_is_written(cuts, max_new, Hq, Hk, D):
    """Single tokens in workspaces of the size asked for, by either kernel."""
    b = Batch([(2900, 1), (900, 1), (0, 0), *((i, 1) for i in range(40))], Hq=Hq, Hk=Hk, D=D, ps=64, seed=7)
    b.q *= 3
    got = b.gpu(max_new=max_new)
    for r, (c, n) in enumerate(b.lens):
        x = slice(int(b.cu[r]), int(b.cu[r + 1]))
        if n:
            check(got[x], b.q[x], b.k[r], b.v[r], c, None, 0, r)
    assert max_new == 1 or cuts.pop() >= 0


@pytest.mark.parametrize("lens", [[(6000, 1), (50, 1)], [(6000, 40), (50, 1)]], ids=["tokens", "chunk"])
def test_the_largest_values(cuts, lens):
    """bf16 values up to 2^93, the sums' range at any length: equal weights, and weights that grow along the keys (a row's
    running maximum then lags behind, and weights up to 2^8 are summed)."""
    for rise in (0.0, 0.004):
        b = Batch(lens, ps=64, seed=30)
        b.q[:] = 1
        for r, x in enumerate(b.k):
            x[:] = (rise * torch.arange(len(x)) / 11.3).to(BF)[:, None, None]
            b.v[r] = b.v[r].clamp(-1, 1) * 2.0 ** 93
            for i in range(-(-len(x) // 64)):
                n = min(64, len(x) - 64 * i)
                b.kc[b.table[r, i], :n], b.vc[b.table[r, i], :n] = x[64 * i:64 * i + n], b.v[r][64 * i:64 * i + n]
        got = b.gpu()
        for r, (c, n) in enumerate(b.lens):
            x = slice(int(b.cu[r]), int(b.cu[r + 1]))
            check(got[x], b.q[x], b.k[r], b.v[r], c, None, 0, (r, rise))
