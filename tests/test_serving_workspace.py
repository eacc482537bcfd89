"""Workspace sizes of the serving attentions (no GPU): a caller that allocates once, for the most tokens, requests, heads
and lengths it serves, has enough for every smaller call, whichever kernel a call takes."""
from __future__ import annotations

import ctypes
import itertools

import pytest

from fftsparse_amd import _lib


def paged_bytes(T=64, B=8, Hq=32, Hk=8, D=128, P=64, page_size=64, max_new=0):
    a = _lib.PagedAttnArgs(dtype=1, B=B, T=T, Hq=Hq, Hk=Hk, D=D, P=P, page_size=page_size, max_new=max_new)
    return _lib.load().fs_paged_attn_work_bytes(ctypes.byref(a))


def window_bytes(L=1000, Lk=None, B=2, Hq=32, Hk=8, D=128):
    a = _lib.WindowAttnArgs(dtype=1, B=B, Hq=Hq, Hk=Hk, Lq=L, Lk=Lk or L, D=D, window=100)
    return _lib.load().fs_window_attn_work_bytes(ctypes.byref(a))


HEADS = [(q, k) for q in (1, 2, 4, 7, 8, 16, 28, 32, 33, 40, 64, 128) for k in range(1, q + 1) if q % k == 0]
# (fewer heads, more heads): neither the query heads nor the KV heads fall
GROWING = [(a, b) for a, b in itertools.product(HEADS, HEADS) if a != b and a[0] <= b[0] and a[1] <= b[1]]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,B,max_new", [(512, 8, 0), (64, 64, 1), (1, 1, 1), (256, 32, 8), (4096, 4, 1000), (100, 4096, 4)])
def test_paged_workspace_serves_fewer_heads(T, B, max_new, D):
    n = {h: paged_bytes(T, B, *h, D, max_new=max_new) for h in HEADS}
    assert min(n.values()) > 0
    assert [(a, b) for a, b in GROWING if n[a] > n[b]] == []


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("L,Lk", [(1, 1), (1, 5000), (8, 8), (1000, 1000), (16384, 16384), (40, 6000)])
def test_window_workspace_serves_fewer_heads(L, Lk, D):
    n = {h: window_bytes(L, Lk, 2, *h, D) for h in HEADS}
    assert min(n.values()) > 0
    assert [(a, b) for a, b in GROWING if n[a] > n[b]] == []


@pytest.mark.parametrize("Hq,Hk", [(32, 1), (32, 8), (32, 32), (4, 1), (64, 8)])
def test_paged_workspace_where_the_key_tiles_are_counted_out(Hq, Hk):
    """Single tokens whose key tiles pass 30 bits take the other kernel: the size does not fall there either, as the
    tokens, the requests, the pages or their length grow."""
    T = sorted({int(2.0 ** (i / 8)) for i in range(8 * 23 + 1) if 2.0 ** (i / 8) * Hq < 2 ** 30} | {8_000_000, 8_300_000})
    T = [t for t in T if t * Hq < 2 ** 30]
    for keys in (64, 4096, 1 << 17, 1 << 26):
        n = [paged_bytes(t, 8, Hq, Hk, P=keys // 64, max_new=1) for t in T]
        assert n == sorted(n)
    for t in (1, 1000, 100_000, T[-1]):
        n = [paged_bytes(t, 4096, Hq, Hk, P=1 << p, max_new=1) for p in range(21)]
        assert n == sorted(n)
        n = [paged_bytes(t, 4096, Hq, Hk, P=1 << 14, page_size=16 << s, max_new=1) for s in range(9)]
        assert n == sorted(n)
        n = [paged_bytes(t, B, Hq, Hk, P=1 << 20, max_new=1) for B in range(1, 4097, 7)]
        assert n == sorted(n)
        n = [paged_bytes(t, 64, Hq, Hk, max_new=m) for m in [*range(1, 150), 0]]
        assert n == sorted(n)


@pytest.mark.parametrize("Hq,Hk", HEADS)
def test_the_wider_head_has_the_larger_workspace(Hq, Hk):
    for T, B, max_new in ((64, 64, 1), (1, 1, 1), (5000, 8, 0)):
        assert paged_bytes(T, B, Hq, Hk, 64, max_new=max_new) <= paged_bytes(T, B, Hq, Hk, 128, max_new=max_new)
    for L in (1, 700, 20000):
        assert window_bytes(L, L, 2, Hq, Hk, 64) <= window_bytes(L, L, 2, Hq, Hk, 128)


def test_window_workspace_serves_shorter_calls():
    for Hq, Hk in ((32, 8), (28, 4), (4, 1)):
        for B in (1, 3):
            n = [window_bytes(L, Lk, B, Hq, Hk) for L in (1, 8, 9, 500, 5000) for Lk in (L, L + 6000, 1 << 20)]
            assert all(window_bytes(L, Lk, B, Hq, Hk) <= window_bytes(M, Mk, B, Hq, Hk)
                       for L, M in ((1, 8), (8, 9), (9, 500), (500, 5000)) for Lk, Mk in ((L, M), (6000, 6000), (L, 1 << 20)))
            assert min(n) > 0
