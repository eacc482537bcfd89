"""CPU tests of the host side of trees and 8-bit pages: what is refused, and with which error, before any launch (through
Python and at the C ABI), the registers of the kernels' forms, and the oracle itself."""
from __future__ import annotations

import ctypes
import re

import pytest
import torch

import fftsparse_amd as fa
from fftsparse_amd import _lib
from oracle import paged, tree
from tests.test_isa_hazards import CSRC, HIPCC, _compile
from tests.test_serving_host import BF, I32, _paged, _rc

E4M3 = torch.float8_e4m3fn
I64 = torch.int64


def _tree(**kw):
    return {**_paged(), "mask": torch.zeros(6, 1, dtype=I64), **kw}


def _eight(f=_paged, **kw):
    cache = torch.zeros(8, 16, 2, 128, dtype=torch.uint8).view(E4M3)
    return {**f(), "k_cache": cache, "v_cache": cache, "k_scale": torch.ones(2), "v_scale": torch.ones(2), **kw}


@pytest.mark.parametrize("error,text,args", [
    (ValueError, "on the GPU", _tree()),
    (ValueError, "mask", _tree(mask=torch.zeros(5, 1, dtype=I64))),
    (ValueError, "mask", _tree(mask=torch.zeros(6, 0, dtype=I64))),
    (ValueError, "mask", _tree(mask=torch.zeros(6, 1, dtype=I32))),
    (ValueError, "mask", _tree(mask=torch.zeros(6, dtype=I64))),
    (ValueError, "mask", _tree(mask=torch.zeros(6, 4, dtype=I64)[:, ::2])),
    (ValueError, "positions", _tree(window=5)),
    (ValueError, "positions", _tree(window=5, positions=torch.zeros(5, dtype=I32))),
    (ValueError, "positions", _tree(window=5, positions=torch.zeros(6, dtype=I64))),
    (ValueError, "window", _tree(window=0)),
    (ValueError, "max_new", _tree(max_new=0)),
    (TypeError, "bf16 or f16", _tree(q=torch.zeros(6, 4, 128))),
    (RuntimeError, "tree_attention has no backward", _tree(q=torch.zeros(6, 4, 128, dtype=BF, requires_grad=True))),
    (ValueError, "on the GPU", _eight(_tree)),
    (ValueError, "need k_scale", _eight(_tree, k_scale=None)),
])
def test_tree_attention_refuses(error, text, args):
    with pytest.raises(error, match=text):
        fa.tree_attention(**args)


@pytest.mark.parametrize("error,text,args", [
    (ValueError, "on the GPU", _eight()),
    (ValueError, "need k_scale", _eight(k_scale=None)),
    (ValueError, "need k_scale", _eight(v_scale=None)),
    (ValueError, "k_scale must be", _eight(k_scale=torch.ones(4))),
    (ValueError, "k_scale must be", _eight(k_scale=torch.ones(2, dtype=torch.float64))),
    (ValueError, "v_scale must be", _eight(v_scale=torch.ones(4)[::2])),
    (ValueError, "v_scale must be", _eight(v_scale=torch.ones(()))),
    (ValueError, "go with caches", {**_paged(), "k_scale": torch.ones(2), "v_scale": torch.ones(2)}),
    (ValueError, "go with caches", {**_paged(), "v_scale": torch.ones(2)}),
    (TypeError, "bf16 or f16", _eight(v_cache=torch.zeros(8, 16, 2, 128, dtype=BF))),
    (TypeError, "bf16 or f16", _eight(k_cache=torch.zeros(8, 16, 2, 128, dtype=BF))),
    (TypeError, "bf16 or f16", _eight(q=torch.zeros(6, 4, 128, dtype=torch.uint8).view(E4M3))),
    (ValueError, "multiples of 16", _eight(k_cache=torch.zeros(8, 16, 2, 136, dtype=torch.uint8).view(E4M3)[..., :128])),
    (ValueError, "k_cache", _eight(k_cache=torch.zeros(8, 16, 256, dtype=torch.uint8).view(E4M3))),
])
def test_paged_attention_in_8_bits_refuses(error, text, args):
    with pytest.raises(error, match=text):
        fa.paged_attention(**args)


def test_window_attention_takes_no_8_bits():
    q, k = torch.zeros(1, 4, 10, 128, dtype=BF), torch.zeros(1, 2, 10, 128, dtype=torch.uint8).view(E4M3)
    with pytest.raises(TypeError, match="bf16 or f16"):
        fa.window_attention(q, k, k, window=4)


def test_rope_cache_in_8_bits_refuses():
    q, k = torch.zeros(6, 4, 128, dtype=BF), torch.zeros(6, 2, 128, dtype=BF)
    pos, inv, slots = torch.zeros(6, dtype=I32), torch.ones(64, dtype=torch.float64), torch.zeros(6, dtype=I64)
    c8, c16 = torch.zeros(4, 16, 2, 128, dtype=torch.uint8).view(E4M3), torch.zeros(4, 16, 2, 128, dtype=BF)
    one = torch.ones(2)
    for text, kc, vc, kw in [("on the GPU", c8, c8, dict(k_scale=one, v_scale=one)), ("need k_scale", c8, c8, {}),
                             ("need k_scale", c8, c8, dict(k_scale=one)), ("go with caches", c16, c16, dict(k_scale=one, v_scale=one)),
                             ("v_cache", c8, c16, dict(k_scale=one, v_scale=one)),
                             ("v_scale must be", c8, c8, dict(k_scale=one, v_scale=torch.ones(1))),
                             ("multiples of 16", torch.zeros(4, 16, 2, 136, dtype=torch.uint8).view(E4M3)[..., :128], c8,
                              dict(k_scale=one, v_scale=one))]:
        with pytest.raises(ValueError, match=text):
            fa.rope_cache(q, k, k, pos, slots, kc, vc, inv, **kw)


def test_plan_and_accept_refuse():
    p, cu, lens, x = torch.zeros(6, dtype=I32), torch.zeros(4, dtype=I32), torch.zeros(3, dtype=I32), torch.zeros(6, dtype=I64)
    for text, args, n in [("on the GPU", (p, cu, lens), 4), ("parents", (x, cu, lens), 4), ("parents", (p[None], cu, lens), 4),
                          ("parents", (torch.zeros(12, dtype=I32)[::2], cu, lens), 4), ("cu_lens", (p, cu.long(), lens), 4),
                          ("cu_lens", (p, cu[:1], lens), 4), ("seq_lens", (p, cu, cu), 4), ("max_new", (p, cu, lens), 0),
                          ("max_new", (p, cu, lens), 1025)]:
        with pytest.raises(ValueError, match=text):
            fa.plan_tree(*args, max_new=n)
    for text, args, n in [("on the GPU", (p, x, x, cu), 4), ("tokens", (p, x.float(), x, cu), 4), ("tokens", (p, x[:5], x, cu), 4),
                          ("chosen", (p, x, p, cu), 4), ("chosen", (p, x, x[:5], cu), 4), ("parents", (x, x, x, cu), 4),
                          ("cu_lens", (p, x, x, cu[None]), 4), ("max_new", (p, x, x, cu), 2000)]:
        with pytest.raises(ValueError, match=text):
            fa.accept_tree(*args, max_new=n)


def test_move_kept_refuses():
    c, t = torch.zeros(8, 16, 2, 128, dtype=BF), torch.zeros(3, 4, dtype=I32)
    cu, lens, kept = torch.zeros(4, dtype=I32), torch.zeros(3, dtype=I32), torch.zeros(6, dtype=I32)
    other = torch.zeros(8, 2, 16, 128, dtype=BF).transpose(1, 2)
    for error, text, k, v, rest in [
            (ValueError, "on the GPU", c, c, {}), (ValueError, "on the GPU", [c, c], [c, c], {}),
            (ValueError, "on the GPU", torch.stack([c, c]), torch.stack([c, c]), {}),
            (ValueError, "k_cache must be", c[0], c, {}), (ValueError, "k_cache must be", [], [], {}),
            (ValueError, "no layer", [c], [], {}), (ValueError, "layers of keys", [c, c], [c], {}),
            (ValueError, "layers of keys", [c], c, {}), (ValueError, "layers of keys", torch.stack([c, c]), c, {}),
            (ValueError, "v_cache", torch.stack([c, c]), torch.stack([c, c]).half(), {}),
            (ValueError, "v_cache", c, torch.stack([c, c])[..., :64], {}),
            (ValueError, "broadcast", torch.stack([c, c]), c[None].expand(2, *c.shape), {}),
            (ValueError, "k_cache must be", [torch.stack([c, c])], [torch.stack([c, c])], {}),
            (ValueError, "one shape", [c, other], [c, c], {}), (ValueError, "one shape", [c, c.half()], [c, c], {}),
            (ValueError, "v_cache", c, c[..., :64], {}), (ValueError, "v_cache", c, c.half(), {}),
            (TypeError, "unsupported", c.double(), c.double(), {}),
            (ValueError, "broadcast", c, c[:, :, :1].expand(8, 16, 2, 128), {}),
            (ValueError, "multiples of 16 bytes", torch.zeros(2 * c.numel() + 4, dtype=BF).as_strided((2, *c.shape), (c.numel() + 4,
             *c.stride())), torch.stack([c, c]), {}),
            (ValueError, "block_table", c, c, dict(block_table=t.long())), (ValueError, "cu_lens", c, c, dict(cu_lens=cu[:3])),
            (ValueError, "seq_lens", c, c, dict(seq_lens=cu)), (ValueError, "kept", c, c, dict(kept=kept.long()))]:
        with pytest.raises(error, match=text):
            fa.move_kept(k, v, **{**dict(block_table=t, cu_lens=cu, seq_lens=lens, kept=kept), **rest})
    with pytest.raises(RuntimeError, match="no backward"):
        fa.move_kept(c.clone().requires_grad_(), c, t, cu, lens, kept)


def test_c_abi_refuses_without_a_launch():
    lib = _lib.load()
    for name in ("fs_tree_plan", "fs_tree_accept", "fs_cache_move"):
        assert getattr(lib, name)(None, None) == -1
        assert b"null args" in lib.fs_last_error()

    def attn(**kw):
        return _lib.PagedAttnArgs(q=16, out=16, k_cache=16, v_cache=16, block_table=16, t_sb=4, cu_lens=16, seq_lens=16,
                                  dtype=1, B=2, T=3, Hq=4, Hk=2, D=128, P=4, page_size=16, num_pages=8, work=16, **kw)
    for text, change in [("come together", dict(k_scale=16)), ("come together", dict(v_scale=16)),
                         ("come together", dict(k_scale=16, v_scale=18)),
                         ("multiples of 16", dict(k_scale=16, v_scale=16, v_ss=8)), ("mask of 0", dict(mask=16)),
                         ("aligned", dict(mask=20, mask_words=1)), ("positions", dict(mask=16, mask_words=1, window=3)),
                         ("aligned", dict(mask=16, mask_words=1, positions=18))]:
        got, said = _rc("fs_paged_attn", attn(), **change)
        assert (got, text in said) == (-1, True), (change, got, said)

    def rope():
        return _lib.RopeArgs(q=16, k=16, v=16, positions=16, inv_freq=16, attention_factor=1.0, pos_bytes=4, half=64, dtype=1,
                             T=2, Hq=4, Hk=2, D=128, q_out=16, slots=16, k_cache=16, v_cache=16, num_pages=2, page_size=16)
    for text, change in [("come together", dict(k_scale=16)), ("come together", dict(k_scale=16, v_scale=16, slots=None, v=None, k_out=16)),
                         ("multiples of 16", dict(k_scale=16, v_scale=16, vc_ss=8))]:
        got, said = _rc("fs_rope", rope(), **change)
        assert (got, text in said) == (-1, True), (change, got, said)

    def plan():
        return _lib.TreePlanArgs(parents=16, cu_lens=16, seq_lens=16, B=2, T=3, words=1, positions=16, mask=16)
    for rc, text, change in [(-1, "B=0", dict(B=0)), (-1, "T=-1", dict(T=-1)), (-1, "0 words", dict(words=0)),
                             (-2, "1088", dict(words=17)), (-1, "null tensor", dict(mask=None)), (-2, "65536", dict(B=65536))]:
        got, said = _rc("fs_tree_plan", plan(), **change)
        assert (got, text in said) == (rc, True), (change, got, said)

    def accept():
        return _lib.TreeAcceptArgs(parents=16, tokens=16, chosen=16, cu_lens=16, token_bytes=8, B=2, T=3, most=4, kept=16,
                                   kept_lens=16, dropped=16, next_tokens=16)
    for rc, text, change in [(-1, "of 2 bytes", dict(token_bytes=2)), (-1, "trees of 0", dict(most=0)),
                             (-2, "trees of 1025", dict(most=1025)), (-1, "null tensor", dict(dropped=None)),
                             (-1, "null tensor", dict(chosen=None))]:
        got, said = _rc("fs_tree_accept", accept(), **change)
        assert (got, text in said) == (rc, True), (change, got, said)

    ptrs = (ctypes.c_void_p * 2)(16, 32)
    odd = (ctypes.c_void_p * 2)(16, 8)

    def move():
        return _lib.CacheMoveArgs(k_caches=ptrs, v_caches=ptrs, block_table=16, t_sb=4, cu_lens=16, seq_lens=16, kept=16,
                                  layers=2, B=2, T=3, Hk=2, D=128, P=4, page_size=16, elem_bytes=2, num_pages=8)
    for rc, text, change in [(-1, "of 3 bytes", dict(elem_bytes=3)), (-2, "heads of 4", dict(D=4)), (-1, "layers=-1", dict(layers=-1)),
                             (-1, "16-byte", dict(k_caches=odd)), (-1, "null tensor", dict(v_caches=None)),
                             (-1, "caches must be given", dict(k_caches=None, v_caches=None)),
                             (-1, "16-byte", dict(k_caches=None, v_caches=None, k_cache=8, v_cache=16)),
                             (-1, "multiples of 16 bytes", dict(k_caches=None, v_caches=None, k_cache=16, v_cache=16, v_sl=4)), (-1, "multiples of 16 bytes", dict(v_ss=4)),
                             (-1, "row stride 3", dict(t_sb=3)), (-1, "null tensor", dict(kept=None)),
                             (-2, "per request", dict(P=1 << 28, t_sb=1 << 28))]:
        got, said = _rc("fs_cache_move", move(), **change)
        assert (got, text in said) == (rc, True), (change, got, said)


@pytest.mark.skipif(HIPCC is None, reason="hipcc is not installed")
@pytest.mark.parametrize("name", ["paged8", "paged_tree", "paged8_tree"])
def test_the_forms_spill_no_vector_registers(tmp_path, name):
    asm = _compile(CSRC / f"{name}.hip", tmp_path / f"{name}.s")
    spills = {}
    for meta in asm.split("  - .agpr_count:")[1:]:
        spills[re.search(r"\.name: +(\S+)", meta)[1]] = int(re.search(r"\.vgpr_spill_count: +(\d+)", meta)[1])
    assert sum("many_kernel" in n for n in spills) == 4 and sum("few_kernel" in n for n in spills) == (6 if "8" in name else 4)
    assert {n: s for n, s in spills.items() if s} == {}


def test_the_oracle_of_a_chain_is_that_of_paged_attention():
    g = torch.Generator().manual_seed(0)
    q, k, v = torch.randn(9, 4, 16, generator=g), *(torch.randn(30, 2, 16, generator=g) for _ in range(2))
    pos, mask = tree.plan([-1, *range(8)], [0, 9], [30], 1)
    assert pos == list(range(21, 30)) and mask == [[(1 << t + 1) - 1] for t in range(9)]
    sees = torch.ones(9, 9).tril().bool()
    for window, sinks in ((None, 0), (25, 2), (10, 0)):
        a = tree.attend(q, k, v, 9, sees, window, sinks, pos=pos)[0]
        b = paged.attend(q, k, v, 21, window, sinks)[0]
        assert torch.allclose(a, b, atol=1e-12)


def test_half_steps_of_e4m3():
    x = torch.tensor([1.0, 1.9, 2.0, 0.5, 448.0, 300.0, 2.0 ** -6, 2.0 ** -7, 0.0, 500.0], dtype=torch.float64)
    assert tree.e4m3_half_step(x).tolist() == [2.0 ** -4, 2.0 ** -4, 2.0 ** -3, 2.0 ** -5, 16.0, 16.0, 2.0 ** -10, 2.0 ** -10,
                                               2.0 ** -10, 16.0]


def _bytes(T=64, B=8, Hq=32, Hk=8, D=128, P=64, max_new=0, eight=True, tree=False):
    a = _lib.PagedAttnArgs(dtype=1, B=B, T=T, Hq=Hq, Hk=Hk, D=D, P=P, page_size=64, max_new=max_new)
    if eight:
        a.k_scale = a.v_scale = 16
    if tree:
        a.mask, a.mask_words = 16, 1
    return _lib.load().fs_paged_attn_work_bytes(ctypes.byref(a))


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("eight", [False, True])
def test_workspaces_of_the_forms_never_fall(eight, tree):
    """One sized for the largest call of a form serves every smaller one of it, and 8-bit calls' serve 16-bit ones'."""
    kw = dict(eight=eight, tree=tree)
    for B in (1, 64, 4096):
        for m in (0, 1, 8, 64):
            n = [_bytes(T, B, max_new=m, **kw) for T in (1, 2, 8, 64, 1000, 4096, 100000)]
            assert n == sorted(n) and n[0] > 0
    for T in (1, 64, 5000):
        for D in (64, 128):
            n = [_bytes(T, 16, D=D, max_new=m, **kw) for m in [*range(1, 200), 0]]
            assert n == sorted(n)
        n = [_bytes(T, 16, P=1 << p, max_new=1, **kw) for p in range(20)]
        assert n == sorted(n)
        for m in (1, 64):
            assert _bytes(T, 16, D=64, max_new=m, **kw) <= _bytes(T, 16, D=128, max_new=m, **kw)
            heads = [(1, 1), (4, 1), (8, 1), (8, 2), (32, 2), (32, 8), (64, 8), (64, 64)]
            n = [_bytes(T, 16, q, k, max_new=m, **kw) for q, k in heads]
            assert n == sorted(n)
            assert _bytes(T, 16, max_new=m, eight=True, tree=tree) >= _bytes(T, 16, max_new=m, eight=False, tree=tree)


def test_scales_and_outputs_that_are_refused():
    with pytest.raises(RuntimeError, match="no backward"):
        fa.paged_attention(**_eight(k_scale=torch.ones(2, requires_grad=True)))
    q, k = torch.zeros(6, 4, 128, dtype=BF), torch.zeros(6, 2, 128, dtype=BF)
    c8 = torch.zeros(4, 16, 2, 128, dtype=torch.uint8).view(E4M3)
    with pytest.raises(RuntimeError, match="no backward"):
        fa.rope_cache(q, k, k, torch.zeros(6, dtype=I32), torch.zeros(6, dtype=I64), c8, c8, torch.ones(64, dtype=torch.float64),
                      k_scale=torch.ones(2), v_scale=torch.ones(2, requires_grad=True))
