"""CPU tests of the serving operators' host side: what is refused, and with which error, before any launch (through
Python and at the C ABI), and the frequencies."""
from __future__ import annotations

import ctypes
import math
import re

import pytest
import torch

import fftsparse_amd as fa
from fftsparse_amd import _lib
from tests.test_isa_hazards import CSRC, HIPCC, _compile

BF = torch.bfloat16


def _paged(T=6, Hq=4, Hk=2, D=128, ps=16, pages=8, B=3, P=4, dtype=BF):
    i32 = torch.int32
    return dict(q=torch.zeros(T, Hq, D, dtype=dtype), k_cache=torch.zeros(pages, ps, Hk, D, dtype=dtype),
                v_cache=torch.zeros(pages, ps, Hk, D, dtype=dtype), block_table=torch.zeros(B, P, dtype=i32),
                cu_lens=torch.zeros(B + 1, dtype=i32), seq_lens=torch.zeros(B, dtype=i32))


def _changed(**kw):
    return {**_paged(), **kw}


I32 = torch.int32
PAGED_BAD = [
    (ValueError, "on the GPU", {}),
    (ValueError, r"\[T, H, D\]", dict(q=torch.zeros(6, 512, dtype=BF))),
    (TypeError, "bf16 or f16", dict(q=torch.zeros(6, 4, 128))),
    (TypeError, "bf16 or f16", dict(q=torch.zeros(6, 4, 128, dtype=torch.float16))),
    (ValueError, "k_cache", dict(k_cache=torch.zeros(8, 16, 256, dtype=BF))),
    (ValueError, "k_cache", dict(q=torch.zeros(6, 4, 64, dtype=BF))),
    (ValueError, "v_cache", dict(v_cache=torch.zeros(8, 16, 1, 128, dtype=BF))),
    (ValueError, "d contiguous", dict(k_cache=torch.zeros(8, 16, 128, 2, dtype=BF).transpose(2, 3))),
    (ValueError, "multiple of key heads", dict(q=torch.zeros(6, 3, 128, dtype=BF))),
    (ValueError, "block_table", dict(block_table=torch.zeros(3, 4, dtype=torch.int64))),
    (ValueError, "block_table", dict(block_table=torch.zeros(4, 3, dtype=I32).t())),
    (ValueError, "overlap", dict(block_table=torch.zeros(4, dtype=I32).expand(3, 4))),
    (ValueError, "cu_lens", dict(cu_lens=torch.zeros(3, dtype=I32))),
    (ValueError, "cu_lens", dict(cu_lens=torch.zeros(4, dtype=torch.int64))),
    (ValueError, "seq_lens", dict(seq_lens=torch.zeros(6, dtype=I32)[::2])),
    (ValueError, "window", dict(window=0)),
    (ValueError, "window", dict(window=-3)),
    (ValueError, "sinks", dict(window=4, sinks=-1)),
    (ValueError, "max_new", dict(max_new=0)),
    (ValueError, "softmax_scale", dict(softmax_scale=-0.1)),
    (ValueError, "softmax_scale", dict(softmax_scale=math.nan)),
    (ValueError, "out must be", dict(out=torch.zeros(6, 4, 64, dtype=BF))),
    (ValueError, "broadcast", dict(out=torch.zeros(1, 4, 128, dtype=BF).expand(6, 4, 128))),
    (RuntimeError, "no backward", dict(q=torch.zeros(6, 4, 128, dtype=BF, requires_grad=True))),
]


@pytest.mark.parametrize("error,text,change", PAGED_BAD, ids=[f"{i}-{t[:12]}" for i, (_, t, _) in enumerate(PAGED_BAD)])
def test_paged_attention_refuses(error, text, change):
    with pytest.raises(error, match=text):
        fa.paged_attention(**_changed(**change))


def test_window_attention_refuses():
    q, k = torch.zeros(1, 4, 10, 128, dtype=BF), torch.zeros(1, 2, 10, 128, dtype=BF)
    for error, text, args, kw in [
            (ValueError, "on the GPU", (q, k, k), dict(window=4)),
            (ValueError, "window", (q, k, k), dict(window=0)),
            (ValueError, "sinks", (q, k, k), dict(window=4, sinks=-1)),
            (ValueError, "softmax_scale", (q, k, k), dict(window=4, softmax_scale=-1.0)),
            (TypeError, "bf16 or f16", (q.float(), k.float(), k.float()), dict(window=4)),
            (ValueError, "do not match", (q, k, k[:, :, :5]), dict(window=4)),
            (ValueError, "do not match", (q, k[..., :64], k[..., :64]), dict(window=4)),
            (ValueError, "multiple of key heads", (q[:, :3], k, k), dict(window=4)),
            (ValueError, "empty", (q[:, :, :0], k, k), dict(window=4)),
            (ValueError, "out must be", (q, k, k), dict(window=4, out=torch.zeros(1, 4, 10, 128, dtype=BF)))]:
        with pytest.raises(error, match=text):
            fa.window_attention(*args, **kw)
    with pytest.raises(RuntimeError, match="no backward"):
        fa.window_attention(q.clone().requires_grad_(), k, k, window=4)


def _plan(B=3, P=4, F=8):
    return dict(block_table=torch.zeros(B, P, dtype=I32), seq_lens=torch.zeros(B, dtype=I32),
                new_lens=torch.zeros(B, dtype=I32), free_pages=torch.zeros(F, dtype=I32),
                free_count=torch.zeros(1, dtype=I32), page_size=16, num_tokens=5)


@pytest.mark.parametrize("text,change", [
    ("on the GPU", {}),
    ("block_table", dict(block_table=torch.zeros(3, 4))),
    ("block_table", dict(block_table=torch.zeros(0, 4, dtype=I32))),
    ("seq_lens", dict(seq_lens=torch.zeros(4, dtype=I32))),
    ("new_lens", dict(new_lens=torch.zeros(3, dtype=torch.int64))),
    ("free_pages", dict(free_pages=torch.zeros(0, dtype=I32))),
    ("free_count", dict(free_count=torch.zeros((), dtype=I32))),
    ("out of range", dict(page_size=0)),
    ("out of range", dict(num_tokens=-1)),
    ("out of range", dict(page_size=1 << 29)),
])
def test_plan_step_refuses(text, change):
    with pytest.raises(ValueError, match=text):
        fa.plan_step(**{**_plan(), **change})


def test_rope_refuses():
    q, k = torch.zeros(6, 4, 128, dtype=BF), torch.zeros(6, 2, 128, dtype=BF)
    pos, inv = torch.zeros(6, dtype=I32), torch.ones(64, dtype=torch.float64)
    slots, cache = torch.zeros(6, dtype=torch.int64), torch.zeros(4, 16, 2, 128, dtype=BF)
    for error, text, args in [
            (ValueError, "on the GPU", (q, k, pos, inv)),
            (ValueError, "do not match", (q, k[:5], pos, inv)),
            (ValueError, "do not match", (q, k[..., :64], pos, inv)),
            (TypeError, "dtypes", (q, k.float(), pos, inv)),
            (TypeError, "dtypes", (q.double(), k.double(), pos, inv)),
            (ValueError, "positions", (q, k, pos[:5], inv)),
            (ValueError, "positions", (q, k, pos.float(), inv)),
            (ValueError, "inv_freq", (q, k, pos, torch.ones(65, dtype=torch.float64))),
            (ValueError, "inv_freq", (q, k, pos, torch.ones(64, dtype=torch.int64)))]:
        with pytest.raises(error, match=text):
            fa.rope(*args)
    with pytest.raises(ValueError, match="q_out"):
        fa.rope(q, k, pos, inv, q_out=torch.zeros(6, 4, 64, dtype=BF))
    with pytest.raises(RuntimeError, match="no backward"):
        fa.rope(q, k.clone().requires_grad_(), pos, inv)
    for text, args in [("on the GPU", (q, k, k, pos, slots, cache, cache, inv)),
                       ("value", (q, k, q, pos, slots, cache, cache, inv)),
                       ("slots", (q, k, k, pos, slots.int(), cache, cache, inv)),
                       ("k_cache", (q, k, k, pos, slots, cache[..., :64], cache, inv)),
                       ("v_cache", (q, k, k, pos, slots, cache, cache.half(), inv))]:
        with pytest.raises(ValueError, match=text):
            fa.rope_cache(*args)


def _rc(name, args, **change):
    for f, v in change.items():
        setattr(args, f, v)
    lib = _lib.load()
    return getattr(lib, name)(ctypes.byref(args), None), lib.fs_last_error().decode()


def test_c_abi_refuses_without_a_launch():
    lib = _lib.load()
    for name in ("fs_plan", "fs_rope", "fs_paged_attn", "fs_window_attn"):
        assert getattr(lib, name)(None, None) == -1
        assert b"null args" in lib.fs_last_error()
    assert lib.fs_paged_attn_work_bytes(None) == lib.fs_window_attn_work_bytes(None) == 0

    def paged():
        return _lib.PagedAttnArgs(q=16, out=16, k_cache=16, v_cache=16, block_table=16, t_sb=4, cu_lens=16, seq_lens=16,
                                  dtype=1, B=2, T=3, Hq=4, Hk=2, D=128, P=4, page_size=16, num_pages=8, work=16)
    for rc, text, change in [(-2, "page size 24", dict(page_size=24)), (-2, "page size 8192", dict(page_size=8192)),
                             (-2, "tokens per request", dict(P=1 << 23, t_sb=1 << 23)), (-2, "head_dim 96", dict(D=96)),
                             (-2, "dtype 0", dict(dtype=0)), (-1, "Hq=3", dict(Hq=3)), (-1, "window", dict(window=-1)),
                             (-1, "16-byte", dict(q=8)), (-1, "multiples of 8", dict(k_ss=100)),
                             (-1, "null tensor", dict(work=None)), (-1, "4-byte", dict(cu_lens=18)),
                             (-1, "row stride", dict(t_sb=3)), (-1, "num_pages=0", dict(num_pages=0)),
                             (-2, "rows of", dict(T=1 << 29)), (-2, "67108864 pages", dict(num_pages=1 << 26)),
                             (-2, "4097 requests", dict(B=4097)), (-2, "slot stride", dict(v_ss=1 << 23)),
                             (-1, "finite", dict(softmax_scale=math.nan)), (-1, "finite", dict(softmax_scale=math.inf)),
                             (-1, "negative", dict(softmax_scale=-0.1))]:
        got, said = _rc("fs_paged_attn", paged(), **change)
        assert (got, text in said) == (rc, True), (change, got, said)
    assert _rc("fs_paged_attn", paged(), T=0)[0] == 0                     # no token: nothing to do

    def window():
        return _lib.WindowAttnArgs(q=16, k=16, v=16, out=16, work=16, dtype=1, B=1, Hq=4, Hk=2, Lq=5, Lk=5, D=128,
                                   window=3)
    for rc, text, change in [(-1, "empty", dict(Lq=0)), (-2, "head_dim", dict(D=80)), (-1, "sinks", dict(sinks=-1)),
                             (-2, "keys", dict(Lk=1 << 27)), (-1, "multiples of 8", dict(o_sl=4))]:
        got, said = _rc("fs_window_attn", window(), **change)
        assert (got, text in said) == (rc, True), (change, got, said)

    def plan():
        return _lib.PlanArgs(block_table=16, t_sb=4, seq_lens=16, new_lens=16, free_pages=16, free_count=16, B=2, P=4,
                             F=8, page_size=16, T=4, cu_lens=16, seq_lens_out=16, positions=16, slots=16,
                             free_count_out=16, lacking=16)
    for rc, text, change in [(-2, "4097 requests", dict(B=4097)), (-1, "page size 0", dict(page_size=0)),
                             (-1, "row stride 3", dict(t_sb=3)), (-1, "null tensor", dict(slots=None)),
                             (-1, "F=0", dict(F=0))]:
        got, said = _rc("fs_plan", plan(), **change)
        assert (got, text in said) == (rc, True), (change, got, said)

    def rope():
        return _lib.RopeArgs(q=16, k=16, positions=16, inv_freq=16, attention_factor=1.0, pos_bytes=4, half=64,
                             dtype=1, T=2, Hq=4, Hk=2, D=128, q_out=16, k_out=16)
    for rc, text, change in [(-1, "positions of 2", dict(pos_bytes=2)), (-1, "rotary dim 130", dict(half=65)),
                             (-2, "head_dim 100", dict(D=100, half=8)), (-2, "dtype 5", dict(dtype=5)),
                             (-1, "slots with v", dict(k_out=None)), (-1, "slots with v", dict(slots=16)),
                             (-1, "multiples of 8", dict(q_st=4)), (-1, "16-byte", dict(q_out=24))]:
        got, said = _rc("fs_rope", rope(), **change)
        assert (got, text in said) == (rc, True), (change, got, said)


def test_frequencies_refuse():
    for kw in (dict(rotary_dim=7), dict(rotary_dim=0), dict(base=-1.0), dict(scaling="other"),
               dict(scaling="yarn", factor=4.0), dict(scaling="linear", factor=0.0),
               dict(scaling="llama3", original_length=100, low_freq_factor=4.0, high_freq_factor=4.0)):
        with pytest.raises(ValueError):
            fa.rope_frequencies(**{"rotary_dim": 64, "device": "cpu", **kw})


def test_frequencies_plain_and_linear():
    inv, f = fa.rope_frequencies(128, base=500000.0, device="cpu")
    assert f == 1.0 and inv.dtype == torch.float64 and inv.shape == (64,)
    assert all(math.isclose(inv[i].item(), 500000.0 ** (-2 * i / 128), rel_tol=1e-14) for i in range(64))
    lin, _ = fa.rope_frequencies(128, base=500000.0, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(lin, inv / 4.0)


@pytest.mark.parametrize("scaling,extra", [
    ("linear", {}), ("dynamic", {}), ("llama3", dict(low_freq_factor=1.0, high_freq_factor=4.0)),
    ("yarn", dict(beta_fast=32.0, beta_slow=1.0))])
@pytest.mark.parametrize("head_dim,base", [(128, 500000.0), (64, 10000.0)])
def test_frequencies_agree_with_transformers(scaling, extra, head_dim, base):
    """fp32 there: 2^-24 per operation, about ten of them on the way."""
    pytest.importorskip("transformers")
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    factor, original, length = 8.0, 4096, 20000
    rope = {"rope_type": scaling, "factor": factor, "original_max_position_embeddings": original,
            "rope_theta": base, **extra}
    cfg = LlamaConfig(hidden_size=4 * head_dim, num_attention_heads=4, head_dim=head_dim,
                      max_position_embeddings=original, rope_parameters=rope)
    want, want_factor = ROPE_INIT_FUNCTIONS[scaling](cfg, "cpu", seq_len=length)
    name = "ntk" if scaling == "dynamic" else scaling
    got, got_factor = fa.rope_frequencies(head_dim, base=base, scaling=name, factor=factor, original_length=original,
                                          length=length, device="cpu", **extra)
    assert math.isclose(got_factor, want_factor, rel_tol=1e-6)
    assert torch.allclose(got.float(), want, rtol=16 * 2.0 ** -24 * math.log(base) * 2, atol=0)


def _paged_bytes(T, B, max_new=0, Hq=32, Hk=8, D=128):
    a = _lib.PagedAttnArgs(dtype=1, B=B, T=T, Hq=Hq, Hk=Hk, D=D, P=64, page_size=64, max_new=max_new)
    return _lib.load().fs_paged_attn_work_bytes(ctypes.byref(a))


@pytest.mark.parametrize("Hq,Hk,D", [(32, 8, 128), (28, 4, 64), (4, 1, 128), (32, 32, 64)])
def test_workspaces_never_fall(Hq, Hk, D):
    """One sized for the largest step serves every smaller one."""
    sizes = sorted({n + d for n in (1, 8, 32, 33, 64, 256, 4096, 100000) for d in (-1, 0, 1) if n + d > 0})
    for B in (1, 8, 256, 4096):
        for m in (0, 1, 8, 100):
            n = [_paged_bytes(T, B, m, Hq, Hk, D) for T in sizes]
            assert n == sorted(n) and n[0] > 0
    for T in (1, 64, 5000):
        n = [_paged_bytes(T, B, 1, Hq, Hk, D) for B in range(1, 4097, 13)]
        assert n == sorted(n)
        n = [_paged_bytes(T, 16, m, Hq, Hk, D) for m in [*range(1, 200), 0]]
        assert n == sorted(n)
    lib = _lib.load()
    n = [lib.fs_window_attn_work_bytes(ctypes.byref(_lib.WindowAttnArgs(dtype=1, B=2, Hq=Hq, Hk=Hk, Lq=L, Lk=L, D=D, window=100)))
         for L in sizes]
    assert n == sorted(n) and n[0] > 0


@pytest.mark.skipif(HIPCC is None, reason="hipcc is not installed")
def test_paged_attention_spills_no_vector_registers(tmp_path):
    """many_kernel's loop holds all that 256 registers can; a spilled one cost it a quarter of its rate."""
    asm = _compile(CSRC / "paged.hip", tmp_path / "paged.s")
    spills = {}
    for meta in asm.split("  - .agpr_count:")[1:]:
        spills[re.search(r"\.name: +(\S+)", meta)[1]] = int(re.search(r"\.vgpr_spill_count: +(\d+)", meta)[1])
    assert sum("many_kernel" in n for n in spills) == sum("few_kernel" in n for n in spills) == 8
    assert {n: s for n, s in spills.items() if s} == {}
