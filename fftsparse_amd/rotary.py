"""Rotary positions on a gfx950 kernel: frequencies (plain or scaled for long
contexts), the rotation of queries and keys, and the same pass writing keys and
values into a paged cache.

``rope_pool`` rotates with the cos / sin rows that a model formed, bit for bit as
the model would; here the angles are formed in the kernel from positions and
frequencies, for any batch of tokens, half or interleaved pairs, and part of the
head.  No counterpart in the reference, which takes the model's embedding
(eval/LongBench/pred.py:195).  Inference only.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from ._lib import RopeArgs
from .paged import _caches, _inference_only, _ints, _rows, _written


def rope_frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                     original_length: int | None = None, length: int | None = None, low_freq_factor: float = 1.0,
                     high_freq_factor: float = 4.0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                     attention_factor: float | None = None, device="cuda") -> tuple[torch.Tensor, float]:
    """(inv_freq float64 [rotary_dim / 2], attention_factor) for ``rope`` and ``rope_cache``.

    inv_freq[i] = base^(-2 i / rotary_dim), then by ``scaling``:

    - None: as it is;
    - "linear": / factor;
    - "ntk": base * (factor length / original_length - factor + 1)^(R / (R - 2)) as the base, once ``length`` (the
      longest position in use) is past ``original_length``;
    - "llama3": / factor where a turn takes more than original_length / low_freq_factor tokens, as it is below
      original_length / high_freq_factor, blended linearly in the number of turns between;
    - "yarn": / factor for dims that make fewer than ``beta_slow`` turns over ``original_length``, as it is for more
      than ``beta_fast``, a linear ramp over the dims between; attention_factor 0.1 ln(factor) + 1.

    ``attention_factor`` (default 1, "yarn" its own) multiplies cos and sin."""
    R = int(rotary_dim)
    if R < 2 or R % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if not base > 0 or not factor > 0:
        raise ValueError(f"base {base} and factor {factor} must be positive")
    if scaling not in (None, "linear", "ntk", "llama3", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if scaling in ("ntk", "llama3", "yarn") and not original_length:
        raise ValueError(f"scaling {scaling!r} needs original_length")
    i = torch.arange(R // 2, dtype=torch.float64)
    if scaling == "ntk" and R > 2:
        n = max(int(length or original_length), original_length)
        base = base * (factor * n / original_length - (factor - 1.0)) ** (R / (R - 2))
    inv = float(base) ** (-2.0 * i / R)
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "llama3":
        if not high_freq_factor > low_freq_factor:
            raise ValueError("high_freq_factor must be above low_freq_factor")
        turns = original_length * inv / (2.0 * math.pi)
        keep = ((turns - low_freq_factor) / (high_freq_factor - low_freq_factor)).clamp(0.0, 1.0)
        inv = inv * (keep + (1.0 - keep) / factor)
    elif scaling == "yarn":
        def dim_of(turns):
            return R * math.log(original_length / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        low, high = max(math.floor(dim_of(beta_fast)), 0), min(math.ceil(dim_of(beta_slow)), R - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        inv = inv * (1.0 - ramp) + inv / factor * ramp
        if attention_factor is None:
            attention_factor = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    return inv.to(device), 1.0 if attention_factor is None else float(attention_factor)


def _common(name, q, k, positions, inv_freq):
    q, qs = _rows(q, "q")
    k, ks = _rows(k, "k")
    T, Hq, D = q.shape
    if k.shape[0] != T or k.shape[2] != D or not Hq or not k.shape[1] or not D:
        raise ValueError(f"query {tuple(q.shape)} and key {tuple(k.shape)} shapes do not match")
    if q.dtype != k.dtype or q.dtype not in _lib.FS_DTYPE:
        raise TypeError(f"unsupported dtypes {q.dtype}, {k.dtype}")
    _ints(positions, "positions", (T,), (torch.int32, torch.int64))
    if inv_freq.dim() != 1 or not inv_freq.numel() or not inv_freq.is_floating_point() or 2 * inv_freq.numel() > D:
        raise ValueError(f"inv_freq must hold half of at most {D} rotated dims, got {inv_freq.dtype} "
                         f"{tuple(inv_freq.shape)}")
    _inference_only(name, q, k)
    if inv_freq.dtype != torch.float64 or not inv_freq.is_contiguous():
        inv_freq = inv_freq.to(torch.float64).contiguous()
    return q, qs, k, ks, inv_freq


def _out(out, name, like):
    """The given output (checked) or a new one, and its strides."""
    if out is None:
        T, H, D = like.shape
        return like.new_empty((T, H, D)), (H * D, D)
    return out, _written(out, name, like.shape, like.dtype)


def _args(q, qs, k, ks, q_out, os_, positions, inv_freq, attention_factor, interleaved) -> RopeArgs:
    return RopeArgs(q=q.data_ptr(), q_st=qs[0], q_sh=qs[1], k=k.data_ptr(), k_st=ks[0], k_sh=ks[1],
                    positions=positions.data_ptr(), inv_freq=inv_freq.data_ptr(),
                    attention_factor=float(attention_factor), pos_bytes=positions.element_size(),
                    half=inv_freq.numel(), interleaved=int(bool(interleaved)), dtype=_lib.FS_DTYPE[q.dtype],
                    T=q.shape[0], Hq=q.shape[1], Hk=k.shape[1], D=q.shape[2],
                    q_out=q_out.data_ptr(), qo_st=os_[0], qo_sh=os_[1])


def rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *,
         attention_factor: float = 1.0, interleaved: bool = False, q_out: torch.Tensor | None = None,
         k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotary embedding of q [T, Hq, D] and k [T, Hk, D] (strided views; bf16, f16 or f32) at ``positions``
    (int32 or int64 [T]): the first 2 len(inv_freq) dims of every head are rotated, in pairs (i, i + half) or,
    ``interleaved``, (2 i, 2 i + 1); the others are copied.  Angles in 64 bits, rounded once.  Returns (q_rot,
    k_rot); ``q_out`` / ``k_out`` may be q / k themselves.  Rows with a negative position are left as they were."""
    q, qs, k, ks, inv_freq = _common("rope", q, k, positions, inv_freq)
    q_out, os_ = _out(q_out, "q_out", q)
    k_out, st = _out(k_out, "k_out", k)
    dev = _lib.same_device(q, k, positions, inv_freq, q_out, k_out)
    if q.shape[0]:
        a = _args(q, qs, k, ks, q_out, os_, positions, inv_freq, attention_factor, interleaved)
        a.k_out, a.ko_st, a.ko_sh = k_out.data_ptr(), st[0], st[1]
        _lib.call("fs_rope", a, dev)
    return q_out, k_out


def rope_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
               k_cache: torch.Tensor, v_cache: torch.Tensor, inv_freq: torch.Tensor, *, attention_factor: float = 1.0,
               interleaved: bool = False, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """``rope`` of q and k, with the rotated keys and the values v [T, Hk, D] written to ``slots`` (int64 [T], from
    ``plan_step``: page * page_size + slot, all different) of ``k_cache`` / ``v_cache`` [pages, page_size, Hk, D].
    Returns q_rot.  A slot outside the cache (-1: none) is not written; a row with a negative position is left as it
    was, in the cache too."""
    q, qs, k, ks, inv_freq = _common("rope_cache", q, k, positions, inv_freq)
    v, vs = _rows(v, "v")
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"value {v.dtype} {tuple(v.shape)} must be like key {k.dtype} {tuple(k.shape)}")
    _ints(slots, "slots", (q.shape[0],), (torch.int64,))
    shape, kc, vc = _caches(k_cache, v_cache, q.dtype, k.shape[1], k.shape[2])
    _inference_only("rope_cache", v, k_cache, v_cache)
    q_out, os_ = _out(q_out, "q_out", q)
    dev = _lib.same_device(q, k, v, positions, slots, k_cache, v_cache, inv_freq, q_out)
    if q.shape[0]:
        a = _args(q, qs, k, ks, q_out, os_, positions, inv_freq, attention_factor, interleaved)
        a.v, a.v_st, a.v_sh, a.slots = v.data_ptr(), vs[0], vs[1], slots.data_ptr()
        a.k_cache, a.kc_sp, a.kc_ss, a.kc_sh = k_cache.data_ptr(), kc[0], kc[1], kc[2]
        a.v_cache, a.vc_sp, a.vc_ss, a.vc_sh = v_cache.data_ptr(), vc[0], vc[1], vc[2]
        a.num_pages, a.page_size = shape[0], shape[1]
        _lib.call("fs_rope", a, dev)
    return q_out
