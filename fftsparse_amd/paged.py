"""Serving over a paged cache: what follows the prefill, on gfx950 kernels.

One decoding or chunk step of a batch of requests, whose lengths stay on the
GPU throughout (no host synchronisation, so a step can be captured in a graph)::

    plan = plan_step(block_table, seq_lens, new_lens, free_pages, free_count, page_size=64, num_tokens=T)
    for layer in layers:                      # q, k, v [T, H, D]: the new tokens of all requests, one after another
        q = rope_cache(q, k, v, plan.positions, plan.slots, k_cache, v_cache, inv_freq)
        out = paged_attention(q, k_cache, v_cache, block_table, plan.cu_lens, plan.seq_lens, max_new=1)

A cache is a [pages, page_size, Hk, D] view for keys and one for values (any
strides that are multiples of 8 elements with d contiguous, e.g. [pages, Hk,
page_size, D] storage transposed).  Token t of request b is in slot t %
page_size of page block_table[b, t // page_size].

A cache of ``torch.float8_e4m3fn`` with one scale for each KV head (``k_scale``,
``v_scale``, float32 [Hk]: a number x stands for x * scale) takes half the place
and, in decoding, about half the time.  Requests whose new tokens are a tree of
drafts instead of a chain: ``fftsparse_amd.tree``.

``window_attention`` is the attention's sliding-window rule on contiguous
[B, H, L, D] tensors, beside ``block_sparse_attention``.  No counterpart in the
reference, which serves decoding from the model's own cache.  Inference only:
tensors that would need a gradient are refused.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import PagedAttnArgs, PlanArgs, WindowAttnArgs
from .attn import _check_layout

_INT32_MAX = 2 ** 31 - 1
E4M3 = torch.float8_e4m3fn


def _inference_only(name: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad() or on detached tensors")


def _strides(t: torch.Tensor):
    """Element strides, 0 for dimensions of size 1 (whose stride says nothing)."""
    st, shape = t.stride(), t.shape
    return [s if n > 1 else 0 for n, s in zip(shape, st)] if 1 in shape else st


def _aligned(t: torch.Tensor, st, eight: bool = False) -> bool:
    """Whether the kernels can read t as it is: d contiguous, 16-byte rows (for elements of 4 bytes: 32); eight: elements of
    one byte."""
    bits = (t.data_ptr() if eight else t.data_ptr() >> 1) if st[-1] == 1 else 1
    for s in st[:-1]:
        bits |= s
    return not bits & (15 if eight else 7)


def _rows(t: torch.Tensor, name: str):
    """[T, H, D] input, copied if its layout cannot be read, and its strides."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be a [T, H, D] tensor, got shape {tuple(t.shape)}")
    st = _strides(t)
    if not _aligned(t, st):
        t = t.contiguous()
        st = _strides(t)
    return t, st


def _written(t: torch.Tensor, name: str, shape, dtype):
    """Strides of a tensor that the kernels read or write as it is, or not at all."""
    if t.shape != shape or t.dtype != dtype:
        raise ValueError(f"{name} must be a {list(shape)} {dtype} tensor, got {t.dtype} {tuple(t.shape)}")
    st = _strides(t)
    if not _aligned(t, st, dtype is E4M3) or (0 in st and any(n > 1 and s == 0 for n, s in zip(shape, st))):
        if t.numel():
            raise ValueError(f"{name} must have d contiguous, strides that are multiples of {16 if dtype is E4M3 else 8} "
                             f"elements and 16-byte alignment, and no broadcast dimension, got strides {t.stride()}")
    return st


def _ints(t: torch.Tensor, name: str, shape, dtypes=(torch.int32,)) -> torch.Tensor:
    if t.shape != shape or t.dtype not in dtypes or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {list(shape)} tensor of {' or '.join(map(str, dtypes))}, got "
                         f"{t.dtype} {tuple(t.shape)}")
    return t


def _table(t: torch.Tensor):
    """[B, P] block table -> B, P, row stride."""
    shape = t.shape
    if len(shape) != 2 or t.dtype != torch.int32 or 0 in shape or (shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"block_table must be an int32 [requests, pages] tensor with contiguous rows, got {t.dtype} "
                         f"{tuple(shape)}")
    B, P = shape
    if B > 1 and t.stride(0) < P:
        raise ValueError("block_table's rows overlap")
    return B, P, t.stride(0) if B > 1 else P


def _caches(k: torch.Tensor, v: torch.Tensor, dtype, Hk=None, D=None):
    """Shape and strides of k_cache and v_cache, views that the kernels read and write as they are."""
    shape = k.shape
    if len(shape) != 4 or not k.numel():
        raise ValueError(f"k_cache must be a [pages, page_size, Hk, D] tensor, got shape {tuple(shape)}")
    want = (shape[0], shape[1], shape[2] if Hk is None else Hk, shape[3] if D is None else D)
    ks = _written(k, "k_cache", want, dtype)
    if v.dtype == dtype and v.shape == shape and v.stride() == k.stride() and not v.data_ptr() & 15:
        return want, ks, ks                        # laid out as k_cache is
    return want, ks, _written(v, "v_cache", want, dtype)


def _scales(k_scale, v_scale, dtype, Hk: int) -> None:
    """Scales come with caches in 8 bits, and only then."""
    if dtype is not E4M3:
        raise ValueError(f"k_scale and v_scale go with caches of {E4M3}, got {dtype}")
    if k_scale is None or v_scale is None:
        raise ValueError(f"caches of {E4M3} need k_scale and v_scale")
    for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        if t.shape != (Hk,) or t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float32 tensor of {Hk} scales, one for each KV head, got "
                             f"{t.dtype} {tuple(t.shape)}")


def _span(t: torch.Tensor) -> tuple[int, int]:
    """From a tensor's first byte to behind its last one."""
    p, n = t.data_ptr(), t.numel()
    if n and not t.is_contiguous():
        n = 1 + sum((m - 1) * s for m, s in zip(t.shape, t.stride()))
    return p, p + n * t.element_size()


def _apart(outs, ins, what: str) -> None:
    """Refuses outputs that share storage with each other, or with what is read while they are written."""
    read, written = [_span(x) for x in ins], [_span(x) for x in outs]
    if any(lo < end and start < hi for lo, hi in written for start, end in read):
        raise ValueError(f"out shares storage with an input: {what}")
    written.sort()
    if any(hi > start for (_, hi), (start, _) in zip(written, written[1:])):
        raise ValueError("out's tensors share storage with each other")


@dataclass
class StepPlan:
    """What ``plan_step`` forms on the GPU for one step."""
    cu_lens: torch.Tensor      # int32 [B + 1]: request b's new tokens are rows cu_lens[b] .. cu_lens[b + 1] - 1
    seq_lens: torch.Tensor     # int32 [B]: tokens of each request after the step
    positions: torch.Tensor    # int32 [T]: position of each new token in its request, -1 past the last one
    slots: torch.Tensor        # int64 [T]: page * page_size + slot of each new token, -1 for none
    free_count: torch.Tensor   # int32 [1]: free pages after the step
    lacking: torch.Tensor      # int32 [1]: new tokens that found no page (0: the step can be taken)


def plan_step(block_table: torch.Tensor, seq_lens: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor,
              free_count: torch.Tensor, *, page_size: int, num_tokens: int, out: StepPlan | None = None) -> StepPlan:
    """Block tables and slot maps of one step, from the requests' lengths (one launch).

    ``block_table`` int32 [B, P], ``seq_lens`` int32 [B] (tokens in the cache),
    ``new_lens`` int32 [B]: tokens each request is given; a negative number takes
    that many of its last tokens back (-seq_lens: the request is finished) and
    returns the pages they leave.  ``free_pages`` int32 [F] is the stack of free
    pages, F the number of pages of the cache, ``free_count`` int32 [1] its height.
    Pages given back are pushed first, then those needed popped, in the requests'
    order.  ``num_tokens`` is the number of rows of the token arrays: at least the
    sum of the positive ``new_lens`` (a fixed size serves a captured graph; the
    rows behind the last request get position and slot -1).

    ``block_table`` and ``free_pages`` are updated in place; ``seq_lens`` and
    ``free_count`` are not: take them from the result for the next step.  A
    step whose ``lacking`` is not 0 is undone by not using its result.
    ``out``: a former result to write into, whose tensors are not this call's inputs."""
    t = block_table
    B, P, t_sb = _table(t)
    _ints(seq_lens, "seq_lens", (B,))
    _ints(new_lens, "new_lens", (B,))
    if free_pages.dim() != 1 or not free_pages.numel():
        raise ValueError("free_pages must hold an entry for every page of the cache")
    _ints(free_pages, "free_pages", free_pages.shape)
    _ints(free_count, "free_count", (1,))
    page_size, num_tokens = int(page_size), int(num_tokens)
    if page_size < 1 or not 0 <= num_tokens <= _INT32_MAX or P * page_size > _INT32_MAX:
        raise ValueError(f"page_size {page_size} and num_tokens {num_tokens} out of range for a table of {P} pages")
    dev = _lib.same_device(t, seq_lens, new_lens, free_pages, free_count)
    if out is None:
        cu_lens, after, positions, count, lacking = t.new_empty(2 * B + 3 + num_tokens).split_with_sizes(
            (B + 1, B, num_tokens, 1, 1))
        out = StepPlan(cu_lens, after, positions, torch.empty(num_tokens, dtype=torch.int64, device=dev), count, lacking)
    else:
        outs = [_ints(out.cu_lens, "out.cu_lens", (B + 1,)), _ints(out.seq_lens, "out.seq_lens", (B,)),
                _ints(out.positions, "out.positions", (num_tokens,)),
                _ints(out.slots, "out.slots", (num_tokens,), (torch.int64,)),
                _ints(out.free_count, "out.free_count", (1,)), _ints(out.lacking, "out.lacking", (1,))]
        _lib.same_device(t, *outs)
        read = [_span(x) for x in (seq_lens, new_lens, free_pages, free_count)]
        read.append((t.data_ptr(), t.data_ptr() + 4 * ((B - 1) * t_sb + P)))
        if any(lo < end and start < hi for lo, hi in map(_span, outs) for start, end in read):
            raise ValueError("out shares storage with an input of the step: the lengths and the free count of a step "
                             "are read while its result is written")
    _lib.call("fs_plan", PlanArgs(
        block_table=t.data_ptr(), t_sb=t_sb, seq_lens=seq_lens.data_ptr(),
        new_lens=new_lens.data_ptr(), free_pages=free_pages.data_ptr(), free_count=free_count.data_ptr(), B=B, P=P,
        F=free_pages.numel(), page_size=page_size, T=num_tokens, cu_lens=out.cu_lens.data_ptr(),
        seq_lens_out=out.seq_lens.data_ptr(), positions=out.positions.data_ptr() or 16,
        slots=out.slots.data_ptr() or 16, free_count_out=out.free_count.data_ptr(), lacking=out.lacking.data_ptr()),
        dev)
    return out


def _window(window, sinks) -> tuple[int, int]:
    if window is not None and not 1 <= int(window) <= _INT32_MAX:
        raise ValueError(f"window must be at least 1, or None, got {window}")
    if not 0 <= int(sinks) <= _INT32_MAX:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    return int(window or 0), int(sinks)


def _scale(scale, D: int) -> float:
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 <= scale < math.inf:
        raise ValueError(f"softmax_scale must be finite and not negative, got {scale}")
    return scale


def _attn_dtype(q, k, v) -> None:
    dt = q.dtype
    if (dt != torch.bfloat16 and dt != torch.float16) or k.dtype != dt or v.dtype != dt:
        raise TypeError(f"expected bf16 or f16 tensors of one type, got {[t.dtype for t in (q, k, v)]}")


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    cu_lens: torch.Tensor, seq_lens: torch.Tensor, *, max_new: int | None = None,
                    window: int | None = None, sinks: int = 0, softmax_scale: float | None = None,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of the new tokens of a batch of requests over their paged caches.

    q [T, Hq, D] (bf16 / f16, D 64 or 128); ``k_cache`` / ``v_cache`` [pages,
    page_size, Hk, D] (page_size a multiple of 16 up to 4096) already hold the
    new tokens too; ``block_table`` int32 [B, P]; ``cu_lens`` int32 [B + 1]: request
    b's new tokens are rows cu_lens[b] .. cu_lens[b + 1] - 1 (none is allowed);
    ``seq_lens`` int32 [B]: its tokens, new ones included.  Returns [T, Hq, D].

    A token sees the tokens of its request up to itself; with ``window`` the last
    ``window`` of them (itself included) and the first ``sinks``.  Query head h
    reads KV head h // (Hq / Hk).  ``max_new``: the most new tokens that one
    request has, if the caller knows it (1 in a decoding step); the result is right
    for any value, the right one is faster.  Rows behind cu_lens[B] are left as
    they were (unset in a new tensor).  A page number outside the cache holds no
    token; a row that sees no token is 0.  Slots that no row sees may hold anything;
    a value of v that is not finite may reach rows of its request that do not see
    it.  Scores, maxima and sums are in 32 bits; the weights are rounded to the input
    type before the product with v (values up to 2^93).  ``out`` may be q.  Up to 4096
    requests of 2^26 tokens.

    Caches of ``torch.float8_e4m3fn`` need ``k_scale`` and ``v_scale`` (float32 [Hk],
    positive and finite): a number x of KV head h stands for x * scale[h].  It is
    taken exactly; queries and weights are not rounded further."""
    return _attend("paged_attention", q, k_cache, v_cache, block_table, cu_lens, seq_lens, None, None, max_new, window, sinks,
                   softmax_scale, k_scale, v_scale, out)


def _attend(name, q, k_cache, v_cache, block_table, cu_lens, seq_lens, mask, positions, max_new, window, sinks, softmax_scale,
            k_scale, v_scale, out):
    """``paged_attention``, and ``tree_attention`` (mask given)."""
    q, qs = _rows(q, "q")
    T, Hq, D = q.shape
    dt = k_cache.dtype
    if dt is not E4M3 or v_cache.dtype is not E4M3 or q.dtype not in (torch.bfloat16, torch.float16):
        _attn_dtype(q, k_cache, v_cache)
    (pages, ps, Hk, _), ks, vs = _caches(k_cache, v_cache, dt, D=D)
    scaled = dt is E4M3 or k_scale is not None or v_scale is not None
    if scaled:
        _scales(k_scale, v_scale, dt, Hk)
    if Hk == 0 or Hq % Hk or Hq == 0:
        raise ValueError(f"query heads {Hq} must be a multiple of key heads {Hk}")
    t = block_table
    B, P, t_sb = _table(t)
    _ints(cu_lens, "cu_lens", (B + 1,))
    _ints(seq_lens, "seq_lens", (B,))
    window, sinks = _window(window, sinks)
    scale = _scale(softmax_scale, D)
    if max_new is not None and int(max_new) < 1:
        raise ValueError(f"max_new must be at least 1, got {max_new}")
    more = (k_scale, v_scale) if scaled else ()
    if mask is not None:
        if mask.dim() != 2 or mask.shape[0] != T or not mask.shape[1] or mask.dtype != torch.int64 or not mask.is_contiguous():
            raise ValueError(f"mask must be a contiguous int64 [{T}, words] tensor, got {mask.dtype} {tuple(mask.shape)}")
        more += (mask,)
        if window:
            if positions is None:
                raise ValueError("a window over a tree needs the tokens' positions")
            more += (_ints(positions, "positions", (T,)),)
    _inference_only(name, q, k_cache, v_cache, *more)
    if out is None:
        dev = _lib.same_device(q, k_cache, v_cache, t, cu_lens, seq_lens, *more)
        out = q.new_empty((T, Hq, D))
        os_ = (Hq * D, D)
    else:
        os_ = _written(out, "out", (T, Hq, D), q.dtype)
        dev = _lib.same_device(q, k_cache, v_cache, t, cu_lens, seq_lens, out, *more)
        if more:
            _apart((out,), more, "masks, positions and scales are read until the last row is written")
    if T == 0:
        return out
    args = PagedAttnArgs(
        q=q.data_ptr(), q_st=qs[0], q_sh=qs[1], out=out.data_ptr(), o_st=os_[0], o_sh=os_[1],
        k_cache=k_cache.data_ptr(), k_sp=ks[0], k_ss=ks[1], k_sh=ks[2],
        v_cache=v_cache.data_ptr(), v_sp=vs[0], v_ss=vs[1], v_sh=vs[2],
        block_table=t.data_ptr(), t_sb=t_sb, cu_lens=cu_lens.data_ptr(),
        seq_lens=seq_lens.data_ptr(), dtype=_lib.FS_DTYPE[q.dtype], B=B, T=T, Hq=Hq, Hk=Hk, D=D, P=P, page_size=ps,
        num_pages=pages, max_new=0 if max_new is None else min(int(max_new), T), window=window, sinks=sinks,
        softmax_scale=scale)
    if scaled:
        args.k_scale, args.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
    if mask is not None:
        args.mask, args.mask_words = mask.data_ptr(), mask.shape[1]
        if window:
            args.positions = positions.data_ptr()
    work = q.new_empty(_lib.load().fs_paged_attn_work_bytes(ctypes.byref(args)), dtype=torch.uint8)
    args.work = work.data_ptr()
    _lib.call("fs_paged_attn", args, dev)
    return out


def window_attention(query_states: torch.Tensor, key_states: torch.Tensor, value_states: torch.Tensor, *,
                     window: int | None, sinks: int = 0, softmax_scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention with a sliding window and a few first tokens that stay visible.

    q [B,Hq,Lq,D], k/v [B,Hk,Lk,D] (bf16 / f16, D 64 or 128; strided views) ->
    [B, Lq, Hq, D], as ``block_sparse_attention`` returns it.  Query t is at
    position t + Lk - Lq and sees the last ``window`` tokens up to itself, itself
    included, and the first ``sinks``; window None: every token up to itself (dense
    causal attention; ``block_sparse_attention`` without lists is the faster one for
    short sequences and for 16384 tokens of few heads).  The mask is exact to the
    token.  A query before the first key sees nothing and gives 0.  Rounding as in
    ``paged_attention``."""
    q, k, v = (_check_layout(x) for x in (query_states, key_states, value_states))
    B, Hq, Lq, D = q.shape
    Hk, Lk = k.shape[1], k.shape[2]
    _attn_dtype(q, k, v)
    if v.shape != k.shape or k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"query {tuple(q.shape)}, key {tuple(k.shape)} and value {tuple(v.shape)} shapes do not match")
    if Hk == 0 or Hq == 0 or Hq % Hk:
        raise ValueError(f"query heads {Hq} must be a multiple of key heads {Hk}")
    if not (B and Lq and Lk):
        raise ValueError("empty sequence")
    window, sinks = _window(window, sinks)
    scale = _scale(softmax_scale, D)
    _inference_only("window_attention", q, k, v)
    if out is None:
        out = q.new_empty((B, Lq, Hq, D))
        os_ = (Lq * Hq * D, Hq * D, D)
    else:
        os_ = _written(out, "out", (B, Lq, Hq, D), q.dtype)
    qs, ks, vs = _strides(q), _strides(k), _strides(v)
    dev = _lib.same_device(q, k, v, out)
    args = WindowAttnArgs(
        q=q.data_ptr(), q_sb=qs[0], q_sh=qs[1], q_sl=qs[2], k=k.data_ptr(), k_sb=ks[0], k_sh=ks[1], k_sl=ks[2],
        v=v.data_ptr(), v_sb=vs[0], v_sh=vs[1], v_sl=vs[2], out=out.data_ptr(), o_sb=os_[0], o_sl=os_[1], o_sh=os_[2],
        dtype=_lib.FS_DTYPE[q.dtype], B=B, Hq=Hq, Hk=Hk, Lq=Lq, Lk=Lk, D=D, window=window, sinks=sinks,
        softmax_scale=scale)
    work = q.new_empty(_lib.load().fs_window_attn_work_bytes(ctypes.byref(args)), dtype=torch.uint8)
    args.work = work.data_ptr()
    _lib.call("fs_window_attn", args, dev)
    return out
