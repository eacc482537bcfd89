"""Drafted tokens as trees, over a paged cache: several guesses of how each request goes on, verified in one step.

A step in which a request's new tokens are a tree: the first one is the token that
the model chose last, every other one a guess of what follows its parent, named
by ``parents`` (int32 [T], the index within the request of the token that row t's
follows, below its own; -1: none)::

    plan = plan_step(block_table, seq_lens, new_lens, ...)        # as ever: places for all of them
    tree = plan_tree(parents, plan.cu_lens, plan.seq_lens, max_new=16)
    for layer in layers:
        q = rope_cache(q, k, v, tree.positions, plan.slots, k_cache, v_cache, inv_freq)
        out = tree_attention(q, k_cache, v_cache, block_table, plan.cu_lens, plan.seq_lens, tree.mask, max_new=16)
    chosen = ...                                                  # what the model takes after each of them
    acc = accept_tree(parents, tokens, chosen, plan.cu_lens, max_new=16)
    move_kept(k_caches, v_caches, block_table, plan.cu_lens, plan.seq_lens, acc.kept)
    back = plan_step(block_table, plan.seq_lens, acc.dropped, free_pages, plan.free_count, ...)   # the others' pages

The lengths stay on the GPU throughout, so all of it can be captured in a graph.
No counterpart in the reference.  Inference only.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Sequence

import torch

from . import _lib
from ._lib import CacheMoveArgs, TreeAcceptArgs, TreePlanArgs
from .paged import _apart, _attend, _inference_only, _ints, _strides, _table, _window, _written

MOST = 1024                    # tokens of a request's tree


def _rows_of(cu_lens: torch.Tensor) -> int:
    if cu_lens.dim() != 1 or cu_lens.shape[0] < 2:
        raise ValueError(f"cu_lens must be an int32 [requests + 1] tensor, got {cu_lens.dtype} {tuple(cu_lens.shape)}")
    _ints(cu_lens, "cu_lens", cu_lens.shape)
    return cu_lens.shape[0] - 1


def _most(max_new) -> int:
    if not 1 <= int(max_new) <= MOST:
        raise ValueError(f"max_new must be 1 to {MOST}, got {max_new}")
    return int(max_new)


def _tokens_by_row(t: torch.Tensor, name: str) -> int:
    if t.dim() != 1:
        raise ValueError(f"{name} must be a [T] tensor, got shape {tuple(t.shape)}")
    _ints(t, name, t.shape)
    return t.shape[0]


@dataclass
class TreePlan:
    """What ``plan_tree`` forms on the GPU."""
    positions: torch.Tensor    # int32 [T]: position of each new token in its request, -1 for rows that no request has
    mask: torch.Tensor         # int64 [T, words]: bit j % 64 of word j / 64: token j of the request is seen


def plan_tree(parents: torch.Tensor, cu_lens: torch.Tensor, seq_lens: torch.Tensor, *, max_new: int,
              window: int | None = None, sinks: int = 0, out: TreePlan | None = None) -> TreePlan:
    """Positions of the new tokens of a batch of trees, and the masks that ``tree_attention`` reads (one launch).

    ``parents`` int32 [T]; ``cu_lens`` int32 [B + 1] and ``seq_lens`` int32 [B] as
    ``plan_step`` gives them (new tokens included).  A token's position is that of
    the token it follows, and one; it sees its ancestors and itself.  A parent that is
    not an index below the token's own counts as none.  ``max_new``: at least the most
    new tokens that one request has, up to 1024; a request's tokens past it (rounded up to
    64) get position -1 and an empty mask.

    For attention under a ``window`` (and ``sinks``) give the same here: a token then sees
    of its ancestors those less than ``window`` positions before it and those at the first
    ``sinks`` positions, as if it had been decoded after them one by one.  Without it a token
    sees all of its ancestors, which is the same for trees no deeper than the window.
    ``out``: a former result to write into, whose tensors are not this call's inputs."""
    T = _tokens_by_row(parents, "parents")
    B = _rows_of(cu_lens)
    _ints(seq_lens, "seq_lens", (B,))
    words = -(-_most(max_new) // 64)
    window, sinks = _window(window, sinks)
    dev = _lib.same_device(parents, cu_lens, seq_lens)
    if out is None:
        out = TreePlan(parents.new_empty(T), parents.new_empty((T, words), dtype=torch.int64))
    else:
        _lib.same_device(parents, _ints(out.positions, "out.positions", (T,)),
                         _ints(out.mask, "out.mask", (T, words), (torch.int64,)))
        _apart((out.positions, out.mask), (parents, cu_lens, seq_lens), "they are read while it is written")
    if T:
        _lib.call("fs_tree_plan", TreePlanArgs(
            parents=parents.data_ptr(), cu_lens=cu_lens.data_ptr(), seq_lens=seq_lens.data_ptr(), B=B, T=T, words=words,
            window=window, sinks=sinks, positions=out.positions.data_ptr(), mask=out.mask.data_ptr()), dev)
    return out


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                   cu_lens: torch.Tensor, seq_lens: torch.Tensor, mask: torch.Tensor, *,
                   positions: torch.Tensor | None = None, max_new: int | None = None, window: int | None = None,
                   sinks: int = 0, softmax_scale: float | None = None, k_scale: torch.Tensor | None = None,
                   v_scale: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``paged_attention`` of new tokens that are not a chain: each sees the tokens of its request before the new ones,
    and of the new ones those that its row of ``mask`` names.

    ``mask`` int64 [T, words]: bit j % 64 of word j / 64 of row t: the j-th new token of
    row t's request (a tree's ancestors and the token itself, from ``plan_tree``, or any
    other set; new tokens past the words are seen by none).  With ``window`` the
    tokens before the new ones are restricted to the last ``window`` up to the row's
    position (``positions`` int32 [T], taken within those of the request's new tokens) and the
    first ``sinks``; among the new ones the mask alone decides: form it with
    ``plan_tree(..., window=, sinks=)`` of the same numbers where trees are deeper than the window.  A row that sees no
    token is 0.  Everything else as in ``paged_attention``, 8-bit caches too: the new
    tokens' keys and values are in the cache, all of them (a value that is not finite may
    reach rows of its request whose mask leaves it out)."""
    return _attend("tree_attention", q, k_cache, v_cache, block_table, cu_lens, seq_lens, mask, positions, max_new, window,
                   sinks, softmax_scale, k_scale, v_scale, out)


@dataclass
class Accepted:
    """What ``accept_tree`` forms on the GPU."""
    kept: torch.Tensor         # int32 [T]: row cu_lens[b] + i: index of request b's i-th kept token, -1 past them
    kept_lens: torch.Tensor    # int32 [B]: how many are kept
    dropped: torch.Tensor      # int32 [B]: kept_lens less the new tokens: plan_step's new_lens that takes the others back
    next_tokens: torch.Tensor  # [B], as chosen: what the model takes after the last kept one, -1 without new tokens


def accept_tree(parents: torch.Tensor, tokens: torch.Tensor, chosen: torch.Tensor, cu_lens: torch.Tensor, *, max_new: int,
                out: Accepted | None = None) -> Accepted:
    """The path of each request's tree that the model agrees with (one launch).

    ``tokens`` (int32 or int64 [T]) are the new tokens, ``chosen`` (like it) what the
    model takes after each of them: its most likely token, or one drawn.  A
    request's first new token is kept; another one if its parent is and the parent's
    chosen token is this one (or the token is negative: given, not drafted), the
    lowest of several such.  ``max_new`` as in ``plan_tree``; a request's tokens past it are
    not kept.  ``out``: a former result to write into, whose tensors are not this call's inputs."""
    T = _tokens_by_row(parents, "parents")
    B = _rows_of(cu_lens)
    kinds = (torch.int32, torch.int64)
    _ints(tokens, "tokens", (T,), kinds)
    _ints(chosen, "chosen", (T,), (tokens.dtype,))
    most = _most(max_new)
    dev = _lib.same_device(parents, tokens, chosen, cu_lens)
    if out is None:
        kept, kept_lens, dropped = parents.new_empty(T + 2 * B).split_with_sizes((T, B, B))
        out = Accepted(kept, kept_lens, dropped, chosen.new_empty(B))
    else:
        _lib.same_device(parents, _ints(out.kept, "out.kept", (T,)), _ints(out.kept_lens, "out.kept_lens", (B,)),
                         _ints(out.dropped, "out.dropped", (B,)),
                         _ints(out.next_tokens, "out.next_tokens", (B,), (chosen.dtype,)))
        _apart((out.kept, out.kept_lens, out.dropped, out.next_tokens), (parents, tokens, chosen, cu_lens),
               "they are read while it is written")
    _lib.call("fs_tree_accept", TreeAcceptArgs(
        parents=parents.data_ptr(), tokens=tokens.data_ptr(), chosen=chosen.data_ptr(), cu_lens=cu_lens.data_ptr(),
        token_bytes=tokens.element_size(), B=B, T=T, most=most, kept=out.kept.data_ptr(), kept_lens=out.kept_lens.data_ptr(),
        dropped=out.dropped.data_ptr(), next_tokens=out.next_tokens.data_ptr()), dev)
    return out


_CACHE_DTYPES = (torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn)


def _layers(caches, name: str, shape, dtype):
    """The caches of one layer [pages, page_size, Hk, D], of several in a tensor [layers, ...], or in a sequence of the
    first: their number, addresses (None: apart by a stride), address of the first, strides (layer, page, slot, head) in
    elements, and the tensors."""
    if isinstance(caches, torch.Tensor):
        if caches.dim() == len(shape):
            return 1, None, caches.data_ptr(), (0, *_written(caches, name, shape, dtype)), (caches,)
        whole, st, size = caches.shape, _strides(caches), caches.element_size()
        if whole[1:] != shape or caches.dtype != dtype:
            raise ValueError(f"{name} must be a [layers, {', '.join(map(str, shape))}] {dtype} tensor, got {caches.dtype} "
                             f"{tuple(whole)}")
        p, (s0, s1, s2, s3, sd) = caches.data_ptr(), st
        if (sd != 1 and shape[3] > 1) or (p | (s0 | s1 | s2 | s3) * size) & 15 or (
                0 in st and any(m > 1 and s == 0 for s, m in zip(st, whole))):
            raise ValueError(f"{name} must have d contiguous, the other strides multiples of 16 bytes, 16-byte alignment and no "
                             f"broadcast dimension, got strides {caches.stride()}")
        return whole[0], None, p, st, (caches,)
    if not len(caches):
        raise ValueError(f"{name} holds no layer")
    st = _written(caches[0], name, shape, dtype)
    like, ptrs = caches[0].stride(), []
    for t in caches:
        p = t.data_ptr()
        if t.dtype != dtype or t.shape != shape or t.stride() != like or p & 15:
            raise ValueError(f"{name}: the layers' caches must be of one shape, type and layout, 16-byte aligned")
        ptrs.append(p)
    return len(ptrs), ptrs, 0, (0, *st), caches


def move_kept(k_cache: torch.Tensor | Sequence[torch.Tensor], v_cache: torch.Tensor | Sequence[torch.Tensor],
              block_table: torch.Tensor, cu_lens: torch.Tensor, seq_lens: torch.Tensor, kept: torch.Tensor) -> None:
    """The kept tokens' keys and values to where they belong in the cache, in place: request b's i-th kept token to the
    place of its i-th new token.

    ``k_cache`` / ``v_cache``: one layer's caches [pages, page_size, Hk, D], those of
    several layers in one tensor [layers, pages, page_size, Hk, D], or a sequence of the
    first (all of one layout; bf16, f16, f32 or ``torch.float8_e4m3fn``; rows of a
    multiple of 16 bytes).  Each cache is moved by itself, so all of them have to be apart:
    one that several layers read is named once (caches that share storage are refused; views of
    one storage that lie between each other's rows are apart).  ``seq_lens`` int32 [B]: new tokens included, as for the step's
    attention; ``kept`` int32 [T] from ``accept_tree``.  Up to 64 layers go in one
    launch.  Tokens without a page stay as they are; of a request the first 1024 are
    looked at."""
    one = k_cache if isinstance(k_cache, torch.Tensor) else k_cache[0] if len(k_cache) else None
    if one is None or one.dim() not in (4, 5) or (one.dim() == 5 and one is not k_cache) or not one.numel():
        raise ValueError("k_cache must be [pages, page_size, Hk, D] or [layers, pages, page_size, Hk, D], or a sequence of the first")
    shape, dtype = one.shape[-4:], one.dtype
    if dtype not in _CACHE_DTYPES:
        raise TypeError(f"unsupported cache type {dtype}")
    pages, ps, Hk, D = shape
    n, kp, k0, ks, kt = _layers(k_cache, "k_cache", shape, dtype)
    if (isinstance(v_cache, torch.Tensor) and one is k_cache and v_cache.dtype == dtype and v_cache.shape == k_cache.shape
            and v_cache.stride() == k_cache.stride() and not v_cache.data_ptr() & 15):
        m, vp, v0, vs, vt = n, None, v_cache.data_ptr(), ks, (v_cache,)    # laid out as k_cache is
    else:
        m, vp, v0, vs, vt = _layers(v_cache, "v_cache", shape, dtype)
    if n != m or (kp is None) != (vp is None):
        raise ValueError(f"{n} layers of keys and {m} of values, or not in one form")
    B, P, t_sb = _table(block_table)
    _ints(cu_lens, "cu_lens", (B + 1,))
    _ints(seq_lens, "seq_lens", (B,))
    T = _tokens_by_row(kept, "kept")
    _inference_only("move_kept", *kt, *vt)
    dev = _lib.same_device(block_table, cu_lens, seq_lens, kept, *kt, *vt)
    if not T:
        return
    args = CacheMoveArgs(
        k_cache=k0, k_sl=ks[0], k_sp=ks[1], k_ss=ks[2], k_sh=ks[3], v_cache=v0, v_sl=vs[0], v_sp=vs[1], v_ss=vs[2], v_sh=vs[3],
        block_table=block_table.data_ptr(), t_sb=t_sb, cu_lens=cu_lens.data_ptr(), seq_lens=seq_lens.data_ptr(),
        kept=kept.data_ptr(), layers=n, B=B, T=T, Hk=Hk, D=D, P=P, page_size=ps, elem_bytes=one.element_size(),
        num_pages=pages)
    if kp is not None:
        array = _lib.c_void_p * n
        args.k_caches, args.v_caches = array(*kp), array(*vp)
    _lib.call("fs_cache_move", args, dev)
