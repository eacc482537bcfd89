"""Plain 64-bit forms of the serving operators (``fftsparse_amd.paged``, ``fftsparse_amd.rotary``), on the CPU.

Written from the definitions: page tables with Python lists, rotations as complex
products, attention row by row over the tokens that a row sees."""
from __future__ import annotations

import math

import torch


def plan(table, seq_lens, new_lens, free_pages, free_count, page_size, num_tokens):
    """Lists in, a dict of lists out; rules as ``plan_step`` states them."""
    table, stack = [list(r) for r in table], list(free_pages)
    width, top = len(table[0]), min(max(free_count, 0), len(stack))
    pages = lambda n: min(-(-n // page_size), width)                      # noqa: E731
    held = [min(max(n, 0), width * page_size) for n in seq_lens]
    after = [max(h + d, 0) for h, d in zip(held, new_lens)]
    for row, h, a in zip(table, held, after):
        for i in range(pages(a), pages(h)):
            if top < len(stack):
                stack[top] = row[i]
                top += 1
    taken = top
    cu, positions, slots, lacking = [0], [], [], 0
    for row, h, a, d in zip(table, held, after, new_lens):
        room = pages(h)
        for i in range(pages(h), pages(a)):
            taken -= 1
            row[i] = stack[taken] if taken >= 0 else -1
            room += taken >= 0
        for p in range(h, h + max(d, 0)):
            i = p // page_size
            page = row[i] if i < width else -1
            positions.append(p)
            slots.append(page * page_size + p % page_size if page >= 0 else -1)
            lacking += p >= max(h, room * page_size)
        cu.append(cu[-1] + max(d, 0))
    pad = [-1] * max(0, num_tokens - len(positions))
    return dict(block_table=table, free_pages=stack, cu_lens=cu, seq_lens=after,
                positions=(positions + pad)[:num_tokens], slots=(slots + pad)[:num_tokens],
                free_count=[max(taken, 0)], lacking=[lacking])


def rotate(x, positions, inv_freq, factor=1.0, interleaved=False):
    """x [T, H, D] -> float64; the pairs of the first 2 len(inv_freq) dims turned by positions * inv_freq."""
    half = len(inv_freq)
    y = x.double().clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    angle = positions.double()[:, None] * inv_freq.double()
    z = torch.complex(y[..., a].contiguous(), y[..., b].contiguous()) * torch.polar(
        torch.full_like(angle, factor), angle)[:, None, :]
    y[..., a], y[..., b] = z.real, z.imag
    return y


def seen(p, length, window=None, sinks=0):
    """Tokens that the row at position p sees."""
    s = torch.arange(length)
    ok = s <= p
    return ok & ((s > p - window) | (s < sinks)) if window else ok


def attend(q, k, v, first, window=None, sinks=0, scale=None, present=None):
    """One request: q [n, Hq, D] at positions first .., k and v [L, Hk, D] -> (out, weight), both [n, Hq, D] float64:
    the softmax average of v over the tokens a row sees, and of |v| (the scale of rounding errors).  ``present``
    [L]: tokens that are there at all.  A row that sees none is 0."""
    n, Hq, D = q.shape
    L, Hk = k.shape[:2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(n, Hq, D, dtype=torch.float64)
    mag = torch.zeros(n, Hq, D, dtype=torch.float64)
    heads = torch.arange(Hq) // (Hq // Hk)
    for i in range(n):
        ok = seen(first + i, L, window, sinks)
        if present is not None:
            ok &= present
        idx = ok.nonzero()[:, 0]
        if not len(idx):
            continue
        ki, vi = k[idx].double()[:, heads], v[idx].double()[:, heads]     # [m, Hq, D]
        w = torch.softmax((q[i].double() * ki).sum(-1) * scale, 0)[..., None]
        out[i], mag[i] = (w * vi).sum(0), (w * vi.abs()).sum(0)
    return out, mag
