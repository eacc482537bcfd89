"""Plain forms of the operators on trees of drafted tokens (``fftsparse_amd.tree``) and of 8-bit pages, on the CPU, in
Python lists and 64 bits, from the definitions."""
from __future__ import annotations

import math

import torch

E4M3 = torch.float8_e4m3fn


def lines(parents):
    """Of each token of one request: itself and its ancestors, nearest first."""
    out = []
    for t, p in enumerate(parents):
        out.append([t] + (out[p] if 0 <= p < t else []))
    return out


def plan(parents, cu, seq_lens, words, window=None, sinks=0):
    """positions [T], mask [T][words] of unsigned 64-bit numbers; under a window without the ancestors that it hides."""
    T = len(parents)
    pos, mask = [-1] * T, [[0] * words for _ in range(T)]
    for b, L in enumerate(seq_lens):
        c0, c1 = cu[b], cu[b + 1]
        own = lines(parents[c0:c1])
        for t, line in enumerate(own[:64 * words]):
            pos[c0 + t] = L - (c1 - c0) + len(line) - 1
            base = L - (c1 - c0)
            for j in line:
                at = base + len(own[j]) - 1
                if window and at <= pos[c0 + t] - window and at >= sinks:
                    continue
                mask[c0 + t][j // 64] |= 1 << (j % 64)
    return pos, mask


def accept(parents, tokens, chosen, cu, most):
    """kept [T], kept_lens [B], dropped [B], next [B]."""
    kept, lens, dropped, after = [-1] * len(parents), [], [], []
    for b in range(len(cu) - 1):
        c0, n = cu[b], cu[b + 1] - cu[b]
        path = [0] if n else []
        while path:
            p = path[-1]
            t = next((t for t in range(p + 1, min(n, most)) if parents[c0 + t] == p
                      and (tokens[c0 + t] < 0 or tokens[c0 + t] == chosen[c0 + p])), None)
            if t is None:
                break
            path.append(t)
        kept[c0:c0 + len(path)] = path
        lens.append(len(path))
        dropped.append(len(path) - n)
        after.append(chosen[c0 + path[-1]] if path else -1)
    return kept, lens, dropped, after


def attend(q, k, v, n, sees, window=None, sinks=0, scale=None, present=None, pos=None):
    """One request: q [n, Hq, D]; k and v [L, Hk, D], the last n of them the new tokens'; sees [n, n] bool; pos [n]
    positions (windows) -> (out, weight of |v|), both [n, Hq, D] float64.  present [L]: tokens that are there."""
    _, Hq, D = q.shape
    L, Hk = k.shape[:2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(n, Hq, D, dtype=torch.float64)
    mag = torch.zeros(n, Hq, D, dtype=torch.float64)
    heads = torch.arange(Hq) // (Hq // Hk)
    base, s = L - n, torch.arange(L)
    for i in range(n):
        ok = s < base
        if window:
            ok &= (s > pos[i] - window) | (s < sinks)
        if base >= 0:
            ok[base:] = sees[i]
        else:
            ok[:] = sees[i][-base:]
        if present is not None:
            ok &= present
        idx = ok.nonzero()[:, 0]
        if not len(idx):
            continue
        ki, vi = k[idx].double()[:, heads], v[idx].double()[:, heads]
        w = torch.softmax((q[i].double() * ki).sum(-1) * scale, 0)[..., None]
        out[i], mag[i] = (w * vi).sum(0), (w * vi.abs()).sum(0)
    return out, mag


def e4m3_half_step(y):
    """Half a step of e4m3 at y (float64): 2^-4 of the power of two below |y|, and no less than 2^-10."""
    _, e = torch.frexp(y.abs().clamp(2.0 ** -9, 448.0))
    return torch.ldexp(torch.full_like(y, 0.5), (e - 1).clamp(min=-6) - 3)
