"""The operators of drafted tokens over a cache of pages, in 64 bits: per-head norms, trees, the append into
pages, the attention of several new tokens and the move of the accepted path.

Plain numpy over float64 and row by row; with bounds of the error that the operators' own roundings explain, in
steps of half a unit in the last place (2^-24 in float32).
"""
from __future__ import annotations

import numpy as np

from .bounded_cache import U32, attend, rotate


def norm(x, weight, eps):
    """(x / sqrt(mean(x^2) + eps) * weight over the last dim, bound): the sum's terms are positive, one rounding
    each in float32; the mean, eps, root, quotient and two products round once each."""
    x, weight = np.asarray(x, np.float64), np.asarray(weight, np.float64)
    y = x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * weight
    return y, (x.shape[-1] + 10) * U32 * np.abs(y)


def norm_rotate(x, weight, eps, positions, inv_freq, *, interleaved=False, factor=1.0):
    """(norm, where a weight is given, and turn; bound before the output's rounding). The turn: cos and sin within
    2 steps (4 halves), their scale, the two products and the sum."""
    x = np.asarray(x, np.float64)
    y, bound = (x, np.zeros_like(x)) if weight is None else norm(x, weight, eps)
    half = len(inv_freq)
    size, off = np.abs(y), bound
    a, b = (np.s_[..., 0:2 * half:2], np.s_[..., 1:2 * half:2]) if interleaved else (np.s_[..., :half], np.s_[..., half:2 * half])
    pair, both = size[a] + size[b], off[a] + off[b]
    bound = bound.copy()
    bound[a] = bound[b] = abs(factor) * (both + 8 * U32 * pair)
    return rotate(y, positions, inv_freq, interleaved=interleaved, factor=factor), bound


def tree(parents):
    """(sees [B, T, T], depths [B, T]) by walking each token up to its root."""
    b, t = parents.shape
    sees = np.zeros((b, t, t), bool)
    for i in range(b):
        for j in range(t):
            at = j
            while True:
                sees[i, j, at] = True
                up = parents[i, at]
                if not 0 <= up < at:
                    break
                at = up
    return sees, sees.sum(axis=-1) - 1


def cells(table, page_tokens, pages, first, n):
    """(page, place) of a row's tokens [first, first + n); page -1 where there is none."""
    at = np.arange(first, first + n)
    index = at // page_tokens
    page = np.where(index < len(table), np.asarray(table)[np.minimum(index, len(table) - 1)] if len(table) else -1, -1)
    return np.where((page >= 0) & (page < pages), page, -1), at % page_tokens


def attend_row(q, keys, values, there, length, n, sees, depths, window, scale, softcap, step, p_step, p_floor):
    """One row and KV head: q [n_rep, T, D], keys and values [length + n, D], there [length + n] (whether the token's
    page is), sees [n, n] among the new tokens. Returns (out [n_rep, T, D], bound); zeros from token n on."""
    out = np.zeros(q.shape)
    bound = np.zeros(q.shape)
    position = np.concatenate([np.arange(length), length + depths[:n]])
    for t in range(n):
        ok = np.concatenate([np.ones(length, bool), sees[t, :n]]) & there
        if window:
            ok &= position > length + depths[t] - window
        if ok.any():
            out[:, t], bound[:, t], _, _ = attend(q[:, t], keys[ok], values[ok], np.zeros(ok.sum()), scale, softcap, step,
                                                  p_step, p_floor)
    return out, bound
