"""Bounded-cache operators in 64 bits: rotary positions, a prompt's attention weights, the choice of
the tokens that stay, the append that evicts, and the weighted decode attention.

Plain numpy over float64, one row at a time. Functions that have a rounding behind them in the
product also return a bound of its error, from the operator's own steps: half a step of the output
type, half a step of P in the K/V type, the float32 dot products (one rounding per term, 2^-24 of
the sum of magnitudes), and the float32 sums.
"""
from __future__ import annotations

import numpy as np

U32 = 2.0**-24  # half a step of float32


def rotate(x, positions, inv_freq, *, interleaved=False, factor=1.0, inverse=False):
    """x [..., D] at positions broadcastable to x's leading dims; inv_freq as given (float32 values)."""
    x = np.asarray(x, np.float64)
    angle = np.asarray(positions, np.float64)[..., None] * np.asarray(inv_freq, np.float64)
    cos, sin = factor * np.cos(angle), factor * np.sin(angle) * (-1.0 if inverse else 1.0)
    half = len(inv_freq)
    out = x.copy()
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    first, second = a * cos - b * sin, a * sin + b * cos
    if interleaved:
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = first, second
    else:
        out[..., :half], out[..., half:2 * half] = first, second
    return out


def scores(q, k, scale, softcap):
    """(s, bound) for q [..., D] and k [n, D]: scale q.k, softcapped; the bound is that of float32
    products added one after the other, the scale and the softcap's tanh included."""
    s = q @ k.T * scale
    size = np.abs(q) @ np.abs(k).T * scale
    bound = (q.shape[-1] + 4) * U32 * size
    if softcap:
        s = softcap * np.tanh(s / softcap)
        bound = bound + 8 * U32 * softcap
    return s, bound


def attend(q, keys, values, weights, scale, softcap, step, p_step=None, p_floor=2.0**-25):
    """One row: q [n_rep, D], keys and values [n, D], weights [n]. Returns (out, out bound, weights, weights
    bound); `step` is half a step of the K/V and output type, p_step (`step`) and p_floor what P may be off by
    as it enters the product with V: relative, and absolute where its largest value is 1."""
    p_step = step if p_step is None else p_step
    n_rep, d = q.shape
    n = len(keys)
    if n == 0:
        return np.zeros((n_rep, d)), np.zeros((n_rep, d)), weights.copy(), np.zeros(0)
    s, ds = scores(q, keys, scale, softcap)
    top = s.max(axis=-1, keepdims=True)
    p = np.exp(s - top)
    p /= p.sum(axis=-1, keepdims=True)
    # A weight's relative error: its score's, the maximum's and the sum's, and the exponent's argument.
    rel = 2 * ds.max(axis=-1, keepdims=True) + (n + 16) * U32 + 4 * U32 * np.abs(s - top)
    out = p @ values
    # P rounded under a maximum of its own: half a step, or half of the smallest fp16 subnormal of weights
    # whose largest is 1; the output's own rounding likewise.
    out_bound = (p * (p_step + rel)) @ np.abs(values) + p_floor * np.abs(values).sum(axis=0)
    out_bound = out_bound + step * (np.abs(out) + out_bound) + 2.0**-25
    new = weights + p.sum(axis=0)
    new_bound = (p * rel).sum(axis=0) + (n_rep + 1) * U32 * np.abs(new)
    return out, out_bound, new, new_bound + 1e-30


def prompt_weights(q, k, lo, scale, softcap):
    """One row: q [n_rep, W, D], k [T, D]. Returns (weights [T], bound)."""
    n_rep, w, _ = q.shape
    t = len(k)
    out, bound = np.zeros(t), np.zeros(t)
    for i in range(w):
        last = t - w + i
        if last < lo:
            continue
        s, ds = scores(q[:, i], k[lo:last + 1], scale, softcap)
        top = s.max(axis=-1, keepdims=True)
        p = np.exp(s - top)
        p /= p.sum(axis=-1, keepdims=True)
        rel = 2 * ds.max(axis=-1, keepdims=True) + (t + 16) * U32 + 4 * U32 * np.abs(s - top)
        out[lo:last + 1] += p.sum(axis=0)
        bound[lo:last + 1] += (p * rel).sum(axis=0)
    return out, bound + n_rep * w * U32 * out + 1e-30


def heaviness(w):
    """Sort key of a weight: NaN is the heaviest, -0 equals 0."""
    w = np.asarray(w, np.float64)
    return np.where(np.isnan(w), np.inf, w), np.isnan(w)


def kept_columns(weights, lo, capacity, keep_first, keep_recent):
    """Columns of one row's prompt that stay, ascending. weights [T]."""
    t = len(weights)
    n = t - lo
    if n <= capacity:
        return np.arange(lo, t)
    held = [j for j in range(n) if j < keep_first or j >= n - keep_recent]
    free = [j for j in range(n) if keep_first <= j < n - keep_recent]
    value, nan = heaviness(weights[lo:])
    free.sort(key=lambda j: (not nan[j], -value[j], j))
    return np.array(sorted(held + free[: capacity - len(held)])) + lo


def append_slot(length, seen, weights, order, capacity, keep_first, keep_recent):
    """The slot one row's next token takes."""
    if length < capacity:
        return length
    value, nan = heaviness(weights)
    held = (order < keep_first) | (order >= seen + 1 - keep_recent)
    return min(range(capacity), key=lambda j: (bool(held[j]), bool(nan[j]), value[j], j))
