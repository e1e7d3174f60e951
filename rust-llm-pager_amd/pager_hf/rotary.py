"""Rotary position embedding over HIP kernels.

The decode paths here take q and k after the rotary embedding (as the reference's patched layers
hand them over, paged_model.py:926-955). These functions make them from a projection's output, for
callers that run a model's layers themselves::

    inv_freq, factor = rotary_frequencies(head_dim, scaling=config.rope_parameters, device=device)
    q, k = rotary_embedding(q, k, positions, inv_freq, factor=factor)

The angle position * inv_freq[i] is taken in 64 bits: in 32 its error grows with the position (2^-7
rad at 131072), which a model's own float32 tables show. Inference only: tensors that require
gradients are refused while gradients are recorded, and forward-mode tangents always; ``inverse=True`` is the transposed map, which
takes a gradient of the outputs back to the inputs.
"""
from __future__ import annotations

import ctypes
import math
from contextlib import nullcontext

import torch
from torch.autograd import forward_ad

from . import _native as N

_CODES = {torch.float16: N.nat.DTYPE_F16, torch.bfloat16: N.nat.DTYPE_BF16, torch.float32: N.nat.DTYPE_F32}


# What the rope types below read; a type passes over what another one reads.
_SETTINGS = {"rope_type", "type", "rope_theta", "partial_rotary_factor", "factor", "original_max_position_embeddings",
             "beta_fast", "beta_slow", "truncate", "attention_factor", "mscale", "mscale_all_dim", "low_freq_factor",
             "high_freq_factor"}


def rotary_frequencies(rotary_dim: int, base: float | None = None, scaling: dict | None = None,
                       device: torch.device | str | None = None) -> tuple[torch.Tensor, float]:
    """(inv_freq float32 [rotary_dim / 2], factor of cos and sin) of a model's rotary settings.

    ``base`` is scaling's "rope_theta" where None, else 10000; both may be given if they agree.
    ``scaling`` (a config's rope_scaling / rope_parameters) is None or a dict whose "rope_type" is

    * "default": inv_freq[i] = base^(-2i / rotary_dim);
    * "linear": positions divided by "factor";
    * "ntk": base * factor^(rotary_dim / (rotary_dim - 2)), which stretches the slow pairs by "factor"
      and leaves the fast ones;
    * "yarn": pairs that turn more than "beta_fast" (32) times within
      "original_max_position_embeddings" stay, those that turn less than "beta_slow" (1) times are
      divided by "factor", linear in the pair's index between; cos and sin are scaled by
      "attention_factor" (0.1 ln(factor) + 1, or with "mscale" and "mscale_all_dim" the ratio of
      0.1 mscale ln(factor) + 1 and 0.1 mscale_all_dim ln(factor) + 1);
    * "llama3": wavelengths below original / "high_freq_factor" stay, those above original /
      "low_freq_factor" are divided by "factor", linear in original / wavelength between.

    Entries that none of these reads raise NotImplementedError, and so does a "partial_rotary_factor" other
    than 1: pass the dims that turn as rotary_dim, and the settings without it.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be a positive even number, got {rotary_dim}")
    scaling = scaling or {}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    unread = sorted(name for name, value in scaling.items() if value is not None and name not in _SETTINGS)
    if unread:
        raise NotImplementedError(f"rope_type {kind!r} with settings that are not supported: {', '.join(unread)}")
    if scaling.get("partial_rotary_factor") not in (None, 1.0):
        raise NotImplementedError("partial_rotary_factor: pass the dims that turn as rotary_dim, without this entry")
    theta = scaling.get("rope_theta")
    if base is not None and theta is not None and float(base) != float(theta):
        raise ValueError(f"base {base} differs from the settings' rope_theta {theta}")
    base = float(base if base is not None else theta if theta is not None else 10000.0)
    if not base > 0 or not math.isfinite(base):
        raise ValueError(f"base (rope_theta) must be positive, got {base}")
    attention_factor = 1.0
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)

    def setting(name, default=None):
        value = scaling.get(name, default)
        if value is None:
            raise ValueError(f"rope_type {kind!r} needs {name!r}")
        value = float(value)
        if not value > 0 or not math.isfinite(value):
            raise ValueError(f"{name} must be positive, got {value}")
        return value

    if kind == "ntk":
        if rotary_dim < 4:
            raise ValueError("rope_type 'ntk' needs a rotary_dim of 4 or more")
        base = base * setting("factor") ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-i / rotary_dim)
    if kind == "linear":
        freq = freq / setting("factor")
    elif kind == "yarn":
        factor, original = setting("factor"), setting("original_max_position_embeddings")
        fast, slow = setting("beta_fast", 32.0), setting("beta_slow", 1.0)

        def index(rotations):  # the pair that turns `rotations` times over the original length
            return rotary_dim * math.log(original / (rotations * 2 * math.pi)) / (2 * math.log(base))

        first, last = index(fast), index(slow)
        if scaling.get("truncate", True):
            first, last = math.floor(first), math.ceil(last)
        first, last = max(first, 0), min(last, rotary_dim - 1)
        if first == last:
            last += 0.001
        ramp = ((i / 2 - first) / (last - first)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        scales = [name for name in ("mscale", "mscale_all_dim") if scaling.get(name) is not None]

        def stretch(m):
            return 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0

        if scaling.get("attention_factor") is not None:
            attention_factor = setting("attention_factor")
        elif len(scales) == 1:
            raise ValueError(f"{scales[0]} needs the other of mscale and mscale_all_dim")
        else:
            attention_factor = stretch(setting("mscale")) / stretch(setting("mscale_all_dim")) if scales else stretch(1.0)
    elif kind == "llama3":
        factor, original = setting("factor"), setting("original_max_position_embeddings")
        low, high = setting("low_freq_factor"), setting("high_freq_factor")
        if not high > low:
            raise ValueError("high_freq_factor must be greater than low_freq_factor")
        turns = original * freq / (2 * math.pi)  # the original length in wavelengths
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        freq = freq / factor * (1 - keep) + freq * keep
    elif kind not in ("default", "ntk"):
        raise NotImplementedError(f"rope_type {kind!r}; supported: default, linear, ntk, yarn, llama3")
    return freq.float().to(device or "cpu"), attention_factor


def _inference_only(*tensors: torch.Tensor | None) -> None:
    recording = torch.is_grad_enabled()
    if any(t is not None and (recording and t.requires_grad or forward_ad.unpack_dual(t).tangent is not None)
           for t in tensors):
        raise RuntimeError("this operator records no gradient and takes no forward-mode tangents; call it under "
                           "torch.no_grad() (gradients) or torch.inference_mode() (both)")


def _on(device: torch.device):
    """Launches go to the tensors' device, whichever is current."""
    return nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _dense_last(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _strides(t: torch.Tensor, dims: int):
    return (ctypes.c_int64 * dims)(*t.stride()[:dims])


def _inv_freq(inv_freq: torch.Tensor, head_dim: int, device: torch.device) -> torch.Tensor:
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1:
        raise ValueError(f"inv_freq must be a float32 vector, got {inv_freq.dtype} {tuple(inv_freq.shape)}")
    if 2 * inv_freq.numel() > head_dim:
        raise ValueError(f"inv_freq turns {2 * inv_freq.numel()} dims of a head of {head_dim}")
    if inv_freq.device != device:
        raise ValueError(f"tensors on different devices: {device} and {inv_freq.device}")
    return inv_freq.contiguous()


def _positions(positions: torch.Tensor, device: torch.device) -> torch.Tensor:
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    if positions.device != device:
        raise ValueError(f"tensors on different devices: {device} and {positions.device}")
    return positions


def rotary_embedding(
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    *,
    interleaved: bool = False,
    factor: float = 1.0,
    inverse: bool = False,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """q and k with the first 2 * len(inv_freq) dims of each head turned by position * inv_freq.

    q [B, Hq, T, D] and k [B, Hk, T, D] (or None), any strides, one dtype (float16, bfloat16, float32), with
    positions [B, T] or [1, T]; or, one token per row, q [B, Hq, D], k [B, Hk, D] and positions [B].
    The pairs are (i, i + len(inv_freq)), or (2i, 2i + 1) with ``interleaved``; ``factor`` scales the
    turned dims (rotary_frequencies' second result). New contiguous tensors are returned."""
    done = N.ops().rotary(q, k, positions, inv_freq, interleaved, factor, inverse)
    if done is not None:
        N.nat.check(done[0], "rotary_embedding")
        return done[1], done[2]
    single = q.dim() == 3
    if q.dim() not in (3, 4):
        raise ValueError(f"q must be [B, H, T, D] or [B, H, D], got {tuple(q.shape)}")
    if k is not None and k.dim() != q.dim():
        raise ValueError(f"k shape {tuple(k.shape)} does not match q shape {tuple(q.shape)}")
    if single:
        if positions.dim() != 1:
            raise ValueError(f"positions must be [B], got {tuple(positions.shape)}")
        out = rotary_embedding(q.unsqueeze(2), None if k is None else k.unsqueeze(2), positions.unsqueeze(1), inv_freq,
                               interleaved=interleaved, factor=factor, inverse=inverse)
        return out[0].squeeze(2), None if k is None else out[1].squeeze(2)
    _inference_only(q, k, inv_freq)
    b, hq, t, d = q.shape
    if k is not None and (k.shape[0], k.shape[2], k.shape[3]) != (b, t, d):
        raise ValueError(f"k shape {tuple(k.shape)} does not match q shape {tuple(q.shape)}")
    if k is not None and k.dtype != q.dtype:
        raise TypeError("q and k must share one dtype")
    if q.dtype not in _CODES:
        raise NotImplementedError(f"rotary_embedding takes float16, bfloat16 or float32, got {q.dtype}")
    device = N.require_cuda(q, k)
    inv_freq = _inv_freq(inv_freq, d, device)
    positions = _positions(positions, device)
    if positions.dim() != 2 or positions.shape[0] not in (1, b) or positions.shape[1] != t:
        raise ValueError(f"positions must be [{b}, {t}] or [1, {t}], got {tuple(positions.shape)}")
    positions = positions.expand(b, t)
    q = _dense_last(q)
    k = _dense_last(k) if k is not None else None
    q_out = torch.empty((b, hq, t, d), dtype=q.dtype, device=device)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=device) if k is not None else None
    with _on(device):
        N.nat.check(
            N.lib().pgr_rotary(
                q.data_ptr(), _strides(q, 3), q_out.data_ptr(), hq, N.ptr(k), _strides(k, 3) if k is not None else None,
                N.ptr(k_out), k.shape[1] if k is not None else 0, positions.data_ptr(), positions.dtype == torch.int64,
                _strides(positions, 2), inv_freq.data_ptr(), 2 * inv_freq.numel(), b, t, d, _CODES[q.dtype],
                bool(interleaved), float(factor), bool(inverse), N.stream_of(device),
            ),
            "rotary_embedding",
        )
    return q_out, k_out


def _norm_weight(weight: torch.Tensor, name: str, head_dim: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    if tuple(weight.shape) != (head_dim,):
        raise ValueError(f"{name} must have shape ({head_dim},), got {tuple(weight.shape)}")
    if weight.dtype not in (dtype, torch.float32):
        raise TypeError(f"{name} must be {dtype} or torch.float32, got {weight.dtype}")
    if weight.device != device:
        raise ValueError(f"tensors on different devices: {device} and {weight.device}")
    return weight.contiguous()


def norm_rotary_embedding(
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor | None,
    *,
    eps: float = 1e-6,
    interleaved: bool = False,
    factor: float = 1.0,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """rotary_embedding of q and k whose heads are normed first: x / sqrt(mean(x^2) + eps) * weight, as models with
    norms of queries and keys (qwen3) have it.

    Shapes, types, pairs and factor as in rotary_embedding; q_weight and k_weight [D] have q's dtype or are float32,
    both the same (a norm that multiplies by 1 + w takes 1 + w here). Computed in float32 and rounded once, where a
    norm and a rotation of their own round twice or more. An inv_freq of no elements norms without a turn."""
    done = N.ops().norm_rotary(q, k, positions, inv_freq, q_weight, k_weight, eps, interleaved, factor)
    if done is not None:
        N.nat.check(done[0], "norm_rotary_embedding")
        return done[1], done[2]
    single = q.dim() == 3
    if q.dim() not in (3, 4):
        raise ValueError(f"q must be [B, H, T, D] or [B, H, D], got {tuple(q.shape)}")
    if k is not None and k.dim() != q.dim():
        raise ValueError(f"k shape {tuple(k.shape)} does not match q shape {tuple(q.shape)}")
    if single:
        if positions.dim() != 1:
            raise ValueError(f"positions must be [B], got {tuple(positions.shape)}")
        out = norm_rotary_embedding(q.unsqueeze(2), None if k is None else k.unsqueeze(2), positions.unsqueeze(1),
                                    inv_freq, q_weight, k_weight, eps=eps, interleaved=interleaved, factor=factor)
        return out[0].squeeze(2), None if k is None else out[1].squeeze(2)
    _inference_only(q, k, inv_freq, q_weight, k_weight)
    b, hq, t, d = q.shape
    if k is not None and (k.shape[0], k.shape[2], k.shape[3]) != (b, t, d):
        raise ValueError(f"k shape {tuple(k.shape)} does not match q shape {tuple(q.shape)}")
    if k is not None and k.dtype != q.dtype:
        raise TypeError("q and k must share one dtype")
    if (k is None) != (k_weight is None):
        raise ValueError("k and k_weight come together")
    if q.dtype not in _CODES:
        raise NotImplementedError(f"norm_rotary_embedding takes float16, bfloat16 or float32, got {q.dtype}")
    device = N.require_cuda(q, k)
    inv_freq = _inv_freq(inv_freq, d, device)
    positions = _positions(positions, device)
    if positions.dim() != 2 or positions.shape[0] not in (1, b) or positions.shape[1] != t:
        raise ValueError(f"positions must be [{b}, {t}] or [1, {t}], got {tuple(positions.shape)}")
    positions = positions.expand(b, t)
    q_weight = _norm_weight(q_weight, "q_weight", d, q.dtype, device)
    if k is not None:
        k_weight = _norm_weight(k_weight, "k_weight", d, q.dtype, device)
        if k_weight.dtype != q_weight.dtype:
            raise TypeError("q_weight and k_weight must share one dtype")
    q = _dense_last(q)
    k = _dense_last(k) if k is not None else None
    q_out = torch.empty((b, hq, t, d), dtype=q.dtype, device=device)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=device) if k is not None else None
    with _on(device):
        N.nat.check(
            N.lib().pgr_norm_rotary(
                q.data_ptr(), _strides(q, 3), q_out.data_ptr(), hq, N.ptr(k), _strides(k, 3) if k is not None else None,
                N.ptr(k_out), k.shape[1] if k is not None else 0, q_weight.data_ptr(), N.ptr(k_weight),
                q_weight.dtype == torch.float32, float(eps), positions.data_ptr(), positions.dtype == torch.int64,
                _strides(positions, 2), inv_freq.data_ptr(), 2 * inv_freq.numel(), b, t, d, _CODES[q.dtype],
                bool(interleaved), float(factor), N.stream_of(device),
            ),
            "norm_rotary_embedding",
        )
    return q_out, k_out
