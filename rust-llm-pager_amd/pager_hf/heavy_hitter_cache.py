"""A KV cache of bounded size that keeps the tokens attention has given the most weight.

The paged store (PagedDecoder, KVBlockStore) keeps every token and places blocks on HBM or the host
by their attention mass. Where a session may forget instead, a bounded cache holds ``capacity``
tokens per row and KV head in HBM: the first ``keep_first``, the last ``keep_recent``, and of the rest
those with the most accumulated attention weight. Per layer::

    cache = HeavyHitterCache(batch, num_query_heads, num_kv_heads, capacity, head_dim, dtype, device)

    # prompt: q, k, v as the layer's own attention takes them ([B, H, T, D], after the rotary
    # embedding), lo = left padding per row
    w = prompt_attention_weights(q[:, :, -64:], k, lo=lo)
    cache.load_prompt(k, v, w, lo=lo)

    # each new token: q, k, v [B, H, D]
    q = cache.append(q, k, v, inv_freq)     # before the rotary embedding (or after it, without inv_freq)
    out = cache.attend(q)

Every call is queued on torch's current stream, reads lengths and weights on the device, and can be
captured in a graph. fp16 or bf16, head dims 16, 32, 64, 128 and 256, up to 16 query heads per KV
head; anything else raises NotImplementedError. Inference only. Calls on one cache belong on one stream, or
on streams that the caller orders.
"""
from __future__ import annotations

import ctypes
from collections.abc import Sequence

import torch

from . import _native as N
from .rotary import _dense_last, _inference_only, _inv_freq, _on, _positions, _strides

_CODES = {torch.float16: N.nat.DTYPE_F16, torch.bfloat16: N.nat.DTYPE_BF16}


def _check_dtype(dtype: torch.dtype) -> int:
    if dtype not in _CODES:
        raise NotImplementedError(f"the bounded cache takes float16 or bfloat16, got {dtype}")
    return _CODES[dtype]


def _first_columns(lo, batch: int, device: torch.device) -> torch.Tensor | None:
    if lo is None:
        return None
    if isinstance(lo, Sequence):
        lo = torch.tensor(lo, dtype=torch.int32, device=device)
    if lo.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"lo must be int32 or int64, got {lo.dtype}")
    if tuple(lo.shape) != (batch,):
        raise ValueError(f"lo must have shape ({batch},), got {tuple(lo.shape)}")
    if lo.device != device:
        raise ValueError(f"tensors on different devices: {device} and {lo.device}")
    return lo.to(torch.int32).contiguous()


def prompt_attention_weights(
    q: torch.Tensor,
    k: torch.Tensor,
    *,
    lo: torch.Tensor | Sequence[int] | None = None,
    scale: float | None = None,
    softcap: float | None = None,
) -> torch.Tensor:
    """The attention weight each token of a prompt gets from the prompt's last W queries: float32
    [B, Hkv, T], summed over those queries and over each KV head's query heads.

    q [B, Hq, W, D]: the last W columns' queries (W <= T; all of them: W = T); k [B, Hkv, T, D]; any
    strides, after the rotary embedding; causal. ``lo`` [B]: each row's first valid column (left
    padding); padded columns get 0 and padded queries give nothing. scale defaults to
    1/sqrt(head_dim); softcap None or 0.0 disables c*tanh(s/c)."""
    done = N.ops().prompt_weights(q, k, lo, scale, softcap)
    if done is not None:
        N.nat.check(done[0], "prompt_attention_weights")
        return done[1]
    _inference_only(q, k)
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"q and k must be [B, H, tokens, D], got {tuple(q.shape)} and {tuple(k.shape)}")
    b, hq, w, d = q.shape
    hkv, t = k.shape[1], k.shape[2]
    if k.shape[0] != b or k.shape[3] != d:
        raise ValueError(f"k shape {tuple(k.shape)} does not match q shape {tuple(q.shape)}")
    if k.dtype != q.dtype:
        raise TypeError("q and k must share one dtype")
    code = _check_dtype(q.dtype)
    device = N.require_cuda(q, k)
    lo = _first_columns(lo, b, device)
    q, k = _dense_last(q), _dense_last(k)
    out = torch.empty((b, hkv, t), dtype=torch.float32, device=device)
    nbytes = N.lib().pgr_hh_prompt_weights_workspace_bytes(b, hq, hkv, t, w, d)
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)
    with _on(device):
        N.nat.check(
            N.lib().pgr_hh_prompt_weights(
                q.data_ptr(), _strides(q, 3), k.data_ptr(), _strides(k, 3), N.ptr(lo), out.data_ptr(), b, hq, hkv, t, w,
                d, code, 1.0 / d**0.5 if scale is None else float(scale), float(softcap or 0.0), ws.data_ptr(), nbytes,
                N.stream_of(device),
            ),
            "prompt_attention_weights",
        )
    return out


class HeavyHitterCache:
    """One layer's bounded cache; see the module's description.

    The buffers can be read (and written, by a program that knows what it does) as ``keys`` and
    ``values`` [B, Hkv, capacity, D], ``weights`` [B, Hkv, capacity] float32, ``order`` [B, Hkv, capacity]
    int32 (a slot's token, counted from the row's first valid one), ``lengths`` and ``seen`` [B, Hkv] int32
    (slots in use, tokens seen so far). Slots from lengths on hold nothing (zeros at first)."""

    def __init__(self, batch: int, num_query_heads: int, num_kv_heads: int, capacity: int, head_dim: int,
                 dtype: torch.dtype, device: torch.device | str, *, keep_first: int = 4, keep_recent: int = 32):
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("HeavyHitterCache expects a CUDA (HIP) device")
        code = _check_dtype(dtype)
        if batch <= 0 or num_query_heads <= 0 or num_kv_heads <= 0 or capacity <= 0 or head_dim <= 0:
            raise ValueError("negative or zero dimension")
        if num_query_heads % num_kv_heads:
            raise ValueError("num_query_heads must be a multiple of num_kv_heads")
        if num_query_heads // num_kv_heads > 16:
            raise NotImplementedError("query heads per KV head are supported up to 16")
        if head_dim not in (16, 32, 64, 128, 256):
            raise NotImplementedError(f"head_dim must be 16, 32, 64, 128 or 256, got {head_dim}")
        if batch * num_kv_heads > 65535:
            raise ValueError("batch * num_kv_heads must not exceed 65535")
        if keep_first < 0 or keep_recent < 1 or keep_first + keep_recent > capacity:
            raise ValueError("need keep_first >= 0, keep_recent >= 1 and their sum within the capacity")
        if capacity > 1 << 26:
            raise ValueError("capacity must not exceed 2^26")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self._dtype, self._device = dtype, device
        rows = (batch, num_kv_heads)
        # Two allocations: what a token holds, and what is kept about it (each part on a 16-byte border).
        self._keys, self._values = torch.zeros((2, *rows, capacity, head_dim), dtype=dtype, device=device).unbind(0)
        slots, count = -(-batch * num_kv_heads * capacity // 4) * 4, -(-batch * num_kv_heads // 4) * 4
        state = torch.zeros(2 * (slots + count), dtype=torch.int32, device=device)
        weights, order, lengths, seen = state.split([slots, slots, count, count])
        self._weights = weights.view(torch.float32)[: batch * num_kv_heads * capacity].view(*rows, capacity)
        self._order = order[: batch * num_kv_heads * capacity].view(*rows, capacity)
        self._lengths, self._seen = (x[: batch * num_kv_heads].view(rows) for x in (lengths, seen))
        self._c = N.nat.HHCache(
            self._keys.data_ptr(), self._values.data_ptr(), self._weights.data_ptr(), self._order.data_ptr(),
            self._lengths.data_ptr(), self._seen.data_ptr(), batch, num_query_heads, num_kv_heads, capacity, head_dim,
            code, keep_first, keep_recent,
        )
        self._ref = ctypes.byref(self._c)
        self._address, self._index, self._ops = ctypes.addressof(self._c), device.index, N.ops()
        self._attend_bytes = N.lib().pgr_hh_attend_workspace_bytes(self._ref)

    # What the kernels go by is fixed with the cache: the buffers can be written to, not replaced.
    batch = property(lambda self: self._c.batch)
    num_query_heads = property(lambda self: self._c.query_heads)
    num_kv_heads = property(lambda self: self._c.kv_heads)
    capacity = property(lambda self: self._c.capacity)
    head_dim = property(lambda self: self._c.head_dim)
    keep_first = property(lambda self: self._c.keep_first)
    keep_recent = property(lambda self: self._c.keep_recent)
    dtype = property(lambda self: self._dtype)
    device = property(lambda self: self._device)
    keys = property(lambda self: self._keys)
    values = property(lambda self: self._values)
    weights = property(lambda self: self._weights)
    order = property(lambda self: self._order)
    lengths = property(lambda self: self._lengths)
    seen = property(lambda self: self._seen)

    def reset(self) -> None:
        """Empties every row."""
        with torch.inference_mode():  # (the cache may have been made in it)
            self._lengths.zero_()
            self._seen.zero_()

    def _apart(self, t: torch.Tensor | None) -> torch.Tensor | None:
        """t, or a copy where it views the cache's own state, which a call changes while it reads t."""
        own = t is not None and t.untyped_storage().data_ptr() == self._seen.untyped_storage().data_ptr()
        return t.clone() if own else t

    def _token(self, t: torch.Tensor, heads: int, name: str) -> torch.Tensor:
        if tuple(t.shape) != (self.batch, heads, self.head_dim):
            raise ValueError(f"{name} must have shape {(self.batch, heads, self.head_dim)}, got {tuple(t.shape)}")
        if t.dtype != self.dtype:
            raise TypeError(f"{name} must be {self.dtype}, got {t.dtype}")
        if t.device != self.device:
            raise ValueError(f"tensors on different devices: {self.device} and {t.device}")
        return _dense_last(t)

    def load_prompt(self, k: torch.Tensor, v: torch.Tensor, weights: torch.Tensor, *,
                    lo: torch.Tensor | Sequence[int] | None = None) -> None:
        """Starts every row over with a prompt: k, v [B, Hkv, T, D] (any strides), weights [B, Hkv, T]
        float32 (prompt_attention_weights). Row b's tokens are the columns from lo[b] on: all of them
        where they fit, else the first keep_first, the last keep_recent and the heaviest of the rest (the
        lowest column first among equals; NaN is the heaviest), in the order of their columns."""
        done = self._ops.load_prompt(self._address, self._index, k, v, weights, lo)
        if done is not None:
            N.nat.check(done, "HeavyHitterCache.load_prompt")
            return
        _inference_only(k, v, weights)
        if k.dim() != 4 or k.shape[0] != self.batch or k.shape[1] != self.num_kv_heads or k.shape[3] != self.head_dim:
            raise ValueError(f"k must have shape ({self.batch}, {self.num_kv_heads}, T, {self.head_dim}), got "
                             f"{tuple(k.shape)}")
        if tuple(v.shape) != tuple(k.shape):
            raise ValueError(f"v shape {tuple(v.shape)} differs from k shape {tuple(k.shape)}")
        if k.dtype != self.dtype or v.dtype != self.dtype:
            raise TypeError(f"k and v must be {self.dtype}")
        t = k.shape[2]
        if weights.dtype != torch.float32:
            raise TypeError(f"weights must be float32, got {weights.dtype}")
        if tuple(weights.shape) != (self.batch, self.num_kv_heads, t):
            raise ValueError(f"weights must have shape {(self.batch, self.num_kv_heads, t)}, got {tuple(weights.shape)}")
        for x in (k, v, weights):
            if x.device != self.device:
                raise ValueError(f"tensors on different devices: {self.device} and {x.device}")
        lo = self._apart(_first_columns(lo, self.batch, self.device))
        k, v, weights = _dense_last(k), _dense_last(v), weights.contiguous()
        nbytes = N.lib().pgr_hh_load_prompt_workspace_bytes(self._ref, t)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        with _on(self.device):
            N.nat.check(
                N.lib().pgr_hh_load_prompt(self._ref, k.data_ptr(), _strides(k, 3), v.data_ptr(), _strides(v, 3),
                                           weights.data_ptr(), N.ptr(lo), t, ws.data_ptr(), nbytes,
                                           N.stream_of(self.device)),
                "HeavyHitterCache.load_prompt",
            )

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, inv_freq: torch.Tensor | None = None, *,
               positions: torch.Tensor | None = None, interleaved: bool = False, factor: float = 1.0) -> torch.Tensor:
        """Stores one new token per row (k, v [B, Hkv, D]) and returns the queries to attend with.

        A full row gives up the token with the least weight that is neither among its first keep_first
        nor among its last keep_recent, the new token counted (the lowest slot among equals). With
        ``inv_freq`` (rotary.rotary_frequencies) q [B, Hq, D] and k are turned as rotary_embedding turns them,
        at the row's number of tokens seen so far or at positions[b]; without it both are taken as they
        are and q is returned itself."""
        done = self._ops.append(self._address, self._index, q, k, v, inv_freq, positions, interleaved, factor)
        if done is not None:
            N.nat.check(done[0], "HeavyHitterCache.append")
            return done[1]
        _inference_only(q, k, v, inv_freq)
        q_out, q = q, self._token(q, self.num_query_heads, "q")
        k = self._token(k, self.num_kv_heads, "k")
        v = self._token(v, self.num_kv_heads, "v")
        turning = 0
        if inv_freq is not None:
            inv_freq = _inv_freq(inv_freq, self.head_dim, self.device)
            turning = 2 * inv_freq.numel()
            q_out = torch.empty((self.batch, self.num_query_heads, self.head_dim), dtype=self.dtype, device=self.device)
        if positions is not None:
            positions = _positions(positions, self.device)
            if tuple(positions.shape) != (self.batch,):
                raise ValueError(f"positions must have shape ({self.batch},), got {tuple(positions.shape)}")
            positions = self._apart(positions.contiguous())
        with _on(self.device):
            N.nat.check(
                N.lib().pgr_hh_append(
                    self._ref, q.data_ptr(), _strides(q, 2), k.data_ptr(), _strides(k, 2), v.data_ptr(), _strides(v, 2),
                    q_out.data_ptr() if inv_freq is not None else None, N.ptr(positions),
                    positions is not None and positions.dtype == torch.int64, N.ptr(inv_freq), turning,
                    bool(interleaved), float(factor), N.stream_of(self.device),
                ),
                "HeavyHitterCache.append",
            )
        return q_out

    def attend(self, q: torch.Tensor, *, scale: float | None = None, softcap: float | None = None) -> torch.Tensor:
        """Attention of q [B, Hq, D] over each row's tokens; their probabilities, summed over each KV
        head's query heads, are added to ``weights``. Returns [B, Hq, D]; zeros for an empty row and
        for a head whose scores are all -inf. scale defaults to 1/sqrt(head_dim); softcap None or 0.0
        disables c*tanh(s/c)."""
        done = self._ops.attend(self._address, self._index, self._attend_bytes, q, scale, softcap)
        if done is not None:
            N.nat.check(done[0], "HeavyHitterCache.attend")
            return done[1]
        _inference_only(q)
        q = self._token(q, self.num_query_heads, "q")
        out = torch.empty((self.batch, self.num_query_heads, self.head_dim), dtype=self.dtype, device=self.device)
        ws = torch.empty(self._attend_bytes, dtype=torch.uint8, device=self.device) if self._attend_bytes else None
        with _on(self.device):
            N.nat.check(
                N.lib().pgr_hh_attend(
                    self._ref, q.data_ptr(), _strides(q, 2), out.data_ptr(),
                    1.0 / self.head_dim**0.5 if scale is None else float(scale), float(softcap or 0.0), N.ptr(ws),
                    self._attend_bytes, N.stream_of(self.device),
                ),
                "HeavyHitterCache.attend",
            )
        return out
