"""A KV cache of pages in HBM for rows that take several new tokens a step: drafted tokens to be verified, a
prompt's chunks, or one token each.

The paged store (PagedDecoder, KVBlockStore) decodes one token a step and places blocks itself. Here the
caller holds the tables: ``table`` [B, W] int32 names each row's pages in order (an entry outside the pool: no
page), ``lengths`` [B] int32 the tokens it holds. All layers share them::

    cache = PageTableCache(num_layers, num_pages, page_tokens, num_query_heads, num_kv_heads, head_dim, dtype, device)

    tree = draft_tree(parents)                     # [B, T]: each drafted token's parent, -1 after the held ones
    for layer in range(num_layers):                # q, k, v [B, H, T, D] before norm and rotary embedding
        q = cache.append(layer, q, k, v, table, lengths, inv_freq, tree=tree, q_weight=qw, k_weight=kw)
        out = cache.attend(layer, q, table, lengths, tree=tree)
    # the caller decides which path is accepted: path [B, A] int32, the drafted tokens in order, -1 behind
    cache.keep(table, lengths, path)
    lengths += accepted

Without ``tree`` the new tokens follow each other: a prompt's chunk (any T), a chain of drafts, or with q, k, v
[B, H, D] one token. New token t is token lengths[b] + t of its row until keep has moved it; its rotary position
is lengths[b] plus its depth in the tree (its number, without one). ``counts`` [B] int32 says how many of the T
columns are a row's own; the others are not stored, and their outputs are zeros.

Every call is queued on torch's current stream, reads tables, lengths and counts on the device, and can be captured
in a graph. Tokens behind the table's end, or in a page that is not there, are not stored and not attended to. fp16
or bf16, head dims 16, 32, 64, 128 and 256, up to 16 query heads per KV head, pages of 16 to 256 tokens; anything
else raises NotImplementedError. Inference only. Calls on one cache belong on one stream, or on streams that the
caller orders; rows may share pages that no call writes to.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _native as N
from .heavy_hitter_cache import _check_dtype
from .rotary import _dense_last, _inference_only, _inv_freq, _norm_weight, _on, _positions, _strides


class DraftTree(NamedTuple):
    """What drafted tokens see of each other: bit j of masks [B, T] int64 is set where the token sees drafted
    token j; depths [B, T] int32 is what its position lies behind the row's held tokens (below 0 counts as 0)."""

    masks: torch.Tensor
    depths: torch.Tensor


def draft_tree(parents: torch.Tensor) -> DraftTree:
    """The masks (a token's ancestors and itself) and depths of trees of up to 64 drafted tokens.

    parents [B, T] int32: each token's parent, an earlier token of its row; anything else (-1) makes it follow
    the held tokens. Made once a step, for all layers."""
    done = N.ops().draft_tree(parents)
    if done is not None:
        N.nat.check(done[0], "draft_tree")
        return DraftTree(done[1], done[2])
    if parents.dim() != 2:
        raise ValueError(f"parents must be [B, T], got {tuple(parents.shape)}")
    if parents.dtype != torch.int32:
        raise TypeError(f"parents must be int32, got {parents.dtype}")
    device = N.require_cuda(parents)
    parents = parents.contiguous()
    masks = torch.empty(parents.shape, dtype=torch.int64, device=device)
    depths = torch.empty(parents.shape, dtype=torch.int32, device=device)
    with _on(device):
        N.nat.check(
            N.lib().pgr_draft_tree(parents.data_ptr(), parents.shape[0], parents.shape[1], masks.data_ptr(),
                                   depths.data_ptr(), N.stream_of(device)),
            "draft_tree",
        )
    return DraftTree(masks, depths)


class PageTableCache:
    """The pages of all layers; see the module's description.

    The buffers can be read (and written, by a program that knows what it does) as ``keys`` and ``values``
    [num_layers, num_pages, Hkv, page_tokens, D]."""

    def __init__(self, num_layers: int, num_pages: int, page_tokens: int, num_query_heads: int, num_kv_heads: int,
                 head_dim: int, dtype: torch.dtype, device: torch.device | str):
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("PageTableCache expects a CUDA (HIP) device")
        code = _check_dtype(dtype)
        if min(num_layers, num_pages, num_query_heads, num_kv_heads, head_dim) <= 0:
            raise ValueError("negative or zero dimension")
        if num_query_heads % num_kv_heads:
            raise ValueError("num_query_heads must be a multiple of num_kv_heads")
        if num_query_heads // num_kv_heads > 16:
            raise NotImplementedError("query heads per KV head are supported up to 16")
        if head_dim not in (16, 32, 64, 128, 256):
            raise NotImplementedError(f"head_dim must be 16, 32, 64, 128 or 256, got {head_dim}")
        if page_tokens not in (16, 32, 64, 128, 256):
            raise NotImplementedError(f"page_tokens must be 16, 32, 64, 128 or 256, got {page_tokens}")
        if num_pages > 1 << 30 or num_layers > 65535 or num_kv_heads > 65535 or num_layers * num_kv_heads > 1 << 28:
            raise ValueError("num_pages must not exceed 2^30, num_layers and num_kv_heads 65535, nor their product 2^28")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self._dtype, self._device = dtype, device
        self._keys, self._values = torch.zeros((2, num_layers, num_pages, num_kv_heads, page_tokens, head_dim),
                                               dtype=dtype, device=device).unbind(0)
        self._c = N.nat.PTCache(self._keys.data_ptr(), self._values.data_ptr(), num_layers, num_pages, num_query_heads,
                                num_kv_heads, page_tokens, head_dim, code)
        self._ref = ctypes.byref(self._c)
        self._address, self._index, self._ops = ctypes.addressof(self._c), device.index, N.ops()

    # What the kernels go by is fixed with the cache: the buffers can be written to, not replaced.
    num_layers = property(lambda self: self._c.layers)
    num_pages = property(lambda self: self._c.pages)
    page_tokens = property(lambda self: self._c.page_tokens)
    num_query_heads = property(lambda self: self._c.query_heads)
    num_kv_heads = property(lambda self: self._c.kv_heads)
    head_dim = property(lambda self: self._c.head_dim)
    dtype = property(lambda self: self._dtype)
    device = property(lambda self: self._device)
    keys = property(lambda self: self._keys)
    values = property(lambda self: self._values)

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.num_layers:
            raise IndexError(f"layer {layer} of {self.num_layers}")
        return int(layer)

    def _new(self, x: torch.Tensor, heads: int, name: str, like: torch.Tensor | None = None) -> torch.Tensor:
        """x as [B, heads, T, D]; with `like`, of its rows and tokens."""
        if x.dim() not in (3, 4) or x.shape[1] != heads or x.shape[-1] != self.head_dim:
            raise ValueError(f"{name} must have shape (B, {heads}, T, {self.head_dim}) or (B, {heads}, "
                             f"{self.head_dim}), got {tuple(x.shape)}")
        if like is not None and (x.dim(), x.shape[0], x.shape[2:]) != (like.dim(), like.shape[0], like.shape[2:]):
            raise ValueError(f"{name} shape {tuple(x.shape)} does not match q shape {tuple(like.shape)}")
        if x.dtype != self.dtype:
            raise TypeError(f"{name} must be {self.dtype}, got {x.dtype}")
        self._here(x)
        return _dense_last(x if x.dim() == 4 else x.unsqueeze(2))

    def _here(self, x: torch.Tensor) -> None:
        if x.device != self.device:
            raise ValueError(f"tensors on different devices: {self.device} and {x.device}")

    def _numbers(self, x: torch.Tensor, name: str, shape: tuple, dtype: torch.dtype = torch.int32) -> torch.Tensor:
        if x.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}, got {x.dtype}")
        if tuple(x.shape) != shape:
            raise ValueError(f"{name} must have shape {shape}, got {tuple(x.shape)}")
        self._here(x)
        return x.contiguous()

    def _rows(self, table: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor | None, batch: int, tokens: int):
        """pgr_pt_rows_t and what has to live as long as the call."""
        if table.dim() != 2 or table.shape[0] != batch:
            raise ValueError(f"table must have shape ({batch}, W), got {tuple(table.shape)}")
        if table.dtype != torch.int32:
            raise TypeError(f"table must be int32, got {table.dtype}")
        self._here(table)
        table = _dense_last(table)
        lengths = self._numbers(lengths, "lengths", (batch,))
        counts = None if counts is None else self._numbers(counts, "counts", (batch,))
        rows = N.nat.PTRows(table.data_ptr(), table.stride(0), table.shape[1], lengths.data_ptr(), N.ptr(counts), batch,
                            tokens)
        return rows, (table, lengths, counts)

    def _tree(self, tree: DraftTree | tuple[torch.Tensor, torch.Tensor] | None, batch: int, tokens: int):
        if tree is None:
            return None, None
        if tokens > 64:
            raise NotImplementedError(f"a tree has up to 64 tokens, got {tokens}")
        if not isinstance(tree, tuple) or len(tree) != 2:
            raise TypeError(f"tree must be a DraftTree or a pair (masks, depths), got {type(tree).__name__}")
        return (self._numbers(tree[0], "tree.masks", (batch, tokens), torch.int64),
                self._numbers(tree[1], "tree.depths", (batch, tokens)))

    def append(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
               lengths: torch.Tensor, inv_freq: torch.Tensor | None = None, *, counts: torch.Tensor | None = None,
               tree: DraftTree | None = None, positions: torch.Tensor | None = None,
               q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
               interleaved: bool = False, factor: float = 1.0) -> torch.Tensor:
        """Stores new tokens k, v [B, Hkv, T, D] in their rows' pages and returns the queries to attend with, shaped
        as q [B, Hq, T, D] (or [B, H, D] throughout: one token), zeros where a token is not its row's own.

        With q_weight and k_weight [D] the heads of q and k are normed as norm_rotary_embedding norms them; with
        ``inv_freq`` (rotary.rotary_frequencies) they are turned, at lengths[b] plus the token's depth in the tree
        (its number, without one), or at positions [B, T] ([B] for one token). ``lengths`` stays as it is."""
        done = self._ops.pt_append(self._address, self._index, layer, q, k, v, table, lengths, inv_freq, counts, tree,
                                   positions, q_weight, k_weight, eps, interleaved, factor)
        if done is not None:
            N.nat.check(done[0], "PageTableCache.append")
            return done[1]
        _inference_only(q, k, v, inv_freq, q_weight, k_weight)
        layer = self._layer(layer)
        x = self._new(q, self.num_query_heads, "q")
        k, v = self._new(k, self.num_kv_heads, "k", q), self._new(v, self.num_kv_heads, "v", q)
        b, t = x.shape[0], x.shape[2]
        rows, held = self._rows(table, lengths, counts, b, t)
        _, depths = self._tree(tree, b, t)
        turning = 0
        if inv_freq is not None:
            inv_freq = _inv_freq(inv_freq, self.head_dim, self.device)
            turning = 2 * inv_freq.numel()
        if positions is not None:
            positions = _positions(positions, self.device)
            if q.dim() == 3:
                positions = positions.unsqueeze(-1)
            if tuple(positions.shape) != (b, t):
                raise ValueError(f"positions must have shape {(b, t) if q.dim() == 4 else (b,)}, got "
                                 f"{tuple(positions.shape) if q.dim() == 4 else tuple(positions.shape[:-1])}")
        if (q_weight is None) != (k_weight is None):
            raise ValueError("q_weight and k_weight come together")
        if q_weight is not None:
            q_weight = _norm_weight(q_weight, "q_weight", self.head_dim, self.dtype, self.device)
            k_weight = _norm_weight(k_weight, "k_weight", self.head_dim, self.dtype, self.device)
            if q_weight.dtype != k_weight.dtype:
                raise TypeError("q_weight and k_weight must share one dtype")
        out = torch.empty((b, self.num_query_heads, t, self.head_dim), dtype=self.dtype, device=self.device)
        with _on(self.device):
            N.nat.check(
                N.lib().pgr_pt_append(
                    self._ref, layer, ctypes.byref(rows), x.data_ptr(), _strides(x, 3), k.data_ptr(), _strides(k, 3),
                    v.data_ptr(), _strides(v, 3), out.data_ptr(), N.ptr(positions),
                    positions is not None and positions.dtype == torch.int64,
                    None if positions is None else _strides(positions, 2), N.ptr(depths), N.ptr(inv_freq), turning,
                    bool(interleaved), float(factor), N.ptr(q_weight), N.ptr(k_weight),
                    q_weight is not None and q_weight.dtype == torch.float32, float(eps), N.stream_of(self.device),
                ),
                "PageTableCache.append",
            )
        return out if q.dim() == 4 else out.squeeze(2)

    def attend(self, layer: int, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
               counts: torch.Tensor | None = None, tree: DraftTree | None = None, window: int | None = None,
               softcap: float | None = None, scale: float | None = None, exact_weights: bool = True) -> torch.Tensor:
        """Attention of the new tokens' queries q [B, Hq, T, D] (or [B, Hq, D]) over what their rows hold and, among
        the new tokens (appended before, with the same lengths), over those before them and themselves, or those
        that the tree's masks name.

        window: only tokens less than this far behind the token's own position (None or 0: all). softcap None or
        0.0 disables c*tanh(s/c); scale defaults to 1/sqrt(head_dim). Returns q's shape, as a view of [B, T, Hq, D]
        in memory: out.transpose(1, 2).reshape(B, T, -1) is the output projection's input and copies nothing.
        Zeros for columns that are not a row's own, for a token that sees nothing and for a head whose scores are all
        -inf. What the pages hold behind a row's new tokens does not matter, nor what they hold before the window of
        its first new one (nor whether those pages are there). A value in V that is not finite, of a token that some new
        token of the row sees, may reach all of the row's new tokens.

        The probabilities enter the product with V as two numbers of the cache's type, whose rounding does not show.
        A caller that may have them rounded to one, each off by up to half a step of the type, says so with
        ``exact_weights=False``: calls of more than 32 tokens times query heads per KV head then take up to a quarter
        less time (smaller ones, and all at head dim 16, keep the two, which cost nothing there)."""
        done = self._ops.pt_attend(self._address, self._index, layer, q, table, lengths, counts, tree, window, softcap, scale,
                                   exact_weights)
        if done is not None:
            N.nat.check(done[0], "PageTableCache.attend")
            return done[1]
        _inference_only(q)
        layer = self._layer(layer)
        x = self._new(q, self.num_query_heads, "q")
        b, t, d = x.shape[0], x.shape[2], self.head_dim
        rows, held = self._rows(table, lengths, counts, b, t)
        masks, depths = self._tree(tree, b, t)
        if window is not None and window < 0:
            raise ValueError(f"window must not be negative, got {window}")
        out = torch.empty((b, t, self.num_query_heads, d), dtype=self.dtype, device=self.device)
        nbytes = N.lib().pgr_pt_attend_workspace_bytes(self._ref, b, t, rows.width)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None
        with _on(self.device):
            N.nat.check(
                N.lib().pgr_pt_attend(
                    self._ref, layer, ctypes.byref(rows), x.data_ptr(), _strides(x, 3), out.data_ptr(), N.ptr(masks),
                    N.ptr(depths), min(int(window or 0), 1 << 31), 1.0 / d**0.5 if scale is None else float(scale),
                    float(softcap or 0.0), bool(exact_weights), N.ptr(ws), nbytes, N.stream_of(self.device),
                ),
                "PageTableCache.attend",
            )
        return out.transpose(1, 2) if q.dim() == 4 else out.squeeze(1)

    def keep(self, table: torch.Tensor, lengths: torch.Tensor, path: torch.Tensor) -> None:
        """The accepted path to the front, in every layer: new token path[b, j] becomes token lengths[b] + j.

        path [B, A] int32, up to 64 new tokens a row; all move at once, from where they were before the call. An
        entry outside [0, 64) leaves token j as it is (-1 behind the last). ``lengths`` stays as it is: the caller
        adds the number of accepted tokens."""
        done = self._ops.pt_keep(self._address, self._index, table, lengths, path)
        if done is not None:
            N.nat.check(done, "PageTableCache.keep")
            return
        if path.dim() != 2:
            raise ValueError(f"path must be [B, A], got {tuple(path.shape)}")
        b, t = path.shape
        if t > 64:
            raise NotImplementedError(f"a path has up to 64 tokens, got {t}")
        path = self._numbers(path, "path", (b, t))
        rows, held = self._rows(table, lengths, None, b, t)
        with _on(self.device):
            N.nat.check(N.lib().pgr_pt_keep(self._ref, ctypes.byref(rows), path.data_ptr(), N.stream_of(self.device)),
                        "PageTableCache.keep")
