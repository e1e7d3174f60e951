"""The operators of drafted tokens on the GPU, further: weights, depths, batches, softcaps, forms of a call, norms."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import drafted_tokens as O
from pager_hf import DraftTree
from pager_hf import _native as N
from pager_hf.rotary import rotary_frequencies
from test_verify_drafts_gpu import CACHE_TYPES, STEP, TINY, _attend_bounds, _check_attend, _filled, _int32, _np, _order, _within

pytestmark = pytest.mark.gpu


def _tree_of(sees, depth):
    t = sees.shape[-1]
    masks = (sees * (np.uint64(1) << np.arange(t, dtype=np.uint64))).sum(axis=-1, dtype=np.uint64)
    return DraftTree(torch.tensor(masks.view(np.int64), device="cuda"), torch.tensor(depth, dtype=torch.int32, device="cuda"))


class _General:
    """No call is a plain one: all go through Python."""

    def __getattr__(self, name):
        return lambda *args: None


@pytest.fixture(params=["native", "general"])
def path(request, monkeypatch):
    if request.param == "general":
        monkeypatch.setattr(N, "_ops", _General())
    return request.param


# ---- the weights' bits ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", CACHE_TYPES)
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_many_rows_keep_the_weights_unless_told_otherwise(d, dtype, path):
    """160 rows a KV head, sums that all but cancel: weights rounded to the cache's type are off by several times the
    bound, and are rounded so only where the caller says that they may be."""
    t = 40
    rng = np.random.default_rng(29)
    cache, table = _filled(rng, 8, 16, 8, 2, d, dtype, [24], t)
    p, o = (torch.tensor(x, device="cuda") for x in O.cells(table[0], 16, 8, 0, 24 + t))
    values = torch.randn(24 + t, 2, d, generator=torch.Generator().manual_seed(3)).to(dtype)
    values[1::2] = -values[: 24 + t - 1: 2][: values[1::2].shape[0]]
    cache.values[0][p, :, o] = values.cuda()
    q = (torch.randn(1, 8, t, d, generator=torch.Generator().manual_seed(4)) / 8).to(dtype).cuda()
    for more, exact in ((dict(), True), (dict(exact_weights=True), True), (dict(exact_weights=False), False)):
        out = cache.attend(0, q, _int32(table), _int32([24]), **more)
        _check_attend(cache, 0, table, [24], q, out, None, *_order(1, t), 0, 1.0 / d**0.5, 0.0, exact=exact)


# ---- depths --------------------------------------------------------------------------------------
DEPTHS = [0, 63, 64, 100, 149, 150, 151, 999, 1 << 20, (1 << 31) - 1, -1, -100]


@pytest.mark.parametrize("window", [1, 100, 150, 1 << 30])
@pytest.mark.parametrize("hq,t", [(4, 12), (16, 12), (8, 60)])
def test_a_window_goes_by_depths_of_any_size(hq, t, window):
    """A tree made by hand: its depths are what they say, however large; those below 0 count as 0."""
    rng = np.random.default_rng(101)
    lengths = [1000, 20, 0]
    cache, table = _filled(rng, 40, 32, hq, 2, 64, torch.float16, lengths, t, garbage=False)
    depth = rng.choice(DEPTHS, (3, t))
    depth[:, : min(t, 12)] = DEPTHS[: min(t, 12)]
    sees = rng.random((3, t, t)) < 0.5
    sees[:, np.arange(t), np.arange(t)] = True
    q = torch.randn(3, hq, t, 64, generator=torch.Generator().manual_seed(6)).half().cuda()
    out = cache.attend(0, q, _int32(table), _int32(lengths), tree=_tree_of(sees, depth), window=window)
    _check_attend(cache, 0, table, lengths, q, out, None, sees, np.maximum(depth, 0), window, 0.125, 0.0, exact=True)


@pytest.mark.parametrize("norm", [False, True])
def test_append_goes_by_depths_of_any_size(norm):
    rng = np.random.default_rng(103)
    depth = np.array([[0, 63, 64, 1 << 20, -1, -100]])
    t, dtype = depth.shape[1], torch.float16
    cache, table = _filled(rng, 4, 16, 4, 2, 64, dtype, [30], t, garbage=False)
    g = torch.Generator().manual_seed(7)
    q, k = torch.randn(1, 4, t, 64, generator=g).half().cuda(), torch.randn(1, 2, t, 64, generator=g).half().cuda()
    inv, _ = rotary_frequencies(64, device="cuda")
    w = torch.ones(64, device="cuda").half() if norm else None
    out = cache.append(0, q, k, k, _int32(table), _int32([30]), inv, tree=_tree_of(np.ones((1, t, t), bool), depth), q_weight=w,
                       k_weight=w)
    pos = 30 + np.maximum(depth, 0)
    p, o = (torch.tensor(x, device="cuda") for x in O.cells(table[0], 16, 4, 30, t))
    for got, x in ((out[0], q), (cache.keys[0][p, :, o].transpose(0, 1), k)):
        ref, bound = O.norm_rotate(_np(x), None if w is None else _np(w), 1e-6, pos[:, None], _np(inv))
        _within(got[None], ref, bound + STEP[dtype] * (np.abs(ref) + bound) + TINY[dtype], "turned")


# ---- batches -------------------------------------------------------------------------------------
@pytest.mark.parametrize("window", [0, 70])
def test_attend_over_more_than_a_thousand_rows(window):
    """One KV head, ragged rows, one of them long."""
    rng = np.random.default_rng(107)
    b, t, dtype = 1100, 2, torch.float16
    lengths = [int(x) for x in rng.integers(0, 40, b)]
    lengths[700] = 4000
    pages = sum(-(-(n + t) // 32) for n in lengths) + 1
    cache, table = _filled(rng, pages, 32, 16, 1, 32, dtype, lengths, t)
    counts = [i % 4 for i in range(b)]  # 3: all of them
    q = torch.randn(b, 16, t, 32, generator=torch.Generator().manual_seed(6)).to(dtype).cuda()
    out = cache.attend(0, q, _int32(table), _int32(lengths), counts=_int32(counts), window=window)
    _check_attend(cache, 0, table, lengths, q, out, counts, *_order(b, t), window, 1.0 / 32**0.5, 0.0, exact=True)


@pytest.mark.parametrize("tokens", [2048, 2049])
def test_prompts_of_one_token_more(tokens):
    """A prompt into an empty cache whose blocks of rows just fill the card, and one token more."""
    rng = np.random.default_rng(109)
    cache, table = _filled(rng, 70, 32, 32, 8, 64, torch.bfloat16, [0], tokens)
    q = torch.randn(1, 32, tokens, 64, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    out = cache.attend(0, q, _int32(table), _int32([0]))
    sees, depth = _order(1, tokens)
    kn, vn, qn = (x[0].double() for x in (cache.keys, cache.values, q))
    p, o = (torch.tensor(x, device="cuda") for x in O.cells(table[0], 32, 70, 0, tokens))
    for at in (0, 1, 63, 64, 65, 1000, 2046, tokens - 1):
        for h in (0, 7):
            ref, bound = O.attend_row(_np(qn[4 * h: 4 * h + 4, at: at + 1]), _np(kn[p, h, o][: at + 1]), _np(vn[p, h, o][: at + 1]),
                                      np.ones(at + 1, bool), at, 1, sees[0, :1, :1], depth[0, :1], 0, 0.125, 0.0,
                                      **_attend_bounds(torch.bfloat16))
            _within(out[0, 4 * h: 4 * h + 4, at: at + 1], ref, bound, f"token {at} head {h}")
