"""The bounded cache's kernels where their loops run long: workgroups of many tiles, waves that come back for
more, rows of more slots and parts than the threads hold at once. Each case states how often its loop turns, from
the call's workspace, so that another plan of the launches cannot empty it."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import _pgr_native as nat
from oracle import bounded_cache as O
from pager_hf.heavy_hitter_cache import HeavyHitterCache, prompt_attention_weights

pytestmark = pytest.mark.gpu
STEP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TILE = 128  # keys or rows of a prompt's scores that a workgroup stages at a time


def _np(t):
    return t.detach().cpu().double().numpy()


def _within(got, ref, bound, what):
    err = np.abs(_np(got) - ref)
    assert np.all(err <= bound), f"{what}: off by {np.nanmax(err)}, {np.nanmax(err / np.maximum(bound, 1e-300)):.3g} x bound"


def _up(n):
    return (n + 255) // 256 * 256


def _ceil(a, b):
    return -(-a // b)


def _prompt_splits(b, hq, hkv, t, w, d):
    """(parts of the keys in the statistics, parts of the rows in the sums): the statistics' partial results (8 bytes
    a query row and part), the norms, and more than one part's sums make up the workspace."""
    have = nat.load().pgr_hh_prompt_weights_workspace_bytes(b, hq, hkv, t, w, d)
    rows, tiles, row_tiles = b * hq * w, _ceil(t, TILE), _ceil(w * (hq // hkv), TILE)
    fits = [(ks, rs) for ks in range(1, tiles + 1) for rs in range(1, row_tiles + 1)
            if _up(rows * ks * 8) + _up(rows * 4) + (_up(b * hkv * t * rs * 4) if rs > 1 else 0) == have]
    assert len(fits) == 1, fits
    return fits[0]


LONG_PROMPTS = [
    # batch, query heads, kv heads, head dim, tokens, window, padded
    (128, 16, 4, 64, 2048, 128, False),   # even parts; rounds of whole queries
    (64, 24, 8, 64, 2050, 190, True),     # three query heads a KV head: rows are not whole queries
    (64, 4, 4, 128, 2047, 700, True),     # one query head; two groups of rows and keys a wave
    (32, 16, 4, 256, 2048, 160, False),
    (256, 4, 2, 16, 1100, 300, True),
    (16, 12, 4, 64, 1025, 1025, True),    # every query
    (100, 8, 2, 128, 2000, 128, False),   # one group of rows and keys a wave at head dim 128
    (48, 16, 4, 128, 1024, 1024, False),
    (64, 4, 4, 256, 1030, 1030, True),
]


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("case", LONG_PROMPTS, ids=[str(c[:6]) for c in LONG_PROMPTS])
def test_prompt_weights_over_many_tiles(case, dtype):
    b, hq, hkv, d, t, w, padded = case
    ks, rs = _prompt_splits(b, hq, hkv, t, w, d)
    per = _ceil(_ceil(t, TILE), ks), _ceil(_ceil(w * (hq // hkv), TILE), rs)
    assert min(per) >= 4, (ks, rs, per)  # (two tiles fill both buffers, the fourth is read in the steady state)
    g = torch.Generator(device="cuda").manual_seed(91)
    q = torch.randn(b, w, hq, d, generator=g, device="cuda").to(dtype).transpose(1, 2)
    k = torch.randn(b, hkv, t, d, generator=g, device="cuda").to(dtype)
    lo = None
    if padded:
        lo = [0 if i % 3 == 0 else (37 * i) % t for i in range(b)]
        lo[-1] = t - w // 2
        cols = torch.arange(t, device="cuda")
        out = cols < torch.tensor(lo, device="cuda")[:, None]
        k.masked_fill_(out[:, None, :, None], float("nan"))
        q.masked_fill_(out[:, None, t - w:, None], float("nan"))
    got = prompt_attention_weights(q, k, lo=lo)
    for i, h in ((0, 0), (1, hkv - 1), (b - 1, 0)):
        ref, bound = O.prompt_weights(_np(q[i, h * (hq // hkv):(h + 1) * (hq // hkv)]), _np(k[i, h]), lo[i] if lo else 0,
                                      1.0 / d**0.5, 0.0)
        _within(got[i, h], ref, bound, f"row {i} head {h}")
    # The same rows alone, in other launches: another split of the same sums.
    alone = prompt_attention_weights(q[1:2], k[1:2], lo=lo[1:2] if lo else None)
    ref, bound = O.prompt_weights(_np(q[1, :hq // hkv]), _np(k[1, 0]), lo[1] if lo else 0, 1.0 / d**0.5, 0.0)
    _within(alone[0, 0], ref, bound, "alone")
    assert torch.equal(prompt_attention_weights(q, k, lo=lo), got)


def _attend_splits(cache):
    have = nat.load().pgr_hh_attend_workspace_bytes(cache._ref)
    heads, stride = cache.batch * cache.num_query_heads, _ceil(cache.capacity, 32) * 32
    fits = [n for n in range(1, 1025)
            if _up(heads * stride * 4) + 2 * _up(heads * n * 4) + _up(heads * n * cache.head_dim * 4) == have]
    assert len(fits) == 1, fits
    return fits[0]


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("case", [(64, 32, 8, 64, 4133), (64, 32, 8, 128, 4133), (32, 8, 8, 256, 4133), (128, 8, 4, 32, 3001),
                                  (256, 2, 2, 16, 2500)], ids=str)
def test_attend_over_many_tiles_of_a_wave(case, softcap, dtype):
    b, hq, hkv, d, c = case
    cache = HeavyHitterCache(b, hq, hkv, c, d, dtype, "cuda", keep_first=0, keep_recent=1)
    n_split = _attend_splits(cache)
    assert _ceil(c, 32) // n_split >= 16  # four tiles and more for each of four waves
    g = torch.Generator(device="cuda").manual_seed(92)
    cache.keys.normal_(generator=g)
    cache.values.normal_(generator=g)
    cache.weights.uniform_(0, 4, generator=g)
    lengths = torch.tensor([c - (53 * i) % c for i in range(b)], dtype=torch.int32, device="cuda")
    cache.lengths.copy_(lengths[:, None].expand(b, hkv))
    free = torch.arange(c, device="cuda") >= cache.lengths[..., None]
    for x in (cache.keys, cache.values):
        x.masked_fill_(free[..., None], float("nan"))
    before = cache.weights.clone()
    q = torch.randn(b, hq, d, generator=g, device="cuda").mul_(2).to(dtype)
    out = cache.attend(q, softcap=softcap)
    rep = hq // hkv
    for i, h in ((0, 0), (1, hkv - 1), (b // 2, 0), (b - 1, hkv - 1)):
        n = int(lengths[i])
        heads = slice(h * rep, (h + 1) * rep)
        ref, bound, new, new_bound = O.attend(_np(q[i, heads]), _np(cache.keys[i, h, :n]), _np(cache.values[i, h, :n]),
                                              _np(before[i, h, :n]), 1.0 / d**0.5, softcap, STEP[dtype])
        _within(out[i, heads], ref, bound, f"out row {i} head {h}")
        _within(cache.weights[i, h, :n], new, new_bound, f"weights row {i} head {h}")
    assert torch.equal(cache.weights[free], before[free])
    again = cache.weights.clone()
    cache.weights.copy_(before)
    assert torch.equal(cache.attend(q, softcap=softcap), out) and torch.equal(cache.weights, again)


@pytest.mark.parametrize("capacity", [4100, 12007])
def test_append_to_rows_of_more_slots_than_are_read_at_once(capacity):
    """4096 slots are asked for ahead; the lightest one lies behind them, before them, or in the odd ones at the end."""
    cache = HeavyHitterCache(3, 4, 2, capacity, 32, torch.float16, "cuda", keep_first=2, keep_recent=3)
    g = torch.Generator(device="cuda").manual_seed(93)
    cache.weights.uniform_(1, 2, generator=g)
    for row, at in enumerate((capacity - 1, capacity - 2, 4097, 4095, 7, capacity // 2)):
        cache.weights.view(6, -1)[row, at] = 0.5
        cache.order.view(6, -1)[row] = (torch.randperm(capacity, generator=g, device="cuda") + 2).int()
    cache.lengths.fill_(capacity)
    cache.seen.fill_(2 * capacity)
    w, order = _np(cache.weights), _np(cache.order)
    k = torch.randn(3, 2, 32, device="cuda").half()
    cache.append(torch.zeros(3, 4, 32, device="cuda").half(), k, k)
    for i in range(3):
        for h in range(2):
            slot = O.append_slot(capacity, 2 * capacity, w[i, h], order[i, h], capacity, 2, 3)
            assert w[i, h, slot] == 0.5
            assert torch.equal(cache.keys[i, h, slot], k[i, h]) and int(cache.order[i, h, slot]) == 2 * capacity


def test_load_prompt_of_more_parts_than_threads():
    """A row of more than 512 parts of 4096 tokens: each part's count of those before it takes a second turn."""
    t, c = 2_200_003, 5000
    assert _ceil(t, 4096) > 512
    cache = HeavyHitterCache(1, 2, 1, c, 16, torch.float16, "cuda", keep_first=4, keep_recent=100)
    g = torch.Generator(device="cuda").manual_seed(94)
    k = torch.randn(1, 1, t, 16, generator=g, device="cuda").half()
    w = torch.randint(0, 1 << 20, (1, 1, t), generator=g, device="cuda").float()  # (some are equal)
    cache.load_prompt(k, k, w)
    host = w[0, 0].cpu().numpy()
    free = np.arange(4, t - 100)
    heavy = free[np.argsort(-host[free], kind="stable")[: c - 104]]
    kept = np.sort(np.concatenate([np.arange(4), heavy, np.arange(t - 100, t)]))
    at = torch.from_numpy(kept).cuda()
    assert torch.equal(cache.order[0, 0], at.int()) and torch.equal(cache.weights[0, 0], w[0, 0, at])
    assert torch.equal(cache.keys[0, 0], k[0, 0, at]) and torch.equal(cache.values[0, 0], k[0, 0, at])
    assert int(cache.lengths) == c and int(cache.seen) == t
