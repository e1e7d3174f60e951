"""The operators of drafted tokens on the GPU, further: weights, depths, batches, softcaps, forms of a call, norms."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import drafted_tokens as O
from pager_hf import DraftTree, draft_tree
from pager_hf import _native as N
from pager_hf.rotary import norm_rotary_embedding, rotary_frequencies
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


LARGE = [
    # batch, query heads, kv heads, head dim, new tokens, window, long rows
    (300, 8, 2, 64, 1, 0, {100: 5000}), (1100, 16, 1, 32, 2, 0, {0: 2100, 700: 4000, 1099: 900}), (257, 16, 1, 64, 20, 0, {256: 3000}),
    (300, 8, 1, 256, 2, 0, {7: 1500}), (400, 4, 4, 128, 3, 500, {5: 2000, 6: 2000, 398: 700}), (2100, 4, 2, 16, 1, 0, {2099: 3000}),
    (1025, 2, 1, 64, 40, 0, {1024: 1300}),
]


@pytest.mark.parametrize("dtype", CACHE_TYPES)
@pytest.mark.parametrize("case", LARGE, ids=[str(c[:6]) for c in LARGE])
def test_long_rows_of_large_batches_are_cut(case, dtype):
    """Parts are listed by a launch of their own: rows of one part, of many and of none."""
    b, hq, hkv, d, t, window, longer = case
    rng = np.random.default_rng(109)
    lengths = [0 if i % 9 == 3 else int(x) for i, x in enumerate(rng.integers(0, 30, b))]
    for i, n in longer.items():
        lengths[i] = n
    pages = sum(-(-(n + t) // 32) for n in lengths) + 1
    cache, table = _filled(rng, pages, 32, hq, hkv, d, dtype, lengths, t, spare=520)
    assert N.lib().pgr_pt_attend_workspace_bytes(cache._ref, b, t, table.shape[1]) > 0
    counts = [t if i in longer else i % (t + 1) for i in range(b)]
    q = torch.randn(b, hq, t, d, generator=torch.Generator().manual_seed(6)).to(dtype).cuda()
    for _ in range(2):
        out = cache.attend(0, q, _int32(table), _int32(lengths), counts=_int32(counts), window=window)
        _check_attend(cache, 0, table, lengths, q, out, counts, *_order(b, t), window, 1.0 / d**0.5, 0.0, exact=True,
                      only=sorted({0, t // 2, t - 1}))
    assert not cache.attend(0, q, _int32(table), _int32(lengths), counts=_int32([0] * b), window=window).any()


def test_a_captured_call_of_a_large_batch_replays():
    """The parts are listed anew from the lengths of each replay."""
    rng = np.random.default_rng(149)
    b, most = 300, 2500
    cache, _ = _filled(rng, 80, 32, 8, 1, 64, torch.float16, [most], 3, garbage=False)
    table = _int32(np.concatenate([rng.permutation(79), np.full(500, -1)])[None]).expand(b, -1)  # (rows that share their pages)
    q = torch.randn(b, 8, 3, 64, generator=torch.Generator().manual_seed(6)).half().cuda()
    lengths = _int32([5] * b)
    cache.attend(0, q, table, lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = cache.attend(0, q, table, lengths)
    for i in range(4):
        now = rng.integers(0, 40, b)
        now[rng.integers(0, b, i)] = rng.integers(1000, most, i)
        lengths.copy_(_int32(now))
        want = cache.attend(0, q, table, lengths)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)
        torch.randn(1000, device="cuda").sort()  # eager work between the replays


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


# ---- softcaps ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", CACHE_TYPES)
@pytest.mark.parametrize("cap", [0.75, 20.0, 60.0, 64.0, 5000.0])
@pytest.mark.parametrize("t", [3, 60])
def test_a_softcap_is_as_near_as_the_score_not_as_the_cap(t, cap, dtype):
    """Two tokens whose weighted values all but cancel, scores of at most 2. Queries and keys of one component: the
    product is exact (8 + 8 bits in bf16, 11 + 2 in fp16). A score then has: the scale's quotient, its product with the cap's
    reciprocal and the last product with a constant of its own, half a step each, which tanh passes on no larger
    than relative to itself, and tanh's own 6; 4 for the softmax's difference and exponential, of a score of 2 at
    most. Two scores: twice that. The sums and quotient: 8 more."""
    rng = np.random.default_rng(113)
    cache, table = _filled(rng, 8, 16, 8, 2, 64, dtype, [2], t, garbage=False)
    p, o = (torch.tensor(x, device="cuda") for x in O.cells(table[0], 16, 8, 0, 2))
    keys = torch.zeros(2, 2, 64)
    keys[0, :, 0], keys[1, :, 0] = 1.0, 1.0 + 2.0**-6
    cache.keys[0][p, :, o] = keys.to(dtype).cuda()
    values = torch.ones(2, 2, 64)
    values[1] = -(1.0 + torch.linspace(-0.04, 0.04, 64)).to(dtype).float()
    cache.values[0][p, :, o] = values.to(dtype).cuda()
    q = torch.zeros(1, 8, t, 64)
    q[..., 0] = torch.rand(1, 8, t, generator=torch.Generator().manual_seed(5)) * 3.9 - 1.95
    q = q.to(dtype).cuda()
    none = _tree_of(np.zeros((1, t, t), bool), np.zeros((1, t), np.int64))  # (the new tokens see the held two alone)
    out = cache.attend(0, q, _int32(table), _int32([2]), tree=none, softcap=cap, scale=1.0)
    s = _np(q)[0, :, :, :1] * np.array([1.0, 1.0 + 2.0**-6])
    y = cap * np.tanh(s / cap)
    w = np.exp(y - y.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    v = _np(values)[:, 0]
    ref = w @ v
    bounds = _attend_bounds(dtype)
    rel = 2 * 14 * 2.0**-24 * np.abs(y).max(-1, keepdims=True) + 8 * 2.0**-24 + bounds["p_step"]
    bound = (w * rel) @ np.abs(v) + bounds["p_floor"] * 2
    bound = bound + STEP[dtype] * (np.abs(ref) + bound) + TINY[dtype]
    _within(out[0], ref, bound, f"cap {cap}")


@pytest.mark.parametrize("dtype", CACHE_TYPES)
@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("cap", [65.0, 200.0])
def test_softcaps_above_64(cap, d, dtype):
    """Scores on both sides of the cap's straight part; a row cut into parts and joined, short rows, many rows."""
    for lengths, hq, t, width in (([3000], 4, 1, 0), ([3000], 16, 9, 0), ([90, 3], 8, 5, 0), ([260], 8, 30, 4000)):
        rng = np.random.default_rng(127)
        pages = sum(-(-(n + t) // 16) for n in lengths) + 3
        cache, table = _filled(rng, pages, 16, hq, 1, d, dtype, lengths, t, spare=2 + width)
        b = len(lengths)
        q = (torch.randn(b, hq, t, d, generator=torch.Generator().manual_seed(4)) * 8).to(dtype).cuda()
        out = cache.attend(0, q, _int32(table), _int32(lengths), softcap=cap, scale=8.0 / d**0.5)
        _check_attend(cache, 0, table, lengths, q, out, None, *_order(b, t), 0, 8.0 / d**0.5, cap, exact=True)


@pytest.mark.parametrize("t", [1, 40])
def test_softcaps_at_the_ends_of_float32(t):
    """The largest change nothing; under the smallest all scores are alike, those of a key of zeros too."""
    cache, table = _filled(np.random.default_rng(151), 8, 16, 4, 1, 64, torch.float16, [20], t, garbage=False)
    p, o = O.cells(table[0], 16, 8, 0, 20 + t)
    cache.keys[0, int(p[3]), :, int(o[3])] = 0.0
    q = torch.randn(1, 4, t, 64, generator=torch.Generator().manual_seed(6)).half().cuda()
    want = cache.attend(0, q, _int32(table), _int32([20]))
    for cap in (3.4e38, 2.0**127, 2.0**100):
        assert torch.equal(cache.attend(0, q, _int32(table), _int32([20]), softcap=cap), want)
    for cap in (1e-40, 2.0**-149, 1e-37, 1e-30):
        out = cache.attend(0, q, _int32(table), _int32([20]), softcap=cap)
        _check_attend(cache, 0, table, [20], q, out, None, *_order(1, t), 0, 0.125, cap, exact=True)


def test_a_softcap_passes_infinities_and_nan_on():
    """Scores of both infinities are the cap's two ends; a score of NaN stays with its token and head."""
    for t in (1, 40):
        cache, table = _filled(np.random.default_rng(131), 8, 16, 4, 1, 64, torch.float16, [20], t, garbage=False)
        p, o = O.cells(table[0], 16, 8, 0, 20 + t)
        q = torch.rand(1, 4, t, 64, generator=torch.Generator().manual_seed(6)).half().cuda() + 0.1
        cache.keys[0, int(p[3]), :, int(o[3])] = float("inf")
        cache.keys[0, int(p[4]), :, int(o[4])] = float("-inf")
        out = cache.attend(0, q, _int32(table), _int32([20]), softcap=20.0)
        kn, vn, qn = _np(cache.keys[0]), _np(cache.values[0]), _np(q)
        kn[p[3], :, o[3]], kn[p[4], :, o[4]] = 1e9, -1e9  # (as good as infinite under the cap)
        ref, _ = O.attend_row(qn[0], kn[p, 0, o], vn[p, 0, o], np.ones(20 + t, bool), 20, t, _order(1, t)[0][0], np.arange(t), 0,
                              0.125, 20.0, **_attend_bounds(torch.float16))
        # (Two scores off by the product's roundings and by 10 half steps of the cap; sums and the exponent; P; the output.)
        plain = [i for i in range(20 + t) if i not in (3, 4)]
        size = (np.abs(qn[0]) @ np.abs(kn[p, 0, o][plain]).T).max() * 0.125
        off = (2 * (64 + 4) * size + 2 * 10 * 20.0 + 20 + t + 16 + 4 * 40.0) * 2.0**-24 + 3 * STEP[torch.float16] ** 2
        bound = off * np.abs(vn[p, 0, o]).max()
        _within(out[0], ref, bound + STEP[torch.float16] * (np.abs(ref) + bound) + TINY[torch.float16], "ends")
        bad = q.clone()
        bad[0, 2, t - 1, 5] = float("nan")
        got = cache.attend(0, bad, _int32(table), _int32([20]), softcap=20.0)
        assert torch.isnan(got[0, 2, t - 1]).all()
        got[0, 2, t - 1] = out[0, 2, t - 1]
        assert torch.equal(got, out)


# ---- forms of a call -----------------------------------------------------------------------------
def test_a_tree_may_be_a_plain_pair(path):
    cache, table = _filled(np.random.default_rng(137), 8, 16, 4, 2, 64, torch.float16, [20], 5, garbage=False)
    q = torch.randn(1, 4, 5, 64, generator=torch.Generator().manual_seed(6)).half().cuda()
    tree = draft_tree(_int32([[-1, 0, 0, 1, 3]]))
    inv, _ = rotary_frequencies(64, device="cuda")
    tab, ln = _int32(table), _int32([20])
    want = cache.append(0, q, q[:, :2], q[:, 2:], tab, ln, inv, tree=tree)
    assert torch.equal(cache.append(0, q, q[:, :2], q[:, 2:], tab, ln, inv, tree=(tree.masks, tree.depths)), want)
    want = cache.attend(0, q, tab, ln, tree=tree)
    assert torch.equal(cache.attend(0, q, tab, ln, tree=(tree.masks, tree.depths)), want)
    for bad in ((tree.masks,), (tree.masks, tree.depths, tree.depths), tree.masks, 3):
        with pytest.raises(TypeError, match="tree"):
            cache.attend(0, q, tab, ln, tree=bad)
        with pytest.raises(TypeError, match="tree"):
            cache.append(0, q, q[:, :2], q[:, 2:], tab, ln, inv, tree=bad)


def test_a_window_of_any_number(path):
    cache, table = _filled(np.random.default_rng(139), 8, 16, 4, 2, 64, torch.float16, [50], 2, garbage=False)
    q = torch.randn(1, 4, 2, 64, generator=torch.Generator().manual_seed(6)).half().cuda()
    want = cache.attend(0, q, _int32(table), _int32([50]))
    for window in (1 << 30, 1 << 31, (1 << 32) + 1, (1 << 63) - 1, 1 << 63, (1 << 64) + 1):
        assert torch.equal(cache.attend(0, q, _int32(table), _int32([50]), window=window), want), window


# ---- the norm ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,r", [(64, 64), (128, 32), (16, 8), (96, 24), (80, 20)])
def test_normed_heads_are_of_unit_size(d, r, interleaved, dtype):
    """Unit weights and no eps: a turn changes no length, so the root mean square is 1 to the output's rounding (and d + 30
    half steps of float32)."""
    x = (torch.randn(2, 3, 7, d, generator=torch.Generator().manual_seed(8)) * 5).to(dtype).cuda()
    inv, _ = rotary_frequencies(r, device="cuda")
    pos = torch.arange(7, device="cuda").repeat(2, 1) * 1000
    w = torch.ones(d, device="cuda").to(dtype)
    y, _ = norm_rotary_embedding(x, None, pos, inv, w, None, eps=0.0, interleaved=interleaved)
    rms = np.sqrt((_np(y) ** 2).mean(-1))
    assert np.all(np.abs(rms - 1) <= STEP[dtype] + (d + 30) * 2.0**-24)


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("r", [0, 64])
def test_a_head_with_an_infinite_element(r, dtype):
    """Its root mean square is infinite: that element (and the one that it turns with) is NaN, as inf * 0 is, the others are
    zeros; other heads do not see it."""
    x = torch.randn(1, 2, 3, 64, generator=torch.Generator().manual_seed(8)).to(dtype).cuda()
    w = torch.ones(64, device="cuda").to(dtype)
    inv = rotary_frequencies(64, device="cuda")[0] if r else torch.empty(0, device="cuda")
    pos = torch.arange(5, 8, device="cuda")[None]
    want, _ = norm_rotary_embedding(x, None, pos, inv, w, None)
    x[0, 1, 2, 7] = float("inf")
    y, _ = norm_rotary_embedding(x, None, pos, inv, w, None)
    bad = [7, 39] if r else [7]
    assert torch.isnan(y[0, 1, 2, bad]).all()
    y[0, 1, 2, bad] = 0.0
    assert not y[0, 1, 2].any()
    y[0, 1, 2] = want[0, 1, 2]
    assert torch.equal(y, want)
