"""The bounded cache on the GPU against the 64-bit oracle, operator by operator and as a run."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import bounded_cache as O
from pager_hf.heavy_hitter_cache import HeavyHitterCache, prompt_attention_weights
from pager_hf.rotary import rotary_embedding, rotary_frequencies

pytestmark = pytest.mark.gpu
STEP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
STATE = ("keys", "values", "weights", "order", "lengths", "seen")


def _np(t):
    return t.detach().cpu().double().numpy()


def _within(got, ref, bound, what):
    got = _np(got) if isinstance(got, torch.Tensor) else got
    err = np.abs(got - ref)
    assert np.all(err <= bound), f"{what}: off by {np.nanmax(err)}, {np.nanmax(err / np.maximum(bound, 1e-300)):.3g} x bound"


def _state(cache):
    return {n: getattr(cache, n).clone() for n in STATE}


def _same(cache, state, *names):
    for n in names or STATE:
        a, b = getattr(cache, n), state[n]
        assert torch.equal(a.view(torch.int16) if a.dtype in STEP else a.view(torch.int32) if a.is_floating_point() else a,
                           b.view(torch.int16) if b.dtype in STEP else b.view(torch.int32) if b.is_floating_point() else b), n


def _filled(b, hq, hkv, c, d, dtype, lengths, seed, garbage=False, **keep):
    """A cache of random tokens; garbage: NaN in the slots that hold nothing."""
    g = torch.Generator().manual_seed(seed)
    cache = HeavyHitterCache(b, hq, hkv, c, d, dtype, "cuda", **keep)
    cache.keys.copy_(torch.randn(b, hkv, c, d, generator=g))
    cache.values.copy_(torch.randn(b, hkv, c, d, generator=g))
    cache.weights.copy_(torch.rand(b, hkv, c, generator=g) * 4)
    cache.lengths.copy_(torch.tensor(lengths, dtype=torch.int32)[:, None].expand(b, hkv))
    cache.seen.copy_(cache.lengths)
    cache.order.copy_(torch.arange(c).expand(b, hkv, c))
    if garbage:
        free = torch.arange(c, device="cuda") >= cache.lengths[..., None]
        for t in (cache.keys, cache.values):
            t.masked_fill_(free[..., None], float("nan"))
        cache.weights.masked_fill_(free, float("nan"))
    return cache, g


# ---- attend --------------------------------------------------------------------------------------
ATTEND = [
    # batch, query heads, kv heads, head dim, capacity, lengths
    (1, 14, 2, 64, 256, [256]),
    (4, 4, 2, 16, 65, [0, 1, 64, 65]),
    (5, 12, 2, 128, 333, [0, 15, 16, 17, 333]),
    (3, 16, 1, 32, 1000, [63, 640, 999]),
    (2, 8, 1, 256, 203, [203, 70]),
    (2, 16, 16, 64, 130, [129, 3]),
    (1, 1, 1, 128, 1, [1]),
    (2, 28, 4, 128, 4133, [4133, 1025]),
    (1, 16, 1, 64, 16387, [16387]),
    (40, 16, 8, 64, 70, [i * 70 // 39 for i in range(40)]),
    (65, 8, 8, 64, 300, [i * 300 // 64 for i in range(65)]),
    (2, 8, 1, 256, 1025, [1025, 0]),
    (3, 8, 1, 256, 300, [300, 257, 0]),
    (1, 8, 4, 128, 512, [511]),
]


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("softcap", [0.0, 5.0])
@pytest.mark.parametrize("case", ATTEND, ids=[str(c[:5]) for c in ATTEND])
def test_attend(case, dtype, softcap):
    b, hq, hkv, d, c, lengths = case
    cache, g = _filled(b, hq, hkv, c, d, dtype, lengths, 11, garbage=True, keep_first=0, keep_recent=1)
    before = _state(cache)
    # Queries as views into a larger tensor.
    q = (torch.randn(b, hq + 2, d + 8, generator=g) * 2).to(dtype).cuda()[:, 1:-1, :d]
    out = cache.attend(q, softcap=softcap)
    _same(cache, before, "keys", "values", "order", "lengths", "seen")
    rep, scale = hq // hkv, 1.0 / d**0.5
    k, v, w, qn = _np(cache.keys), _np(cache.values), _np(before["weights"]), _np(q)
    for i in range(b):
        n = lengths[i]
        for h in range(hkv):
            heads = slice(h * rep, (h + 1) * rep)
            ref, bound, new, new_bound = O.attend(qn[i, heads], k[i, h, :n], v[i, h, :n], w[i, h, :n], scale, softcap,
                                                  STEP[dtype])
            _within(out[i, heads], ref, bound, f"out row {i} head {h}")
            _within(cache.weights[i, h, :n], new, new_bound, f"weights row {i} head {h}")
            assert torch.isnan(cache.weights[i, h, n:]).all()


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("capacity", [200, 2000])
def test_attend_keeps_more_of_p_than_the_cache_type(d, capacity, dtype):
    """P enters the product with V as a part cut off after it was lowered by half a step, and the rest, rounded:
    with half a step u the rest is at most p u + 2 u p, its rounding 3 u^2 p. Under fp16 P's largest value is
    2^14, so that half of the smallest subnormal is 2^-39 of it. Few tokens of like weights, whose sums all but
    cancel in some dims: rounding P to the type itself is off by several times the bound."""
    n, u = 24, STEP[dtype]
    cache, g = _filled(4, 8, 2, capacity, d, dtype, [n] * 4, 15, keep_first=0, keep_recent=1)
    q = (torch.randn(4, 8, d, generator=g) / 8).to(dtype).cuda()
    out = cache.attend(q)
    for i in range(4):
        for h in range(2):
            heads = slice(4 * h, 4 * h + 4)
            ref, bound, _, _ = O.attend(_np(q[i, heads]), _np(cache.keys[i, h, :n]), _np(cache.values[i, h, :n]),
                                        np.zeros(n), 1.0 / d**0.5, 0.0, u, p_step=3 * u * u, p_floor=2.0**-39)
            _within(out[i, heads], ref, bound, f"row {i} head {h}")


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("d,capacity", [(16, 90), (64, 300), (64, 2000), (256, 900)])
def test_attend_over_infinite_values(d, capacity, dtype):
    """A value of inf or -inf makes its dim that, however small its token's weight or exact in the type."""
    cache, g = _filled(2, 4, 2, capacity, d, dtype, [capacity, 1], 16, keep_first=0, keep_recent=1)
    q = torch.randn(2, 4, d, generator=g).to(dtype).cuda()
    want = cache.attend(q)
    cache.values[:, :, 0, 3] = float("inf")  # (row 1 holds this token alone: its weight is 1)
    cache.values[0, :, 77, 5] = -float("inf")
    out = cache.attend(q)
    assert torch.equal(out[:, :, 3], torch.full_like(out[:, :, 3], float("inf")))
    assert torch.equal(out[0, :, 5], torch.full_like(out[0, :, 5], -float("inf")))
    for i, dims in ((0, (3, 5)), (1, (3,))):
        rest = [e for e in range(d) if e not in dims]
        assert torch.equal(out[i][:, rest], want[i][:, rest])


def test_attend_with_a_few_heavy_and_far_scores():
    """Scores spread over hundreds: the running maximum moves, most weights underflow."""
    cache, g = _filled(1, 4, 1, 700, 64, torch.float16, [700], 3, keep_first=0, keep_recent=1)
    cache.keys.mul_(6)
    w = _np(cache.weights)
    q = (torch.randn(1, 4, 64, generator=g) * 8).half().cuda()
    out = cache.attend(q, scale=0.5)
    ref, bound, new, nb = O.attend(_np(q)[0], _np(cache.keys)[0, 0], _np(cache.values)[0, 0], w[0, 0], 0.5, 0.0,
                                   STEP[torch.float16])
    _within(out[0], ref, bound, "out")
    _within(cache.weights[0, 0], new, nb, "weights")


@pytest.mark.parametrize("d,capacity", [(16, 400), (64, 300), (64, 2000), (256, 200), (256, 900)])
def test_attend_with_scores_of_minus_infinity(d, capacity):
    """Scores of -inf weigh nothing: a head that has no others gives zeros and no weight to any token, and takes
    none from the other heads; tokens that have no others weigh nothing, in whole tiles and beside others."""
    for lone in (True, False):
        cache, g = _filled(2, 4, 1, capacity, d, torch.bfloat16, [capacity] * 2, 17, keep_first=0, keep_recent=1)
        q = torch.randn(2, 4, d, generator=g).bfloat16()
        q[..., 0] = 0.0
        cache.keys[1, 0, :, 0] = -2.0**120
        q[1, 1, 0] = 2.0**100  # the products are past float32, the other heads' are 0
        if not lone:
            q[1, :, 0] = 2.0**100
        before = _state(cache)
        out = cache.attend(q.cuda())
        _same(cache, before, "keys", "values", "order", "lengths", "seen")
        assert not out[1, 1].any()
        if not lone:
            assert not out[1].any()
            assert torch.equal(cache.weights[1], before["weights"][1])
        k, v, w, qn = _np(cache.keys), _np(cache.values), _np(before["weights"]), _np(q)
        k[..., 0] = 0.0
        for i, heads in ((0, [0, 1, 2, 3]), (1, [0, 2, 3])):
            if i == 1 and not lone:
                continue
            ref, bound, new, new_bound = O.attend(qn[i, heads], k[i, 0], v[i, 0], w[i, 0], 1.0 / d**0.5, 0.0,
                                                  STEP[torch.bfloat16])
            _within(out[i, heads], ref, bound, f"out {i}")
            _within(cache.weights[i, 0], new, new_bound, f"weights {i}")
    # Tokens without weight beside others.
    cache, g = _filled(1, 4, 1, capacity, d, torch.float16, [capacity], 18, keep_first=0, keep_recent=1)
    q = torch.randn(1, 4, d, generator=g).half()
    q[..., 0] = 1.0
    gone = torch.zeros(capacity, dtype=torch.bool)
    gone[:70], gone[75], gone[128:160] = True, True, True
    cache.keys[0, 0, gone.cuda(), 0] = -float("inf")
    w = _np(cache.weights)[0, 0]
    out = cache.attend(q.cuda())
    at = (~gone).numpy()
    ref, bound, new, new_bound = O.attend(_np(q)[0], _np(cache.keys)[0, 0][at], _np(cache.values)[0, 0][at], w[at],
                                          1.0 / d**0.5, 0.0, STEP[torch.float16])
    _within(out[0], ref, bound, "out")
    got = _np(cache.weights)[0, 0]
    _within(got[at], new, new_bound, "weights")
    assert np.array_equal(got[~at], w[~at])


@pytest.mark.parametrize("d,capacity", [(64, 300), (64, 2000), (256, 200), (256, 900)])
def test_attend_over_tokens_that_are_nan(d, capacity):
    """Keys of NaN in a row's tokens make that row NaN, a whole tile of them and nothing else too; others stay."""
    for first, last in ((64, 96), (0, 150), (37, 38), (0, capacity)):
        cache, g = _filled(3, 4, 2, capacity, d, torch.bfloat16, [capacity] * 3, 13, keep_first=0, keep_recent=1)
        before = _state(cache)
        cache.keys[1, 0, first:last] = float("nan")
        q = torch.randn(3, 4, d, generator=g).bfloat16().cuda()
        out, weights = cache.attend(q), cache.weights.clone()
        assert torch.isnan(out[1, :2]).all() and torch.isnan(weights[1, 0]).all(), (first, last)
        cache.keys.copy_(before["keys"])
        cache.weights.copy_(before["weights"])
        want = cache.attend(q)
        for i, h in ((0, 0), (0, 1), (1, 1), (2, 0), (2, 1)):
            assert torch.equal(out[i, 2 * h:2 * h + 2], want[i, 2 * h:2 * h + 2])
            assert torch.equal(weights[i, h], cache.weights[i, h])


def test_attend_is_the_same_every_time():
    cache, g = _filled(2, 8, 2, 3000, 128, torch.bfloat16, [3000, 1234], 4)
    q = torch.randn(2, 8, 128, generator=g).bfloat16().cuda()
    before = cache.weights.clone()
    first, w = cache.attend(q), cache.weights.clone()
    for _ in range(5):
        cache.weights.copy_(before)
        assert torch.equal(cache.attend(q), first) and torch.equal(cache.weights, w)


def test_offsets_past_32_bits():
    """The last rows of a cache of more than 2^32 bytes and 2^31 elements of keys."""
    b, hkv, c, d = 9, 1, 1 << 20, 256
    cache = HeavyHitterCache(b, 2, hkv, c, d, torch.float16, "cuda", keep_first=0, keep_recent=1)
    assert cache.keys.numel() > 1 << 31
    g = torch.Generator().manual_seed(1)
    n = 50
    cache.keys[-1, 0, :n] = torch.randn(n, d, generator=g).half().cuda()
    cache.values[-1, 0, :n] = torch.randn(n, d, generator=g).half().cuda()
    cache.lengths[-1] = n
    q = torch.randn(b, 2, d, generator=g).half().cuda()
    out = cache.attend(q)
    ref, bound, new, nb = O.attend(_np(q[-1]), _np(cache.keys[-1, 0, :n]), _np(cache.values[-1, 0, :n]), np.zeros(n),
                                   1 / 16, 0.0, STEP[torch.float16])
    _within(out[-1], ref, bound, "out")
    _within(cache.weights[-1, 0, :n], new, nb, "weights")
    assert not out[:-1].any()
    cache.lengths[-1] = c  # full: the lightest slot is the first of the untouched ones
    cache.seen[-1] = c
    k = torch.randn(b, 1, d, generator=g).half().cuda()
    cache.append(q, k, k)
    assert torch.equal(cache.keys[-1, 0, n], k[-1, 0]) and cache.order[-1, 0, n] == c
    assert torch.equal(cache.keys[0, 0, 0], k[0, 0]) and cache.lengths[0, 0] == 1


# ---- append --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("case", [(1, 14, 2, 64, 256, 64), (3, 4, 2, 16, 20, 8), (4, 12, 2, 128, 1031, 128),
                                  (2, 8, 1, 256, 4099, 128), (2, 16, 16, 64, 33, 62), (2, 16, 1, 32, 6, 32)],
                         ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(case, dtype, interleaved):
    b, hq, hkv, d, c, r = case
    lengths = [c] * b
    if b > 2:
        lengths[1] = c - 2
    cache, g = _filled(b, hq, hkv, c, d, dtype, lengths, 21, keep_first=2, keep_recent=4)
    # Full rows have seen more than they hold, out of order, with weights that tie and a few NaN.
    for i in range(b):
        if lengths[i] == c:
            for h in range(hkv):
                cache.order[i, h] = torch.randperm(2 * c, generator=g)[:c].int()
            cache.seen[i] = 2 * c
    cache.weights.copy_((cache.weights * 2).round() / 2)
    cache.weights[:, :, 3] = float("nan")
    inv, factor = rotary_frequencies(r, device="cuda")
    for step in range(4):
        before = _state(cache)
        # Views of one projection, as a fused q/k/v product gives them.
        x = torch.randn(b, (hq + 2 * hkv) * d, generator=g).to(dtype).cuda()
        q, k, v = (t.view(b, -1, d) for t in x.split([hq * d, hkv * d, hkv * d], dim=1))
        positions = None if step % 2 == 0 else torch.randint(0, 1 << 18, (b,), generator=g).cuda()
        got = cache.append(q, k, v, inv, positions=positions, interleaved=interleaved, factor=1.5)
        pos = before["seen"][:, 0] if positions is None else positions
        want_q, want_k = rotary_embedding(q, k, pos, inv, interleaved=interleaved, factor=1.5)
        assert torch.equal(got, want_q)
        for i in range(b):
            for h in range(hkv):
                slot = O.append_slot(int(before["lengths"][i, h]), int(before["seen"][i, h]),
                                     _np(before["weights"][i, h]), _np(before["order"][i, h]), c, 2, 4)
                before["keys"][i, h, slot], before["values"][i, h, slot] = want_k[i, h], v[i, h]
                before["weights"][i, h, slot], before["order"][i, h, slot] = 0.0, before["seen"][i, h]
        before["lengths"].add_(1).clamp_(max=c)
        before["seen"].add_(1)
        _same(cache, before)


def test_append_without_rotation_returns_the_queries():
    cache, g = _filled(2, 4, 2, 8, 32, torch.float16, [0, 8], 5, keep_first=1, keep_recent=2)
    q, k, v = (torch.randn(2, h, 32, generator=g).half().cuda() for h in (4, 2, 2))
    assert cache.append(q, k, v) is q
    assert torch.equal(cache.keys[0, :, 0], k[0]) and torch.equal(cache.values[0, :, 0], v[0])
    assert cache.lengths.tolist() == [[1, 1], [8, 8]] and cache.seen.tolist() == [[1, 1], [9, 9]]
    strided = torch.randn(2, 32, 4, generator=g).half().cuda().transpose(1, 2)  # head_dim not contiguous
    assert torch.equal(cache.append(strided, k, v), strided)


def test_append_without_rotation_returns_strided_queries_themselves():
    cache = HeavyHitterCache(2, 4, 2, 48, 32, torch.float16, "cuda")
    q = torch.randn(2, 32, 4, device="cuda").half().transpose(1, 2)  # head_dim not contiguous
    k = torch.randn(2, 2, 32, device="cuda").half()
    assert cache.append(q, k, k) is q
    assert cache.lengths.tolist() == [[1, 1], [1, 1]]


def test_what_the_kernels_go_by_is_fixed():
    import copy

    cache = HeavyHitterCache(2, 4, 2, 64, 32, torch.float16, "cuda", keep_first=3, keep_recent=5)
    assert (cache.batch, cache.num_query_heads, cache.num_kv_heads, cache.capacity, cache.head_dim) == (2, 4, 2, 64, 32)
    assert (cache.keep_first, cache.keep_recent, cache.dtype, cache.device) == (3, 5, torch.float16, torch.device("cuda", 0))
    for name in ("batch", "capacity", "dtype", "device", *STATE):
        with pytest.raises(AttributeError):
            setattr(cache, name, getattr(cache, name))
    with pytest.raises((ValueError, TypeError)):  # a copy would hold the original's addresses
        copy.deepcopy(cache)


def test_a_cache_made_under_inference_mode_can_be_reset_outside():
    with torch.inference_mode():
        cache = HeavyHitterCache(1, 2, 1, 48, 32, torch.float16, "cuda")
        k = torch.ones(1, 1, 32, device="cuda").half()
        cache.append(torch.ones(1, 2, 32, device="cuda").half(), k, k)
    assert int(cache.lengths) == 1
    cache.reset()
    assert int(cache.lengths) == 0 and int(cache.seen) == 0


def test_a_cache_of_one_slot():
    cache = HeavyHitterCache(1, 1, 1, 1, 16, torch.float16, "cuda", keep_first=0, keep_recent=1)
    for n in range(3):
        k = torch.full((1, 1, 16), n + 1.0, dtype=torch.float16, device="cuda")
        cache.append(k, k, k)
        assert torch.equal(cache.attend(k), k)
        assert (int(cache.lengths), int(cache.seen), int(cache.order), float(cache.weights)) == (1, n + 1, n, 1.0)


# ---- prompt weights ------------------------------------------------------------------------------
PROMPT = [
    # batch, query heads, kv heads, head dim, tokens, window, lo
    (1, 4, 2, 64, 1, 1, None),
    (2, 14, 2, 64, 77, 5, [0, 30]),
    (3, 4, 2, 16, 130, 130, [0, 129, 130]),
    (1, 12, 2, 128, 515, 64, None),
    (2, 8, 1, 256, 300, 33, [299, 1]),
    (1, 16, 1, 32, 1000, 17, None),
    (1, 16, 16, 64, 257, 257, None),
    (2, 28, 4, 128, 384, 200, [128, 200]),
    (1, 8, 1, 256, 260, 260, [100]),
    (1, 1, 1, 128, 2500, 1, None),
    (8, 128, 8, 128, 300, 128, [0, 0, 5, 40, 171, 200, 299, 300]),  # two groups of rows and keys per wave
]


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("softcap", [0.0, 5.0])
@pytest.mark.parametrize("case", PROMPT, ids=[str(c[:6]) for c in PROMPT])
def test_prompt_weights(case, dtype, softcap):
    b, hq, hkv, d, t, w, lo = case
    g = torch.Generator().manual_seed(31)
    # [B, T, H, D] seen as [B, H, T, D]; the window is a slice of all queries.
    q = (torch.randn(b, t, hq, d, generator=g) * 2).to(dtype).cuda().transpose(1, 2)[:, :, t - w:]
    k = torch.randn(b, t, hkv, d, generator=g).to(dtype).cuda().transpose(1, 2)
    if lo is not None:  # what the padding holds does not matter
        for i in range(b):
            k[i, :, : lo[i]] = float("nan")
            q[i, :, : max(0, lo[i] - (t - w))] = float("nan")
    forms = [lo] if lo is None else [lo, torch.tensor(lo, device="cuda")]
    for form in forms:
        got = prompt_attention_weights(q, k, lo=form, softcap=softcap)
        assert got.dtype == torch.float32 and got.is_contiguous()
        for i in range(b):
            for h in range(hkv):
                qn = _np(q[i, h * (hq // hkv):(h + 1) * (hq // hkv)])
                ref, bound = O.prompt_weights(qn, _np(k[i, h]), lo[i] if lo else 0, 1.0 / d**0.5, softcap)
                _within(got[i, h], ref, bound, f"row {i} head {h}")


@pytest.mark.parametrize("d", [16, 128, 256])
@pytest.mark.parametrize("w", [3, 700])
def test_prompt_weights_of_scores_of_minus_infinity(d, w):
    """Keys whose every score is -inf weigh nothing, in whole tiles and beside others; no mask is involved."""
    g = torch.Generator().manual_seed(12)
    t, hq, hkv = 1500, 4, 2
    q = torch.randn(1, hq, w, d, generator=g).to(torch.bfloat16)
    k = torch.randn(1, hkv, t, d, generator=g).to(torch.bfloat16)
    q[..., 0] = 1.0
    gone = torch.zeros(t, dtype=torch.bool)
    gone[:650], gone[701], gone[1408:1440] = True, True, True
    k[:, :, gone, 0] = -float("inf")
    got = prompt_attention_weights(q.cuda(), k.cuda())
    assert not got[:, :, gone].any()
    for h in range(hkv):
        qn, ref, bound = _np(q[0, 2 * h:2 * h + 2]), np.zeros(t), np.zeros(t)
        for i in range(w):
            last = t - w + i
            at = np.flatnonzero(~gone[:last + 1].numpy())
            r, e = O.prompt_weights(qn[:, i:i + 1], _np(k[0, h])[at], 0, 1.0 / d**0.5, 0.0)
            ref[at], bound[at] = ref[at] + r, bound[at] + e
        _within(got[0, h], ref, bound + 2 * w * 2.0**-24 * ref, f"head {h}")  # (the sum over the queries)


def test_prompt_weights_of_more_than_2_to_the_30_query_rows():
    """Within the stated limits, and more than one dimension of a launch holds at four threads a row. Every
    batch row is the same one (expanded, so that the operands stay small)."""
    b, hq, d, t = 65535, 16, 16, 1025
    assert b * hq * t > 1 << 30
    g = torch.Generator().manual_seed(13)
    q = torch.randn(1, hq, t, d, generator=g).half().cuda()
    k = torch.randn(1, 1, t, d, generator=g).half().cuda()
    got = prompt_attention_weights(q.expand(b, hq, t, d), k.expand(b, 1, t, d))
    ref, bound = O.prompt_weights(_np(q[0]), _np(k[0, 0]), 0, 0.25, 0.0)
    _within(got[0, 0], ref, bound, "row 0")
    assert torch.equal(got, got[:1].expand_as(got))


def test_prompt_weights_are_the_same_every_time():
    g = torch.Generator().manual_seed(6)
    q = torch.randn(1, 8, 700, 64, generator=g).half().cuda()
    k = torch.randn(1, 2, 3000, 64, generator=g).half().cuda()
    first = prompt_attention_weights(q, k)
    for _ in range(4):
        assert torch.equal(prompt_attention_weights(q, k), first)
    assert abs(first.double().sum().item() - 8 * 700) < 8 * 700 * 1e-5


def test_prompt_weights_refusals():
    q, k = torch.zeros(1, 4, 9, 32, device="cuda").half(), torch.zeros(1, 2, 8, 32, device="cuda").half()
    with pytest.raises(ValueError, match="window"):
        prompt_attention_weights(q, k)
    with pytest.raises(ValueError, match="window"):
        prompt_attention_weights(q[:, :, :0], k)
    with pytest.raises(NotImplementedError, match="head_dim"):
        prompt_attention_weights(q[:, :, :8, :24], k[..., :24])
    with pytest.raises(ValueError, match="scale"):
        prompt_attention_weights(q[:, :, :8], k, scale=-1.0)
    with pytest.raises(ValueError, match="lo"):
        prompt_attention_weights(q[:, :, :8], k, lo=[0, 0])
    with pytest.raises(TypeError, match="lo"):
        prompt_attention_weights(q[:, :, :8], k, lo=torch.zeros(1, device="cuda"))
    assert prompt_attention_weights(q[:, :, :0], k[:, :, :0]).shape == (1, 2, 0)


# ---- prompt selection ----------------------------------------------------------------------------
LOAD = [
    # batch, kv heads, head dim, tokens, capacity, keep_first, keep_recent, lo
    (2, 2, 64, 300, 100, 4, 32, [0, 210]),
    (1, 2, 16, 1, 40, 4, 32, None),
    (3, 1, 32, 65, 64, 0, 1, [0, 1, 65]),
    (1, 8, 128, 5000, 1031, 4, 100, None),
    (2, 1, 256, 1025, 36, 4, 32, [0, 989]),
    (1, 1, 64, 70000, 4096, 4, 256, None),
    (1, 2, 64, 0, 40, 4, 32, None),
    (4, 2, 16, 9001, 36, 4, 32, [0, 4500, 8970, 9001]),
    (1, 2, 16, 20001, 12000, 5000, 1, [3]),
    (2, 1, 16, 8193, 8192, 0, 1, [0, 1]),
]


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("kind", ["plain", "ties", "odd"])
@pytest.mark.parametrize("case", LOAD, ids=[str(c[:7]) for c in LOAD])
def test_load_prompt(case, kind, dtype):
    b, hkv, d, t, c, first, recent, lo = case
    g = torch.Generator().manual_seed(41)
    cache, _ = _filled(b, 2 * hkv, hkv, c, d, dtype, [c] * b, 42, keep_first=first, keep_recent=recent)
    k = torch.randn(b, t, hkv, d, generator=g).to(dtype).cuda().transpose(1, 2)
    v = torch.randn(b, hkv, t, d + 8, generator=g).to(dtype).cuda()[..., :d]
    w = torch.rand(b, hkv, t, generator=g)
    if kind == "ties":
        w = (w * 6).floor() - 1  # six values, one of them negative
    elif kind == "odd":
        w = torch.where(w < 0.2, torch.tensor(float("nan")), torch.where(w < 0.4, torch.tensor(float("inf")), w - 0.7))
        w = torch.where(w > 0.2, torch.tensor(-0.0), w)
        w[..., ::7] = 0.0
    before = _state(cache)
    cache.load_prompt(k, v, w.cuda(), lo=lo)
    for i in range(b):
        at0 = lo[i] if lo else 0
        for h in range(hkv):
            kept = torch.from_numpy(O.kept_columns(w[i, h].double().numpy(), at0, c, first, recent))
            m = len(kept)
            before["keys"][i, h, :m], before["values"][i, h, :m] = k[i, h, kept], v[i, h, kept]
            before["weights"][i, h, :m] = w[i, h, kept].cuda()
            before["order"][i, h, :m] = (kept - at0).int().cuda()
            before["lengths"][i, h], before["seen"][i, h] = m, t - at0
    _same(cache, before)


def test_load_prompt_refusals():
    cache = HeavyHitterCache(1, 4, 2, 64, 32, torch.float16, "cuda")
    k = torch.zeros(1, 2, 10, 32, device="cuda").half()
    w = torch.zeros(1, 2, 10, device="cuda")
    for bad, err in ((lambda: cache.load_prompt(k[..., :16], k, w), ValueError),
                     (lambda: cache.load_prompt(k, k[:, :, :9], w), ValueError),
                     (lambda: cache.load_prompt(k.bfloat16(), k.bfloat16(), w), TypeError),
                     (lambda: cache.load_prompt(k, k, w.half()), TypeError),
                     (lambda: cache.load_prompt(k, k, w[..., :9]), ValueError),
                     (lambda: cache.load_prompt(k, k, w.cpu()), ValueError),
                     (lambda: cache.load_prompt(k, k, w, lo=[0, 0]), ValueError),
                     (lambda: cache.load_prompt(cache.keys, cache.values, cache.weights, lo=[3]), ValueError),
                     (lambda: cache.append(torch.zeros(1, 4, 32, device="cuda").half(), cache.keys[:, :, 3], k[:, :, 0]),
                      ValueError),
                     (lambda: cache.append(k[:, 0, :1], k[:, :, 0], k[:, :, 0]), ValueError),
                     (lambda: cache.append(torch.zeros(1, 4, 32, device="cuda"), k[:, :, 0], k[:, :, 0]), TypeError),
                     (lambda: cache.append(torch.zeros(1, 4, 32).half(), k[:, :, 0], k[:, :, 0]), ValueError),
                     (lambda: cache.attend(torch.zeros(1, 2, 32, device="cuda").half()), ValueError),
                     (lambda: cache.attend(torch.zeros(1, 4, 32, device="cuda").half(), scale=0.0), ValueError)):
        with pytest.raises(err):
            bad()


@pytest.mark.parametrize("batch", [1, 2])
def test_index_operands_that_view_the_caches_state(batch):
    """positions and lo may be the cache's own counters: they are taken as they were before the call."""
    g = torch.Generator().manual_seed(51)
    lengths = [5, 40][:batch]
    inv, _ = rotary_frequencies(64, device="cuda")
    q, k, v = (torch.randn(batch, h, 64, generator=g).half().cuda() for h in (64, 32, 32))
    k4, v4 = (torch.randn(batch, 32, 200, 64, generator=g).half().cuda() for _ in range(2))
    w = torch.rand(batch, 32, 200, generator=g).cuda()
    got = []
    for name in ("seen", "lengths", "order"):
        for own in (True, False):
            cache, _ = _filled(batch, 64, 32, 48, 64, torch.float16, lengths, 50, keep_recent=8)
            view = getattr(cache, name).flatten(1)[:, 0]
            out = [cache.append(q, k, v, inv, positions=view if own else view.clone())]
            got.append(out + list(_state(cache).values()))
            cache.load_prompt(k4, v4, w, lo=view if own else view.clone())
            got[-1] += list(_state(cache).values())
    for a, b in zip(got[::2], got[1::2]):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


# ---- a run of them -------------------------------------------------------------------------------
def test_prompt_then_decode():
    """A padded batch's prompt into the cache, then decode steps past its capacity: each operator
    against the oracle on the state before it, and the masses that must add up."""
    b, hq, hkv, d, t, c, steps = 2, 6, 2, 64, 150, 64, 40
    dtype, lo = torch.bfloat16, [0, 100]
    g = torch.Generator().manual_seed(77)
    inv, factor = rotary_frequencies(d, device="cuda")
    cache = HeavyHitterCache(b, hq, hkv, c, d, dtype, "cuda", keep_first=4, keep_recent=16)
    q, k, v = (torch.randn(b, h, t, d, generator=g).to(dtype).cuda() for h in (hq, hkv, hkv))
    pos = (torch.arange(t)[None] - torch.tensor(lo)[:, None]).clamp(min=0).cuda()
    q, k = rotary_embedding(q, k, pos, inv, factor=factor)
    w = prompt_attention_weights(q[:, :, -32:], k, lo=lo)
    cache.load_prompt(k, v, w, lo=lo)
    assert cache.lengths.tolist() == [[64, 64], [50, 50]] and cache.seen.tolist() == [[150, 150], [50, 50]]
    for step in range(steps):
        before = _state(cache)
        q, k, v = ((torch.randn(b, h, d, generator=g) * 2).to(dtype).cuda() for h in (hq, hkv, hkv))
        turned = cache.append(q, k, v, inv, factor=factor)
        want_q, want_k = rotary_embedding(q, k, before["seen"][:, 0], inv, factor=factor)
        assert torch.equal(turned, want_q)
        for i in range(b):
            for h in range(hkv):
                slot = O.append_slot(int(before["lengths"][i, h]), int(before["seen"][i, h]),
                                     _np(before["weights"][i, h]), _np(before["order"][i, h]), c, 4, 16)
                assert torch.equal(cache.keys[i, h, slot], want_k[i, h]) and int(cache.order[i, h, slot]) == 150 + step - lo[i]
        after = _state(cache)
        out = cache.attend(turned)
        for i in range(b):
            n = int(after["lengths"][i, 0])
            for h in range(hkv):
                ref, bound, new, nb = O.attend(_np(turned[i, 3 * h:3 * h + 3]), _np(after["keys"][i, h, :n]),
                                               _np(after["values"][i, h, :n]), _np(after["weights"][i, h, :n]), 1 / 8, 0.0,
                                               STEP[dtype])
                _within(out[i, 3 * h:3 * h + 3], ref, bound, f"step {step}")
                _within(cache.weights[i, h, :n], new, nb, f"step {step} weights")
    # Row 1 filled up after 14 steps; the sinks and the last 16 tokens are still there in both.
    for i in range(b):
        for h in range(hkv):
            held = set(cache.order[i, h].tolist())
            assert len(held) == c and set(range(4)) <= held
            assert set(range(int(cache.seen[i, h]) - 16, int(cache.seen[i, h]))) <= held
    cache.reset()
    assert not cache.lengths.any() and not cache.attend(turned).any()


def test_captured_steps_replay():
    """append and attend captured once and replayed, with eager work between, equal eager steps."""
    b, hq, hkv, d, c = 3, 8, 2, 128, 300
    inv, _ = rotary_frequencies(d, device="cuda")
    caches = [_filled(b, hq, hkv, c, d, torch.float16, [0, 297, 300], 9, keep_first=2, keep_recent=8)[0] for _ in range(2)]
    g = torch.Generator().manual_seed(10)
    q, k, v = (torch.randn(b, h, d, generator=g).half().cuda() for h in (hq, hkv, hkv))
    warm, _ = _filled(b, hq, hkv, c, d, torch.float16, [1, 2, 3], 9, keep_first=2, keep_recent=8)
    warm.attend(warm.append(q, k, v, inv))
    start = _state(caches[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = caches[0].attend(caches[0].append(q, k, v, inv))
    _same(caches[0], start)
    for _ in range(6):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        want = caches[1].attend(caches[1].append(q, k, v, inv))
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        _same(caches[0], _state(caches[1]))


def test_captured_prompt_replays():
    g = torch.Generator().manual_seed(12)
    cache = HeavyHitterCache(2, 4, 2, 64, 64, torch.float16, "cuda")
    other = HeavyHitterCache(2, 4, 2, 64, 64, torch.float16, "cuda")
    q = torch.randn(2, 4, 40, 64, generator=g).half().cuda()
    k, v = (torch.randn(2, 2, 500, 64, generator=g).half().cuda() for _ in range(2))
    lo = torch.tensor([0, 450], dtype=torch.int32, device="cuda")
    other.load_prompt(k, v, prompt_attention_weights(q, k, lo=lo), lo=lo)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w = prompt_attention_weights(q, k, lo=lo)
        cache.load_prompt(k, v, w, lo=lo)
    for n in range(4):
        k.copy_(torch.randn(k.shape, generator=g))
        lo.copy_(torch.tensor([n, 500 - 30 * n], dtype=torch.int32))
        graph.replay()
        other.reset()
        other.load_prompt(k, v, prompt_attention_weights(q, k, lo=lo), lo=lo)
        torch.cuda.synchronize()
        m = other.lengths.clone()
        assert torch.equal(cache.lengths, m) and torch.equal(cache.seen, other.seen)
        for i in range(2):
            n_i = int(m[i, 0])
            for name in ("keys", "values", "weights", "order"):
                assert torch.equal(getattr(cache, name)[i, :, :n_i], getattr(other, name)[i, :, :n_i])


def test_two_caches_on_two_streams():
    """Calls on different caches from two streams at once: nothing is shared between them."""
    inv, _ = rotary_frequencies(64, device="cuda")
    g = torch.Generator().manual_seed(14)
    runs = []
    for seed in (1, 2):
        pair = [_filled(2, 8, 2, 500, 64, torch.bfloat16, [500, 100], seed)[0] for _ in range(2)]
        x = [torch.randn(2, h, 64, generator=g).bfloat16().cuda() for h in (8, 2, 2)]
        runs.append((pair, x, torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for (a, _), x, stream in runs:
            with torch.cuda.stream(stream):
                outs.append(a.attend(a.append(*x, inv)))
    torch.cuda.synchronize()
    want = [c.attend(c.append(*x, inv)) for _ in range(5) for (_, c), x, _ in runs]
    for a, b in zip(outs, want):
        assert torch.equal(a, b)
    for (a, c), _, _ in runs:
        _same(a, _state(c))


# ---- the two call paths ----------------------------------------------------------------------------
class _General:
    """_pgr_ops that hands every call to the general path."""

    def __getattr__(self, name):
        return lambda *args: None


def _forms():
    g = torch.Generator().manual_seed(60)
    b, hq, hkv, d, t = 3, 6, 2, 64, 90
    a = dict(q4=torch.randn(b, hq, t, d, generator=g).half().cuda(), k4=torch.randn(b, hkv, t, d, generator=g).half().cuda(),
             v4=torch.randn(b, hkv, t, d, generator=g).half().cuda(), q=torch.randn(b, hq, d, generator=g).half().cuda(),
             k=torch.randn(b, hkv, d, generator=g).half().cuda(), v=torch.randn(b, hkv, d, generator=g).half().cuda(),
             pos=torch.arange(t).repeat(b, 1).cuda(), one=torch.tensor([3, 900, 41]).cuda(), lo=None, scale=None, softcap=None,
             factor=1.0, interleaved=False)
    yield "plain", a, 9
    yield "masked, softcapped", dict(a, lo=torch.tensor([0, 5, 60], dtype=torch.int32).cuda(), softcap=9.0, scale=0.2), 9
    yield "interleaved, int32 positions", dict(a, interleaved=True, factor=1.5, pos=a["pos"].int(), one=a["one"].int()), 9
    yield "shared positions, none for the step", dict(a, pos=a["pos"][:1], one=None), 9
    yield "transposed", dict(a, **{n: a[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("q4", "k4", "v4")}), 9
    yield "lists and integers", dict(a, lo=[0, 5, 60], scale=1, softcap=30, factor=2), None
    yield "strided head_dim", dict(a, **{n: a[n].transpose(-1, -2).contiguous().transpose(-1, -2) for n in ("q4", "k", "q")}), None
    yield "64-bit lo", dict(a, lo=torch.tensor([0, 5, 60]).cuda()), None
    yield "parameters", dict(a, q=torch.nn.Parameter(a["q"].clone()), k4=torch.nn.Parameter(a["k4"].clone())), None


def test_both_call_paths_agree(monkeypatch):
    from pager_hf import _native as N

    inv, _ = rotary_frequencies(32, device="cuda")

    class Counting:
        def __init__(self):
            self.taken = 0

        def __getattr__(self, name):
            def call(*args):
                got = getattr(ops, name)(*args)
                self.taken += got is not None
                return got
            return call

    ops = N.ops()
    for name, a, taken in _forms():
        print(f"call path: {name}", flush=True)
        got = []
        count = Counting()
        for path in (count, _General()):
            monkeypatch.setattr(N, "_ops", path)
            with torch.no_grad():
                cache = HeavyHitterCache(3, 6, 2, 48, 64, torch.float16, "cuda", keep_recent=8)
                out = list(rotary_embedding(a["q4"], a["k4"], a["pos"], inv, interleaved=a["interleaved"], factor=a["factor"],
                                            inverse=True))
                out += rotary_embedding(a["q"], a["k"], a["one"] if a["one"] is not None else a["pos"][0, :3], inv)
                w = prompt_attention_weights(a["q4"][:, :, -7:], a["k4"], lo=a["lo"], scale=a["scale"], softcap=a["softcap"])
                cache.load_prompt(a["k4"], a["v4"], w, lo=a["lo"])
                turned = cache.append(a["q"], a["k"], a["v"], inv, positions=a["one"], interleaved=a["interleaved"],
                                      factor=a["factor"])
                out += [w, turned, cache.attend(turned, scale=a["scale"], softcap=a["softcap"])]
                same = cache.append(a["q"], a["k"], a["v"])
                assert same is a["q"] or torch.equal(same, a["q"])
                out.append(cache.attend(a["q"]))
                rotary_embedding(a["q"], None, a["pos"][0, :3], inv)
            got.append(out + [getattr(cache, n) for n in STATE])
        for x, y in zip(*got):
            assert x.dtype == y.dtype and torch.equal(x, y), name
        # the calls above: three of rotary_embedding, two appends, two attends, weights, load
        assert taken is None or count.taken == taken, (name, count.taken)


def test_gradients_are_refused():
    from pager_hf import _native as N

    assert N.ops() is not None
    cache = HeavyHitterCache(1, 2, 1, 48, 32, torch.float16, "cuda")
    q, k = torch.zeros(1, 2, 32, device="cuda").half(), torch.zeros(1, 1, 32, device="cuda").half()
    w = torch.zeros(1, 1, 5, device="cuda", requires_grad=True)
    k4 = torch.zeros(1, 1, 5, 32, device="cuda").half()
    inv, _ = rotary_frequencies(32, device="cuda")
    for bad in (lambda: cache.attend(q.clone().requires_grad_()), lambda: cache.append(q, k.clone().requires_grad_(), k),
                lambda: cache.append(q, k, k, inv.clone().requires_grad_()),
                lambda: cache.load_prompt(k4, k4, w), lambda: prompt_attention_weights(k4.clone().requires_grad_(), k4),
                lambda: rotary_embedding(q, None, torch.zeros(1, dtype=torch.int64, device="cuda"), inv.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="gradient"):
            bad()
    assert not cache.seen.any()
    with torch.inference_mode():
        cache.attend(cache.append(q, k, k, inv))
    assert int(cache.seen) == 1


def test_forward_tangents_are_refused():
    from torch.autograd import forward_ad

    cache = HeavyHitterCache(1, 2, 1, 48, 32, torch.float16, "cuda")
    q, k = torch.zeros(1, 2, 32, device="cuda").half(), torch.zeros(1, 1, 32, device="cuda").half()
    w, k4 = torch.zeros(1, 1, 5, device="cuda"), torch.zeros(1, 1, 5, 32, device="cuda").half()
    inv, _ = rotary_frequencies(32, device="cuda")
    pos = torch.zeros(1, dtype=torch.int64, device="cuda")
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for bad in (lambda: cache.attend(dual(q)), lambda: cache.append(dual(q), k, k), lambda: cache.append(q, dual(k), k),
                    lambda: cache.append(q, k, dual(k)), lambda: cache.append(q, k, k, dual(inv)),
                    lambda: cache.load_prompt(dual(k4), k4, w), lambda: cache.load_prompt(k4, dual(k4), w),
                    lambda: cache.load_prompt(k4, k4, dual(w)), lambda: prompt_attention_weights(dual(k4), k4),
                    lambda: prompt_attention_weights(k4, dual(k4)), lambda: rotary_embedding(dual(q), None, pos, inv),
                    lambda: rotary_embedding(q, dual(k), pos, inv), lambda: rotary_embedding(q, None, pos, dual(inv))):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(RuntimeError, match="gradient"):
                    bad()
        assert not cache.seen.any()
        cache.attend(cache.append(q, k, k, inv))
    assert int(cache.seen) == 1
