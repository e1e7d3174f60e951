"""The normed rotary embedding and the cache of pages on the GPU against the 64-bit oracle, and as a run."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import bounded_cache as B
from oracle import drafted_tokens as O
from pager_hf import DraftTree, PageTableCache, draft_tree
from pager_hf.rotary import norm_rotary_embedding, rotary_embedding, rotary_frequencies

pytestmark = pytest.mark.gpu
STEP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
CACHE_TYPES = [torch.float16, torch.bfloat16]
# Half of the smallest subnormal.
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134, torch.float32: 2.0**-150}


def _np(t):
    return t.detach().cpu().double().numpy()


def _within(got, ref, bound, what):
    got = _np(got) if isinstance(got, torch.Tensor) else got
    err = np.abs(got - ref)
    assert np.all(err <= bound), f"{what}: off by {np.nanmax(err)}, {np.nanmax(err / np.maximum(bound, 1e-300)):.3g} x bound"


def _bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---- normed rotary embedding ----------------------------------------------------------------------
NORM = [
    # batch, query heads, kv heads, tokens, head dim, dims that turn
    (1, 14, 2, 1, 64, 64), (2, 4, 2, 37, 128, 128), (1, 3, 1, 5, 256, 128), (3, 2, 1, 9, 80, 80), (1, 4, 4, 33, 96, 32),
    (2, 2, 1, 3, 16, 16), (1, 2, 2, 7, 20, 12), (1, 2, 1, 4, 65, 64), (1, 2, 1, 2, 1024, 1024), (1, 1, 1, 3, 2000, 2000),
    (1, 5, 1, 6, 128, 0), (2, 3, 1, 4, 128, 24), (1, 2, 1, 3, 16, 6), (1, 40, 8, 300, 128, 128), (1, 2, 1, 11, 1, 0),
]


@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", NORM, ids=str)
def test_norm_rotary(case, dtype, interleaved):
    b, hq, hk, t, d, r = case
    g = torch.Generator().manual_seed(3)
    # Views of a projection whose heads are padded, and start at an odd element.
    x = (torch.randn(b, t, hq + hk, d + 3, generator=g) * 3).to(dtype).cuda()[..., 1: d + 1]
    q, k = x[:, :, :hq].transpose(1, 2), x[:, :, hq:].transpose(1, 2)
    wide = t % 2 == 0  # float32 weights, or the operands' type
    w = [(1 + torch.randn(d, generator=g) / 4).to(torch.float32 if wide else dtype).cuda() for _ in range(2)]
    inv, _ = rotary_frequencies(r, device="cuda") if r else (torch.empty(0, device="cuda"), 1.0)
    pos = torch.randint(0, 200000, (b, t), generator=g).cuda()
    got = norm_rotary_embedding(q, k, pos, inv, *w, eps=1e-5, interleaved=interleaved, factor=1.25)
    for y, src, weight in zip(got, (q, k), w):
        assert y.is_contiguous() and y.dtype == dtype
        ref, bound = O.norm_rotate(_np(src), _np(weight), 1e-5, _np(pos)[:, None], _np(inv), interleaved=interleaved,
                                   factor=1.25)
        _within(y, ref, bound + STEP[dtype] * (np.abs(ref) + bound) + TINY[dtype], f"{case}")


def test_norm_rotary_forms():
    g = torch.Generator().manual_seed(4)
    q, k = torch.randn(3, 4, 64, generator=g).half().cuda(), torch.randn(3, 2, 64, generator=g).half().cuda()
    qw, kw = torch.rand(64, generator=g).half().cuda(), torch.rand(64, generator=g).half().cuda()
    inv, _ = rotary_frequencies(64, device="cuda")
    pos = torch.tensor([0, 7, 131071], device="cuda")
    a = norm_rotary_embedding(q, k, pos, inv, qw, kw)
    b = norm_rotary_embedding(q[:, :, None], k[:, :, None], pos[:, None].int(), inv, qw, kw)
    assert a[0].shape == q.shape and torch.equal(a[0], b[0][:, :, 0]) and torch.equal(a[1], b[1][:, :, 0])
    alone = norm_rotary_embedding(q, None, pos, inv, qw, None)
    assert torch.equal(alone[0], a[0]) and alone[1] is None
    # One row of positions for all; unit weights and no eps leave a turned vector of root mean square 1.
    x = torch.randn(2, 4, 5, 64, generator=g).half().cuda()
    shared = norm_rotary_embedding(x, None, torch.arange(5, device="cuda")[None], inv, qw, None)[0]
    each = norm_rotary_embedding(x, None, torch.arange(5, device="cuda").repeat(2, 1), inv, qw, None)[0]
    assert torch.equal(shared, each)
    empty = norm_rotary_embedding(x[:0], None, torch.zeros(0, 5, dtype=torch.int64, device="cuda"), inv, qw, None)[0]
    assert empty.shape == (0, 4, 5, 64)
    # A head of zeros stays zeros; one with an infinite element gives NaN there and zeros elsewhere, as inf * 0.
    z = torch.zeros(1, 1, 1, 64, device="cuda").half()
    assert not norm_rotary_embedding(z, None, torch.zeros(1, 1, dtype=torch.int64, device="cuda"), inv, qw, None)[0].any()


def test_norm_rotary_refusals():
    q = torch.zeros(1, 2, 4, 64, device="cuda").half()
    w, inv, pos = torch.ones(64, device="cuda").half(), torch.ones(32, device="cuda"), torch.zeros(1, 4, dtype=torch.int64,
                                                                                                device="cuda")
    with pytest.raises(ValueError, match="q_weight"):
        norm_rotary_embedding(q, None, pos, inv, w[:32], None)
    with pytest.raises(TypeError, match="q_weight"):
        norm_rotary_embedding(q, None, pos, inv, w.bfloat16(), None)
    with pytest.raises(ValueError, match="devices"):
        norm_rotary_embedding(q, None, pos, inv, w.cpu(), None)
    with pytest.raises(TypeError, match="share"):
        norm_rotary_embedding(q, q, pos, inv, w, w.float())
    with pytest.raises(ValueError, match="turns"):
        norm_rotary_embedding(q, None, pos, torch.ones(33, device="cuda"), w, None)
    with pytest.raises(ValueError, match="positions"):
        norm_rotary_embedding(q, None, pos[:, :3], inv, w, None)
    with pytest.raises(Exception, match="eps"):
        norm_rotary_embedding(q, None, pos, inv, w, None, eps=-1.0)


# ---- trees ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", [1, 2, 31, 33, 63, 64])
def test_draft_tree(t):
    rng = np.random.default_rng(t)
    parents = np.stack([np.arange(t) - 1, np.full(t, -1), rng.integers(-1, np.maximum(np.arange(t), 0)),
                        rng.integers(-9, 99, t), np.arange(t)]).astype(np.int32)
    tree = draft_tree(_int32(parents)[:, : t])
    sees, depth = O.tree(parents)
    bits = (tree.masks.cpu().numpy().astype(np.uint64)[:, :, None] >> np.arange(t, dtype=np.uint64)) & np.uint64(1)
    assert np.array_equal(bits.astype(bool), sees) and np.array_equal(tree.depths.cpu().numpy(), depth)


# ---- a cache filled with random tokens -------------------------------------------------------------
def _parents(rng, b, t):
    return np.maximum(np.arange(t) - rng.integers(1, 4, (b, t)), -1).astype(np.int32)


def _filled(rng, pages, page, hq, hkv, d, dtype, lengths, t, layers=1, spare=2, garbage=True):
    """A cache whose rows' pages are scattered, and its table: `spare` entries more than the longest row needs. NaN
    in what no row holds."""
    width = max(-(-(n + t) // page) for n in lengths)
    order = iter(rng.permutation(pages))
    table = np.full((len(lengths), width + spare), -1, np.int32)
    for i, n in enumerate(lengths):
        for j in range(-(-(n + t) // page)):
            table[i, j] = next(order)
    table[:, width:] = rng.choice([-1, pages, 1 << 30, -(1 << 31)], (len(lengths), spare))
    cache = PageTableCache(layers, pages, page, hq, hkv, d, dtype, "cuda")
    g = torch.Generator(device="cuda").manual_seed(int(rng.integers(1 << 30)))
    for x in (cache.keys, cache.values):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
    if garbage:
        held = np.zeros((pages, page), bool)
        for i, n in enumerate(lengths):
            p, o = O.cells(table[i], page, pages, 0, n + t)
            held[p, o] = True
        for x in (cache.keys, cache.values):
            x.masked_fill_(~torch.tensor(held, device="cuda")[None, :, None, :, None], float("nan"))
    return cache, table


CASES = [
    # batch, query heads, kv heads, head dim, new tokens, page, lengths
    (1, 14, 2, 64, 1, 16, [1000]),
    (4, 4, 2, 16, 5, 16, [0, 11, 12, 130]),
    (5, 12, 2, 128, 13, 32, [0, 15, 16, 19, 333]),
    (3, 16, 1, 32, 64, 64, [63, 640, 999]),
    (2, 8, 1, 256, 7, 128, [203, 70]),
    (2, 8, 1, 256, 33, 16, [203, 0]),
    (3, 16, 16, 64, 2, 16, [129, 3, 31]),
    (2, 28, 4, 128, 9, 256, [4133, 1025]),
    (1, 1, 1, 64, 3, 16, [0]),
    (1, 16, 1, 64, 1, 32, [16387]),
    (33, 16, 8, 64, 4, 16, [i * 70 // 32 for i in range(33)]),
    (2, 4, 2, 128, 200, 64, [70, 0]),
    (1, 32, 8, 64, 129, 16, [500]),
]
IDS = [str(c[:6]) for c in CASES]


def _counts(kind, rng, b, t):
    return None if kind != "ragged" else [t if i == 0 else int(rng.integers(0, t + 3)) - 1 for i in range(b)]


def _clip(counts, b, t):
    return [t] * b if counts is None else [min(max(c, 0), t) for c in counts]


# ---- append --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", CACHE_TYPES)
@pytest.mark.parametrize("kind", ["plain", "ragged", "tree", "positions", "apart"])
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_append(case, kind, dtype):
    b, hq, hkv, d, t, page, lengths = case
    if kind == "tree" and t > 64:
        pytest.skip("a tree has up to 64 tokens")
    rng = np.random.default_rng(7)
    pages = sum(-(-(n + t) // page) for n in lengths) + 3
    cache, table = _filled(rng, pages, page, hq, hkv, d, dtype, lengths, t, layers=2)
    if kind == "apart":  # a page that is not there: its tokens go nowhere
        table[0, lengths[0] // page] = -1
    counts = _counts(kind, rng, b, t)
    norm, turn, interleaved = kind != "ragged", kind != "apart", kind == "positions"
    half = d // 2 if kind != "positions" else d // 4
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(b, t, hq + 2 * hkv, d + 1, generator=g) * 2).to(dtype).cuda()[..., 1:].transpose(1, 2)
    q, k, v = x[:, :hq], x[:, hq: hq + hkv], x[:, hq + hkv:]
    w = [(1 + torch.randn(d, generator=g) / 4).to(dtype if kind == "tree" else torch.float32).cuda() for _ in range(2)]
    inv, _ = rotary_frequencies(2 * half, device="cuda")
    parents = _parents(rng, b, t)
    sees, depth = O.tree(parents)
    pos = np.asarray(lengths)[:, None] + (depth if kind == "tree" else np.arange(t))
    given = torch.randint(0, 1 << 20, (b, t + 1), generator=g).int().cuda()[:, 1:]
    if kind == "positions":
        pos = _np(given)
    before = [cache.keys.clone(), cache.values.clone()]
    out = cache.append(1, q, k, v, _int32(table), _int32(lengths), inv if turn else None,
                       counts=None if counts is None else _int32(counts),
                       tree=draft_tree(_int32(parents)) if kind == "tree" else None,
                       positions=given if kind == "positions" else None, q_weight=w[0] if norm else None,
                       k_weight=w[1] if norm else None, eps=1e-5, interleaved=interleaved, factor=0.75 if turn else 1.0)
    assert out.shape == q.shape and out.is_contiguous()
    empty = np.zeros(0)
    ref = [O.norm_rotate(_np(y), _np(z) if norm else None, 1e-5, pos[:, None], _np(inv) if turn else empty,
                         interleaved=interleaved, factor=0.75) for y, z in zip((q, k), w)]
    off = [bound + STEP[dtype] * (np.abs(r) + bound) + TINY[dtype] for r, bound in ref]
    want = [_np(y[1]) for y in before]
    slack = np.zeros(want[0].shape)
    for i, n in enumerate(_clip(counts, b, t)):
        _within(out[i, :, :n], ref[0][0][i, :, :n], off[0][i, :, :n], f"q of row {i}")
        assert not out[i, :, n:].any()
        p, o = O.cells(table[i], page, pages, lengths[i], n)
        here = p >= 0
        want[0][p[here], :, o[here]] = ref[1][0][i, :, :n][:, here].transpose(1, 0, 2)
        slack[p[here], :, o[here]] = off[1][i, :, :n][:, here].transpose(1, 0, 2)
        want[1][p[here], :, o[here]] = _np(v)[i, :, :n][:, here].transpose(1, 0, 2)
    nan = np.isnan(want[0])
    got = _np(cache.keys[1])
    assert np.array_equal(np.isnan(got), nan)
    _within(got[~nan], want[0][~nan], slack[~nan], "keys")
    np.testing.assert_array_equal(_np(cache.values[1]), want[1])
    for x, y in zip((cache.keys, cache.values), before):
        assert torch.equal(_bits(x[0]), _bits(y[0]))


def test_append_agrees_with_the_operators_apart():
    """The bits of norm_rotary_embedding, and without a norm of rotary_embedding."""
    rng = np.random.default_rng(9)
    g = torch.Generator().manual_seed(9)
    for d in (64, 128, 256):
        cache, table = _filled(rng, 9, 16, 4, 2, d, torch.bfloat16, [5], 21)
        q, k = torch.randn(1, 4, 21, d, generator=g).bfloat16().cuda(), torch.randn(1, 2, 21, d, generator=g).bfloat16().cuda()
        w = [torch.rand(d, generator=g).bfloat16().cuda() for _ in range(2)]
        inv, _ = rotary_frequencies(d, device="cuda")
        pos = torch.arange(5, 26, device="cuda")[None]
        p, o = (torch.tensor(x, device="cuda") for x in O.cells(table[0], 16, 9, 5, 21))
        for weights in (w, (None, None)):
            out = cache.append(0, q, k, k, _int32(table), _int32([5]), inv, q_weight=weights[0], k_weight=weights[1])
            a = norm_rotary_embedding(q, k, pos, inv, *w) if weights[0] is not None else rotary_embedding(q, k, pos, inv)
            assert torch.equal(out, a[0]) and torch.equal(cache.keys[0][p, :, o], a[1][0].transpose(0, 1))
            assert torch.equal(cache.values[0][p, :, o], k[0].transpose(0, 1))


# ---- attend --------------------------------------------------------------------------------------
def _attend_bounds(dtype, two=True):
    """P enters the product with V as two numbers, off by 3 u^2 of it, u half a step, or rounded to one, off by u; in fp16
    under a largest value of at least 2^14, so that half of the smallest subnormal is 2^-39 of it."""
    u = STEP[dtype]
    return dict(step=u, p_step=3 * u * u if two else u, p_floor=2.0**-39 if dtype == torch.float16 else 0.0)


def _check_attend(cache, layer, table, lengths, q, out, counts, sees, depth, window, scale, softcap, only=None, exact=False):
    b, hq, t, d = q.shape
    # (As documented: one number where there are more than 32 rows a KV head.)
    two = exact or t * (hq // cache.num_kv_heads) <= 32
    hkv, page, pages = cache.num_kv_heads, cache.page_tokens, cache.num_pages
    rep, kn, vn, qn = hq // hkv, _np(cache.keys[layer]), _np(cache.values[layer]), _np(q)
    for i, n in enumerate(_clip(counts, b, t)):
        room = table.shape[1] * page
        length = min(max(lengths[i], 0), room)
        n = min(n, room - length)
        p, o = O.cells(table[i], page, pages, 0, length + n)
        for h in range(hkv):
            heads = slice(h * rep, (h + 1) * rep)
            ref, bound = O.attend_row(qn[i, heads], kn[p, h, o], vn[p, h, o], p >= 0, length, n, sees[i], depth[i], window,
                                      scale, softcap, **_attend_bounds(q.dtype, two))
            rows = slice(0, n) if only is None else [x for x in only if x < n]
            _within(out[i, heads][:, rows], ref[:, rows], bound[:, rows], f"row {i} head {h}")
        assert not out[i, :, n:].any()


def _order(b, t):
    return np.broadcast_to(np.tril(np.ones((t, t), bool)), (b, t, t)), np.broadcast_to(np.arange(t), (b, t))


@pytest.mark.parametrize("dtype", CACHE_TYPES)
@pytest.mark.parametrize("kind", ["plain", "ragged", "tree", "softcap", "window", "tree window", "apart"])
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_attend(case, kind, dtype):
    b, hq, hkv, d, t, page, lengths = case
    if "tree" in kind and t > 64:
        pytest.skip("a tree has up to 64 tokens")
    rng = np.random.default_rng(17)
    pages = sum(-(-(n + t) // page) for n in lengths) + 3
    cache, table = _filled(rng, pages, page, hq, hkv, d, dtype, lengths, t, layers=2)
    if kind == "apart":  # pages that are not there, the last one's among them
        for i, n in enumerate(lengths):
            table[i, rng.integers(0, -(-(n + t) // page))] = [-1, pages, -7][i % 3]
        table[0, (lengths[0] + t - 1) // page] = -1
    counts = _counts(kind, rng, b, t)
    window = [1, 2, 17, 100][b % 4] if "window" in kind else 0
    softcap = 5.0 if kind == "softcap" else 0.0
    g = torch.Generator().manual_seed(5)
    # Queries as views into a larger tensor.
    q = (torch.randn(b, t, hq + 2, d + 1, generator=g) * 2).to(dtype).cuda()[:, :, 1:-1, 1:].transpose(1, 2)
    sees, depth = _order(b, t)
    tree = None
    if "tree" in kind:
        parents = _parents(rng, b, t)
        sees, depth = O.tree(parents)
        tree = draft_tree(_int32(parents))
    before = [cache.keys.clone(), cache.values.clone()]
    scale = 0.3 if kind == "window" else None
    exact = kind in ("ragged", "tree")
    out = cache.attend(1, q, _int32(table), _int32(lengths), counts=None if counts is None else _int32(counts), tree=tree,
                       window=window, softcap=softcap, scale=scale, exact_weights=exact)
    assert out.shape == q.shape and out.transpose(1, 2).is_contiguous()
    for x, y in zip((cache.keys, cache.values), before):
        assert torch.equal(_bits(x), _bits(y))
    _check_attend(cache, 1, table, lengths, q, out, counts, sees, depth, window, scale or 1.0 / d**0.5, softcap, exact=exact)


@pytest.mark.parametrize("dtype", CACHE_TYPES)
@pytest.mark.parametrize("t", [1, 8, 64, 300])
def test_attend_long_rows(t, dtype):
    """Many splits, or many blocks of rows; some of the queries are checked."""
    rng = np.random.default_rng(23)
    lengths = [9000, 4097, 0]
    pages = sum(-(-(n + t) // 64) for n in lengths) + 1
    cache, table = _filled(rng, pages, 64, 16, 2, 128, dtype, lengths, t, spare=40)
    g = torch.Generator().manual_seed(t)
    q = (torch.randn(3, 16, t, 128, generator=g) * 2).to(dtype).cuda()
    sees, depth = _order(3, t)
    for window in (0, 5000):
        out = cache.attend(0, q, _int32(table), _int32(lengths), window=window)
        _check_attend(cache, 0, table, lengths, q, out, None, sees, depth, window, 1.0 / 128**0.5, 0.0,
                      only=sorted({0, t // 3, t - 1}))


RAGGED = [
    # query heads, kv heads, head dim, new tokens, window, lengths
    (4, 1, 64, 3, 0, [0] * 30 + [3000] + [40] * 38 + [2000]),  # more rows than a wave has lanes, few of them long
    (4, 2, 128, 1, 0, [7, 0, 5000, 31]),
    (4, 1, 64, 20, 0, [1] * 129),
    (4, 1, 32, 30, 700, [2500, 10, 0, 4000, 699, 700, 701]),
    (8, 1, 128, 40, 0, [6000, 0, 100]),
    (4, 1, 256, 12, 0, [1500, 3, 1500, 800]),
    (4, 4, 16, 5, 33, [2000, 1, 31, 32, 33]),
    (16, 1, 64, 64, 0, [900, 0, 0, 0, 0, 0, 0, 64]),
    # Rows enough to fill the card, of which one is cut and the others are finished by their workgroups.
    (4, 4, 64, 2, 0, [4500] + [20] * 30 + [0] * 5 + [130] * 34),
    (16, 1, 64, 20, 0, [50] * 69 + [4200]),
    (4, 4, 128, 3, 900, [4100, 899, 900, 901] * 17),
]


@pytest.mark.parametrize("dtype", CACHE_TYPES)
@pytest.mark.parametrize("case", RAGGED, ids=[str(c[:5]) for c in RAGGED])
def test_attend_ragged_batches(case, dtype):
    """Rows of very different lengths, cut into parts of one size; some of them have no new tokens."""
    hq, hkv, d, t, window, lengths = case
    b = len(lengths)
    rng = np.random.default_rng(83)
    pages = sum(-(-(n + t) // 32) for n in lengths) + 1
    cache, table = _filled(rng, pages, 32, hq, hkv, d, dtype, lengths, t)
    g = torch.Generator().manual_seed(b)
    q = (torch.randn(b, hq, t, d, generator=g) * 2).to(dtype).cuda()
    counts = [0 if i % 5 == 4 else t - i % 3 % t for i in range(b)]
    for sees, depth, tree in ((*_order(b, t), None), (*O.tree(_parents(rng, b, t)), True)):
        if tree is not None:
            masks = (sees * (np.uint64(1) << np.arange(t, dtype=np.uint64))).sum(axis=-1, dtype=np.uint64)
            tree = DraftTree(torch.tensor(masks.view(np.int64), device="cuda"), _int32(depth))
        out = cache.attend(0, q, _int32(table), _int32(lengths), counts=_int32(counts), tree=tree, window=window)
        _check_attend(cache, 0, table, lengths, q, out, counts, sees, depth, window, 1.0 / d**0.5, 0.0,
                      only=sorted({0, t // 2, t - 1}))
    none = cache.attend(0, q, _int32(table), _int32(lengths), counts=_int32([0] * b), window=window)
    assert not none.any()


@pytest.mark.parametrize("dtype", CACHE_TYPES)
@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("t", [1, 5, 40])
def test_attend_keeps_more_of_p_than_the_cache_type(t, d, dtype):
    """Few tokens of like weights, whose sums all but cancel in some dims: rounding P to the cache's type is off by
    several times the bound."""
    rng = np.random.default_rng(29)
    cache, table = _filled(rng, 8, 16, 8, 2, d, dtype, [24], t)
    cells = O.cells(table[0], 16, 8, 0, 24 + t)
    p, o = (torch.tensor(x, device="cuda") for x in cells)
    values = torch.randn(24 + t, 2, d, generator=torch.Generator().manual_seed(3)).to(dtype)
    values[1::2] = -values[: 24 + t - 1: 2][: values[1::2].shape[0]]
    cache.values[0][p, :, o] = values.cuda()
    q = (torch.randn(1, 8, t, d, generator=torch.Generator().manual_seed(4)) / 8).to(dtype).cuda()
    out = cache.attend(0, q, _int32(table), _int32([24]), exact_weights=True)
    sees, depth = _order(1, t)
    _check_attend(cache, 0, table, [24], q, out, None, sees, depth, 0, 1.0 / d**0.5, 0.0, exact=True)


@pytest.mark.parametrize("t", [1, 5, 40])
def test_attend_with_scores_of_infinity_and_nan(t):
    """A key that makes every score -inf gives zeros alone and no weight beside others; NaN in a query stays with its
    head and token; keys that a token does not see do not reach it."""
    rng = np.random.default_rng(31)
    cache, table = _filled(rng, 8, 16, 4, 2, 64, torch.float16, [20], t)
    tab, ln = _int32(table), _int32([20])
    q = torch.rand(1, 4, t, 64, generator=torch.Generator().manual_seed(6)).half().cuda() + 0.1
    plain = cache.attend(0, q, tab, ln)
    p, o = O.cells(table[0], 16, 8, 0, 20 + t)
    keys = cache.keys.clone()
    cache.keys[0, int(p[3]), :, int(o[3])] = float("-inf")
    some = cache.attend(0, q, tab, ln)
    assert torch.isfinite(some).all()
    at = np.ones(20 + t, bool)
    at[3] = False
    sees, _ = _order(1, t)
    kn, vn, qn = _np(keys[0]), _np(cache.values[0]), _np(q)
    for h in range(2):
        ref, bound = O.attend_row(qn[0, 2 * h: 2 * h + 2], kn[p, h, o], vn[p, h, o], at, 20, t, sees[0], np.arange(t), 0, 0.125,
                                  0.0, **_attend_bounds(torch.float16, t < 17))
        _within(some[0, 2 * h: 2 * h + 2], ref, bound, "without the token")
    cache.keys.fill_(float("-inf"))
    assert not cache.attend(0, q, tab, ln).any()
    cache.keys.copy_(keys)
    bad = q.clone()
    bad[0, 1, t - 1, 5] = float("nan")
    out = cache.attend(0, bad, tab, ln)
    assert torch.isnan(out[0, 1, t - 1]).all()
    out[0, 1, t - 1] = plain[0, 1, t - 1]
    assert torch.equal(out, plain)
    if t > 1:  # the last new token's key is seen by itself alone
        cache.keys[0, int(p[-1]), :, int(o[-1])] = float("nan")
        out = cache.attend(0, q, tab, ln)
        assert torch.isnan(out[0, :, t - 1]).all()
        assert torch.equal(out[0, :, : t - 1], plain[0, :, : t - 1])


@pytest.mark.parametrize("t", [1, 5, 40])
def test_a_far_softcap_changes_nothing(t):
    """c tanh(s / c) differs from s by s^3 / (3 c^2): 2e-7 at c = 1e5 and scores up to 20, less than half a step (2^-24) of
    the 16 that the scores' terms add up to in magnitude. So the output is within its bound without a cap."""
    rng = np.random.default_rng(73)
    cache, table = _filled(rng, 12, 16, 8, 2, 64, torch.float16, [100], t)
    q = (torch.randn(1, 8, t, 64, generator=torch.Generator().manual_seed(4)) * 2).half().cuda()
    out = cache.attend(0, q, _int32(table), _int32([100]), softcap=1e5, exact_weights=True)
    _check_attend(cache, 0, table, [100], q, out, None, *_order(1, t), 0, 1.0 / 64**0.5, 0.0, exact=True)


@pytest.mark.parametrize("cap", [0.5, 3.0, 50.0])
@pytest.mark.parametrize("t", [1, 5, 40])
def test_softcaps(t, cap):
    rng = np.random.default_rng(79)
    cache, table = _filled(rng, 12, 16, 8, 2, 64, torch.float16, [100], t)
    q = (torch.randn(1, 8, t, 64, generator=torch.Generator().manual_seed(4)) * 4).half().cuda()
    out = cache.attend(0, q, _int32(table), _int32([100]), softcap=cap, exact_weights=True)
    _check_attend(cache, 0, table, [100], q, out, None, *_order(1, t), 0, 1.0 / 64**0.5, cap, exact=True)


def test_one_token_at_given_positions():
    rng = np.random.default_rng(89)
    cache, table = _filled(rng, 9, 16, 4, 2, 64, torch.float16, [3, 40], 1, garbage=False)
    g = torch.Generator().manual_seed(4)
    q, k = torch.randn(2, 4, 64, generator=g).half().cuda(), torch.randn(2, 2, 64, generator=g).half().cuda()
    inv, _ = rotary_frequencies(64, device="cuda")
    pos = torch.tensor([7, 90000], device="cuda")
    want = rotary_embedding(q, k, pos, inv)
    for given in (pos, pos.int(), torch.stack([pos, pos], dim=1)[:, 0]):
        assert torch.equal(cache.append(0, q, k, k, _int32(table), _int32([3, 40]), inv, positions=given), want[0])
        for i, n in enumerate([3, 40]):
            p, o = O.cells(table[i], 16, 9, n, 1)
            assert torch.equal(cache.keys[0, int(p[0]), :, int(o[0])], want[1][i])


def test_masks_that_leave_a_token_nothing():
    rng = np.random.default_rng(37)
    cache, table = _filled(rng, 8, 16, 4, 2, 64, torch.bfloat16, [0, 18], 6)
    q = torch.randn(2, 4, 6, 64, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    sees = rng.random((2, 6, 6)) < 0.5
    sees[:, 2] = False
    masks = torch.tensor((sees * (1 << np.arange(6))).sum(-1), device="cuda")
    masks |= ~63  # bits of tokens that are not there
    depth = rng.integers(0, 6, (2, 6))
    for window in (0, 3):
        out = cache.attend(0, q, _int32(table), _int32([0, 18]), tree=DraftTree(masks, _int32(depth)), window=window)
        assert not out[0, :, 2].any() and (window == 3 or out[1, :, 2].any())
        _check_attend(cache, 0, table, [0, 18], q, out, None, sees, depth, window, 0.125, 0.0)


def test_no_room_behind_the_table():
    """Tokens behind the table's end are not stored and give zeros; lengths beyond it (or below 0) are cut off."""
    rng = np.random.default_rng(41)
    cache, table = _filled(rng, 9, 16, 4, 2, 64, torch.float16, [30, 32, 8], 2, spare=0)
    lengths = [30, 45, -5]
    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn(3, h, 5, 64, generator=g).half().cuda() for h in (4, 2, 2))
    before = cache.keys.clone()
    cache.append(0, q, k, v, _int32(table), _int32(lengths))
    p, o = O.cells(table[0], 16, 9, 30, 5)
    put = [i for i in range(5) if p[i] >= 0]
    for i in put:
        assert torch.equal(cache.keys[0, int(p[i]), :, int(o[i])], k[0, :, i])
        before[0, int(p[i]), :, int(o[i])] = k[0, :, i]
    p, o = O.cells(table[2], 16, 9, 0, 5)
    for i in range(5):
        before[0, int(p[i]), :, int(o[i])] = k[2, :, i]
    assert table.shape[1] == 3  # (row 1: tokens 45, 46 and 47)
    before[0, table[1, 2], :, 13:] = k[1, :, :3]
    assert torch.equal(_bits(cache.keys), _bits(before))
    cache.values.nan_to_num_(0.0)
    cache.keys.nan_to_num_(0.0)
    out = cache.attend(0, q, _int32(table), _int32(lengths))
    sees, depth = _order(3, 5)
    _check_attend(cache, 0, table, lengths, q, out, None, sees, depth, 0, 0.125, 0.0)
    # A table of no entries: nothing is held, nothing is stored.
    none = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    assert torch.equal(cache.append(0, q, k, v, none, _int32(lengths)), q)
    assert torch.equal(_bits(cache.keys), _bits(torch.nan_to_num(before, 0.0)))
    assert not cache.attend(0, q, none, _int32(lengths)).any()
    cache.keep(none, _int32(lengths), _int32([[2, 3]] * 3))


def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements: its last pages."""
    page, hkv, d = 256, 8, 128
    pages = (1 << 32) // (page * hkv * d) + 5
    cache = PageTableCache(1, pages, page, 8, hkv, d, torch.bfloat16, "cuda")
    table = np.array([[pages - 1, 0, pages - 3]], np.int32)
    g = torch.Generator().manual_seed(2)
    kv = torch.randn(2, 1, hkv, 600, d, generator=g).bfloat16().cuda()
    q = torch.randn(1, 8, 600, d, generator=g).bfloat16().cuda()
    cache.append(0, q, kv[0], kv[1], _int32(table), _int32([0]))
    small = PageTableCache(1, 3, page, 8, hkv, d, torch.bfloat16, "cuda")
    small.append(0, q, kv[0], kv[1], _int32([[2, 0, 1]]), _int32([0]))
    for a, b in ((pages - 1, 2), (0, 0)):
        assert torch.equal(cache.keys[0, a], small.keys[0, b]) and torch.equal(cache.values[0, a], small.values[0, b])
    for tokens in (q[:, :, -1:], q[:, :, -60:]):
        n = tokens.shape[2]
        a = cache.attend(0, tokens, _int32(table), _int32([600 - n]))
        assert torch.equal(a, small.attend(0, tokens, _int32([[2, 0, 1]]), _int32([600 - n])))
    path = _int32([[5, 9, 40]])
    cache.keep(_int32(table), _int32([512]), path)
    small.keep(_int32([[2, 0, 1]]), _int32([512]), path)
    assert torch.equal(cache.keys[0, pages - 3], small.keys[0, 1]) and cache.keys[0, 0].any()


# ---- keep ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", CACHE_TYPES)
@pytest.mark.parametrize("d,page", [(16, 16), (64, 32), (128, 16), (256, 256)])
def test_keep(d, page, dtype):
    rng = np.random.default_rng(43)
    lengths, t, layers = [0, 5, 16, 300, 31], 64, 3
    pages = sum(-(-(n + t) // page) for n in lengths) + 2
    cache, table = _filled(rng, pages, page, 4, 2, d, dtype, lengths, t, layers=layers)
    table[3, (300 + 40) // page] = -1
    path = np.full((5, 64), -1, np.int32)
    path[0, :7] = [0, 2, 3, 9, 30, 62, 63]
    path[1] = np.arange(64)  # in place already
    path[2] = rng.permutation(64)  # each from where it was before
    path[3, :20] = np.sort(rng.choice(64, 20, replace=False))  # some in a page that is not there
    path[4, :6] = [5, 5, -3, 64, 1 << 30, 1]  # a token twice, entries that move nothing
    want = [cache.keys.clone(), cache.values.clone()]
    old = [x.clone() for x in want]
    for i in range(5):
        for j in range(64):
            if not 0 <= path[i, j] < 64:
                continue
            sp, so = O.cells(table[i], page, pages, lengths[i] + path[i, j], 1)
            tp, to = O.cells(table[i], page, pages, lengths[i] + j, 1)
            if sp[0] >= 0 and tp[0] >= 0:
                for x, y in zip(want, old):
                    x[:, int(tp[0]), :, int(to[0])] = y[:, int(sp[0]), :, int(so[0])]
    wide = torch.full((5, table.shape[1] + 3), 7, dtype=torch.int32, device="cuda")  # a strided table
    wide[:, 1: 1 + table.shape[1]] = _int32(table)
    cache.keep(wide[:, 1: 1 + table.shape[1]], _int32(lengths), _int32(path))
    for x, y in zip((cache.keys, cache.values), want):
        assert torch.equal(_bits(x), _bits(y))


# ---- as a run ------------------------------------------------------------------------------------
def test_draft_verify_and_keep():
    """Two layers, ragged rows: a prompt, then steps of drafted trees of which a path is kept. At the end the cache holds
    what it would hold had each row's accepted tokens come in order, and attends alike."""
    hq, hkv, d, page, layers, dtype = 8, 2, 64, 16, 2, torch.float16
    rng = np.random.default_rng(47)
    prompts = [21, 1, 40]
    b, width = len(prompts), 12
    pages = b * width
    table = _int32(rng.permutation(pages).reshape(b, width))
    cache = PageTableCache(layers, pages, page, hq, hkv, d, dtype, "cuda")
    inv, _ = rotary_frequencies(d, device="cuda")
    w = [torch.rand(d, device="cuda").half() + 0.5 for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(1)

    def tokens(t):
        return [torch.randn(layers, b, h, t, d, generator=g, device="cuda").half() for h in (hq, hkv, hkv)]

    lengths = torch.zeros(b, dtype=torch.int32, device="cuda")
    q, k, v = tokens(max(prompts))
    counts = _int32(prompts)
    accepted = [[(k[:, i, :, j], v[:, i, :, j]) for j in range(n)] for i, n in enumerate(prompts)]
    for layer in range(layers):
        turned = cache.append(layer, q[layer], k[layer], v[layer], table, lengths, inv, counts=counts, q_weight=w[0],
                              k_weight=w[1])
        cache.attend(layer, turned, table, lengths, counts=counts)
    lengths += counts
    for step in range(4):
        t = [5, 1, 16, 9][step]
        parents = _parents(rng, b, t)
        sees, _ = O.tree(parents)
        tree = draft_tree(_int32(parents))
        q, k, v = tokens(t)
        for layer in range(layers):
            turned = cache.append(layer, q[layer], k[layer], v[layer], table, lengths, inv, tree=tree, q_weight=w[0],
                                  k_weight=w[1])
            cache.attend(layer, turned, table, lengths, tree=tree)
        path = np.full((b, t), -1, np.int32)
        for i in range(b):
            taken = np.flatnonzero(sees[i, rng.integers(t)])
            path[i, : len(taken)] = taken
            accepted[i] += [(k[:, i, :, j], v[:, i, :, j]) for j in taken]
        cache.keep(table, lengths, _int32(path))
        lengths += _int32((path >= 0).sum(axis=1))
    assert lengths.tolist() == [len(x) for x in accepted]

    plain = PageTableCache(layers, pages, page, hq, hkv, d, dtype, "cuda")
    zero = torch.zeros(b, dtype=torch.int32, device="cuda")
    most = max(len(x) for x in accepted)
    k, v = (torch.zeros(layers, b, hkv, most, d, device="cuda").half() for _ in range(2))
    for i, x in enumerate(accepted):
        for j, (kj, vj) in enumerate(x):
            k[:, i, :, j], v[:, i, :, j] = kj, vj
    q = torch.zeros(b, hq, most, d, device="cuda").half()
    for layer in range(layers):
        plain.append(layer, q, k[layer], v[layer], table, zero, inv, counts=lengths, q_weight=w[0], k_weight=w[1])
    q, k, v = (x[0, :, :, 0] for x in tokens(1))
    for layer in range(layers):
        for i in range(b):
            p, o = (torch.tensor(x, device="cuda") for x in O.cells(table[i].tolist(), page, pages, 0, len(accepted[i])))
            assert torch.equal(cache.keys[layer, p, :, o], plain.keys[layer, p, :, o])
            assert torch.equal(cache.values[layer, p, :, o], plain.values[layer, p, :, o])
        out = []
        for c in (cache, plain):  # one token a row
            turned = c.append(layer, q, k, v, table, lengths, inv)
            out.append(c.attend(layer, turned, table, lengths))
        assert out[0].shape == q.shape and torch.equal(*out)


def test_a_chunked_prompt_is_the_whole_one():
    """A prompt in one call and in chunks holds the same, and its last token's attention is that of one token alone."""
    rng = np.random.default_rng(53)
    hq, hkv, d, n = 8, 4, 128, 301
    caches = [PageTableCache(1, 12, 32, hq, hkv, d, torch.bfloat16, "cuda") for _ in range(2)]
    table = _int32(rng.permutation(12)[None])
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(1, h, n, d, generator=g).bfloat16().cuda() for h in (hq, hkv, hkv))
    inv, _ = rotary_frequencies(d, device="cuda")
    whole = caches[0].attend(0, caches[0].append(0, q, k, v, table, _int32([0]), inv), table, _int32([0]))
    parts, at = [], 0
    for t in (1, 64, 100, 135, 1):
        now = _int32([at])
        s = slice(at, at + t)
        parts.append(caches[1].attend(0, caches[1].append(0, q[:, :, s], k[:, :, s], v[:, :, s], table, now, inv), table, now))
        at += t
    assert torch.equal(caches[0].keys, caches[1].keys)
    # (The order of the sums differs: each is within its bound of the same value.)
    _check_attend(caches[0], 0, table.cpu().numpy(), [0], rotary_embedding(q, None, torch.arange(n, device="cuda")[None], inv)[0],
                  torch.cat(parts, dim=2), None, *_order(1, n), 0, 1.0 / d**0.5, 0.0, only=[0, 1, 64, 65, 164, 165, 299, 300])
    _check_attend(caches[0], 0, table.cpu().numpy(), [0], rotary_embedding(q, None, torch.arange(n, device="cuda")[None], inv)[0],
                  whole, None, *_order(1, n), 0, 1.0 / d**0.5, 0.0, only=[0, 1, 64, 65, 164, 165, 299, 300])


def test_captured_steps_replay():
    """A step in a graph, replayed on new tokens and lengths, against the eager calls."""
    rng = np.random.default_rng(59)
    caches = [_filled(np.random.default_rng(59), 60, 16, 8, 2, 64, torch.float16, [100, 3], 20, spare=10)[0] for _ in range(2)]
    table = _int32(rng.permutation(60)[:58].reshape(2, 29))
    for c in caches:
        c.keys.nan_to_num_(0.5)
        c.values.nan_to_num_(0.5)
    inv, _ = rotary_frequencies(64, device="cuda")
    w = torch.ones(64, device="cuda").half()
    q, k, v = (torch.zeros(2, h, 7, 64, device="cuda").half() for h in (8, 2, 2))
    lengths, parents, path = _int32([100, 3]), _int32([[-1] * 7] * 2), _int32([[-1] * 7] * 2)

    def step(c):
        tree = draft_tree(parents)
        out = c.attend(0, c.append(0, q, k, v, table, lengths, inv, tree=tree, q_weight=w, k_weight=w), table, lengths, tree=tree)
        c.keep(table, lengths, path)
        n = norm_rotary_embedding(q, k, lengths[:, None].expand(2, 7), inv, w, w)
        return out, n[0], n[1]

    for c in caches:
        step(c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(caches[0])
    for i in range(4):
        g = torch.Generator(device="cuda").manual_seed(i)
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        lengths.copy_(_int32([100 + 9 * i, 200 - 50 * i]))
        parents.copy_(_int32(_parents(rng, 2, 7)))
        path.copy_(_int32([[0, 3, 4, 6, -1, -1, -1], [2, 5, -1, -1, -1, -1, -1]]))
        want = step(caches[1])
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(held, want):
            assert torch.equal(x, y)
        assert torch.equal(caches[0].keys, caches[1].keys) and torch.equal(caches[0].values, caches[1].values)
        torch.randn(1000, device="cuda").sort()  # eager work between the replays


def test_the_same_every_time_and_on_two_streams():
    rng = np.random.default_rng(61)
    made = [_filled(np.random.default_rng(61 + i), 300, 32, 16, 2, 128, torch.bfloat16, [4000, 2100, 77], 40) for i in range(2)]
    q = torch.randn(3, 16, 40, 128, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    lengths, tree = _int32([4000, 2100, 77]), draft_tree(_int32(_parents(rng, 3, 40)))
    tables = [_int32(t) for _, t in made]
    want = [c.attend(0, q, t, lengths, tree=tree) for (c, _), t in zip(made, tables)]
    streams = [torch.cuda.current_stream(), torch.cuda.Stream()]
    streams[1].wait_stream(streams[0])
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(made[i][0].attend(0, q, tables[i], lengths, tree=tree))
    torch.cuda.synchronize()
    for a, xs in zip(want, got):
        for x in xs:
            assert torch.equal(a, x)


def test_refusals():
    cache = PageTableCache(2, 4, 16, 4, 2, 64, torch.float16, "cuda")
    q, k = torch.zeros(1, 4, 3, 64, device="cuda").half(), torch.zeros(1, 2, 3, 64, device="cuda").half()
    table, ln, inv = _int32([[0, 1]]), _int32([0]), torch.ones(32, device="cuda")
    w = torch.ones(64, device="cuda").half()
    with pytest.raises(IndexError):
        cache.append(2, q, k, k, table, ln)
    with pytest.raises(IndexError):
        cache.attend(-1, q, table, ln)
    for bad in (q[:, :3], q[..., :32], q[0, 0]):
        with pytest.raises(ValueError, match="q must"):
            cache.attend(0, bad, table, ln)
    with pytest.raises(ValueError, match="match"):
        cache.append(0, q, k[:, :, :2], k, table, ln)
    with pytest.raises(ValueError, match="match"):
        cache.append(0, q, k, k[:, :, 0], table, ln)
    with pytest.raises(TypeError, match="k must"):
        cache.append(0, q, k.bfloat16(), k, table, ln)
    with pytest.raises(ValueError, match="devices"):
        cache.append(0, q, k.cpu(), k, table, ln)
    with pytest.raises(TypeError, match="table"):
        cache.attend(0, q, table.long(), ln)
    with pytest.raises(ValueError, match="table"):
        cache.attend(0, q, table[0], ln)
    with pytest.raises(TypeError, match="lengths"):
        cache.attend(0, q, table, ln.long())
    with pytest.raises(ValueError, match="counts"):
        cache.attend(0, q, table, ln, counts=_int32([1, 2]))
    with pytest.raises(ValueError, match="masks"):
        cache.attend(0, q, table, ln, tree=draft_tree(_int32([[-1, 0]])))
    with pytest.raises(NotImplementedError, match="64"):
        cache.attend(0, torch.zeros(1, 4, 65, 64, device="cuda").half(), table, ln, tree=draft_tree(_int32([[-1]])))
    with pytest.raises(Exception, match="64"):
        draft_tree(torch.zeros(1, 65, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="window"):
        cache.attend(0, q, table, ln, window=-1)
    with pytest.raises(Exception, match="scale"):
        cache.attend(0, q, table, ln, scale=0.0)
    with pytest.raises(ValueError, match="together"):
        cache.append(0, q, k, k, table, ln, q_weight=w)
    with pytest.raises(TypeError, match="share"):
        cache.append(0, q, k, k, table, ln, q_weight=w, k_weight=w.float())
    with pytest.raises(ValueError, match="positions"):
        cache.append(0, q, k, k, table, ln, inv, positions=_int32([[0, 1]]))
    with pytest.raises(TypeError, match="positions"):
        cache.append(0, q, k, k, table, ln, inv, positions=torch.zeros(1, 3, device="cuda"))
    with pytest.raises(NotImplementedError, match="64"):
        cache.keep(table, ln, torch.zeros(1, 65, dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError, match="path"):
        cache.keep(table, ln, torch.zeros(1, 3, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="path"):
        cache.keep(table, ln, _int32([0, 1]))
    for name in ("keys", "num_pages", "page_tokens"):
        with pytest.raises(AttributeError):
            setattr(cache, name, 1)
    # Operands in the cache's pages.
    with pytest.raises(Exception, match="own buffers"):
        cache.append(0, q, cache.keys[0, :1, :, :3], k, table, ln)
    for x in (q, k, inv):
        y = x.clone().requires_grad_()
        with pytest.raises(RuntimeError, match="gradient"):
            cache.append(0, y if x is q else q, y if x is k else k, k, table, ln, y if x is inv else inv)
    with pytest.raises(RuntimeError, match="gradient"):
        cache.attend(0, q.clone().requires_grad_(), table, ln)
    # No rows, or no tokens.
    assert cache.attend(0, q[:0], table[:0], ln[:0]).shape == (0, 4, 3, 64)
    assert cache.attend(0, q[:, :, :0], table, ln).shape == (1, 4, 0, 64)
    assert cache.append(0, q[:, :, :0], k[:, :, :0], k[:, :, :0], table, ln, inv).shape == (1, 4, 0, 64)
    cache.keep(table, ln, torch.zeros(1, 0, dtype=torch.int32, device="cuda"))


def test_both_call_paths_agree(monkeypatch):
    """Plain tensors go through the native call path, others through Python; either way the same bits."""
    from pager_hf import _native as N

    ops = N.ops()

    class Counting:
        def __init__(self):
            self.taken = 0

        def __getattr__(self, name):
            def call(*args):
                got = getattr(ops, name)(*args)
                self.taken += got is not None
                return got
            return call

    class General:
        def __getattr__(self, name):
            return lambda *args: None

    rng = np.random.default_rng(67)
    g = torch.Generator().manual_seed(6)
    inv, _ = rotary_frequencies(64, device="cuda")
    x = torch.randn(3, 5, 8, 64, generator=g).half().cuda().transpose(1, 2)
    w = torch.rand(64, generator=g).half().cuda()
    parents, counts = _int32(_parents(rng, 3, 5)), _int32([5, 2, 0])
    pos = torch.randint(0, 999, (3, 5), generator=g).cuda()
    path = _int32([[1, 4, -1], [0, 2, 3], [3, -1, -1]])
    forms = {  # name: (overrides, whether every call takes the native path)
        "plain": (dict(), True),
        "ragged": (dict(counts=counts, window=7, softcap=3.0, scale=0.2, exact=True), True),
        "positions": (dict(positions=pos, interleaved=True, factor=1.5, weight=w.float()), True),
        "strided positions": (dict(positions=pos.t().contiguous().t().int()), True),
        "no norm, no turn": (dict(weight=None, inv=None), True),
        "strided table": (dict(wide=True), True),
        "int softcap": (dict(softcap=2), None),
        "strided counts": (dict(counts=_int32([[5, 0], [2, 0], [1, 0]])[:, 0]), None),
        "dense last": (dict(x=x.transpose(2, 3).contiguous().transpose(2, 3)), None),
    }
    for name, (o, taken) in forms.items():
        print(f"call path: {name}", flush=True)
        got = []
        for path_taken in (Counting(), General()):
            monkeypatch.setattr(N, "_ops", path_taken)
            cache, table = _filled(np.random.default_rng(71), 20, 16, 4, 2, 64, torch.float16, [30, 9, 0], 5, garbage=False)
            table = _int32(table)
            if o.get("wide"):
                table = torch.cat([table, table], dim=1)[:, : table.shape[1]]
            y = o.get("x", x)
            q, k, v = y[:, :4], y[:, 4:6], y[:, 6:]
            weight = o.get("weight", w)
            common = dict(counts=o.get("counts"), tree=draft_tree(parents))
            turned = cache.append(0, q, k, v, table, _int32([30, 9, 0]), o.get("inv", inv), positions=o.get("positions"),
                                  q_weight=weight, k_weight=weight, eps=1e-5, interleaved=o.get("interleaved", False),
                                  factor=o.get("factor", 1.0), **common)
            out = cache.attend(0, turned, table, _int32([30, 9, 0]), window=o.get("window"), softcap=o.get("softcap"),
                               scale=o.get("scale"), exact_weights=o.get("exact", False), **common)
            one = cache.attend(0, turned[:, :, 0], table, _int32([30, 9, 0]))
            last = cache.append(0, q[:, :, 0], k[:, :, 0], v[:, :, 0], table, _int32([30, 9, 0]), inv)
            cache.keep(table, _int32([30, 9, 0]), path)
            n = norm_rotary_embedding(q, k, pos, inv, w, w, eps=1e-5)
            n1 = norm_rotary_embedding(q[:, :, 0], None, pos[:, 0], inv, w, None)
            got.append([turned, out, one, last, cache.keys, cache.values, *n, n1[0], common["tree"].masks,
                        common["tree"].depths])
            assert out.stride() == got[0][1].stride() and out.transpose(1, 2).is_contiguous()
            if isinstance(path_taken, Counting) and taken:
                assert path_taken.taken == 8, (name, path_taken.taken)
        for a, b in zip(*got):
            assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b), name
