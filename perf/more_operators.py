"""Cases of the operators that verify drafted tokens over a cache of pages: per-head norms with rotary
positions, the append into pages, the attention of a tree of drafted tokens (or of a prompt's chunk, or of one
token), and the move of the accepted tokens to the front.

Four kinds of case, each over a range of sizes:

``norm``    norm_rotary_embedding: RMS norm of each head of q and k, then the rotation;
``append``  PageTableCache.append: a row's new tokens, normed and rotated on the way, into its pages;
``attend``  PageTableCache.attend: the new tokens' attention over the row's pages, among themselves
            along the tree (or in order);
``keep``    PageTableCache.keep: the accepted path's keys and values to the front, in every layer.

``run`` computes the plain form (elementary torch operations) where ``own`` is false and calls the
framework's operators where it is true. ``exact`` gives the same values from their definitions in 64
bits."""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
EPS = 1e-6

# (query heads, KV heads, head dim)
QWEN_05B, QWEN_7B, TINYLLAMA, MISTRAL_7B = (14, 2, 64), (28, 4, 128), (32, 4, 64), (32, 8, 128)
WIDE = (8, 1, 256)
GEOMETRIES = [QWEN_05B, (12, 2, 128), QWEN_7B, TINYLLAMA, MISTRAL_7B, WIDE, (16, 1, 32), (16, 16, 64), (4, 2, 16)]


def _case(name, kind, geometry, dtype, batch, tokens, **more):
    hq, hkv, d = geometry
    return dict(name=name, kind=kind, q_heads=hq, kv_heads=hkv, head_dim=d, dtype=dtype, batch=batch, tokens=tokens,
                **more)


def listed():
    return [
        # The smallest: q and k of one decode step of one sequence. Latency.
        _case("norm_step", "norm", QWEN_7B, "bfloat16", 1, 1, rotary=128, interleaved=False, first=131071),
        # A batch of prompts. Bandwidth.
        _case("norm_prompts", "norm", MISTRAL_7B, "bfloat16", 4, 8191, rotary=128, interleaved=False, first=0),
        # A prompt's chunk in 32 bits, adjacent pairs, half of the head turned.
        _case("norm_float32", "norm", TINYLLAMA, "float32", 2, 1023, rotary=32, interleaved=True, first=4096),
        # A decode step of one sequence. Latency.
        _case("append_one", "append", QWEN_05B, "float16", 1, 1, context=4096, shortest=4096, page=16, tree=False,
              norm=False, ragged=False),
        # A batch's drafted trees of ragged sizes, heads normed on the way.
        _case("append_tree", "append", MISTRAL_7B, "bfloat16", 16, 29, context=2047, shortest=100, page=32, tree=True,
              norm=True, ragged=True),
        # Prompts into empty caches. Bandwidth.
        _case("append_prompts", "append", MISTRAL_7B, "bfloat16", 4, 8191, context=0, shortest=0, page=64, tree=False,
              norm=True, ragged=True),
        # One sequence, one token, a short cache: latency and launches.
        _case("attend_one", "attend", QWEN_05B, "float16", 1, 1, context=1000, shortest=1000, page=16, tree=False,
              ragged=False, window=0, softcap=0.0),
        # Drafted trees over ragged rows, the shortest empty, softcapped.
        _case("attend_tree", "attend", TINYLLAMA, "bfloat16", 8, 13, context=8191, shortest=0, page=32, tree=True,
              ragged=True, window=0, softcap=30.0),
        # Trees of the largest size over long rows: the largest read.
        _case("attend_wide", "attend", QWEN_7B, "bfloat16", 8, 64, context=32768, shortest=30011, page=64, tree=True,
              ragged=False, window=0, softcap=0.0),
        # A prompt's chunk behind what is cached already: bound by arithmetic.
        _case("attend_chunk", "attend", MISTRAL_7B, "bfloat16", 1, 2048, context=16384, shortest=16384, page=128,
              tree=False, ragged=False, window=0, softcap=0.0),
        # The accepted path of one sequence, layers of a small model.
        _case("keep_one", "keep", QWEN_05B, "float16", 1, 16, context=4096, shortest=4096, page=16, layers=24),
        # A batch's accepted paths, layers of a large one.
        _case("keep_batch", "keep", MISTRAL_7B, "bfloat16", 64, 61, context=333, shortest=5, page=32, layers=32),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "append", "attend", "attend", "keep"])
    geometry = rng.choice(GEOMETRIES)
    hq, hkv, d = geometry
    dtype = rng.choice(["float16", "bfloat16"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "norm":
        batch = _spread(rng, 1, 32)
        tokens = _spread(rng, 1, max(1, (1 << 26) // (batch * (hq + hkv) * d)))
        return _drawn(_case("", kind, geometry, rng.choice(list(DTYPES)), batch, tokens,
                            rotary=rng.choice([d, d // 2, d // 4 * 2]), interleaved=rng.random() < 0.5,
                            first=_spread(rng, 1, 1 << 20) - 1))
    if kind == "keep":
        batch, tokens = _spread(rng, 1, 64), _spread(rng, 2, 64)
        layers = _spread(rng, 1, max(1, min(48, (1 << 26) // (batch * tokens * hkv * d))))
        context = _spread(rng, 1, 256)
        return _drawn(_case("", kind, geometry, dtype, batch, tokens, context=context, shortest=rng.randrange(context + 1),
                            page=page, layers=layers))
    if kind == "append":
        batch, tree = _spread(rng, 1, 32), rng.random() < 0.5
        tokens = _spread(rng, 1, 64) if tree else _spread(rng, 1, max(1, (1 << 26) // (batch * (hq + 2 * hkv) * d)))
        context = _spread(rng, 1, 4096)
        return _drawn(_case("", kind, geometry, dtype, batch, tokens, context=context, shortest=rng.randrange(context + 1),
                            page=page, tree=tree, norm=rng.random() < 0.5, ragged=rng.random() < 0.5))
    # One token, a tree or a chain of drafts, or a prompt's chunk.
    form = rng.choice(["one", "draft", "draft", "chunk"])
    tokens = {"one": 1, "draft": _spread(rng, 2, 64), "chunk": _spread(rng, 65, 2048)}[form]
    batch = _spread(rng, 1, 32 if form != "chunk" else 2)
    most = (1 << 26) // (batch * hkv * d) if form != "chunk" else (1 << 37) // (batch * hq * tokens * d)
    context = _spread(rng, 1, max(1, min(32768, most)))
    return _drawn(_case("", kind, geometry, dtype, batch, tokens, context=context, shortest=rng.randrange(context + 1),
                        page=page, tree=form == "draft" and rng.random() < 0.7, ragged=rng.random() < 0.5,
                        window=rng.choice([0, 0, 0, _spread(rng, 1, 4096)]), softcap=rng.choice([0.0, 0.0, 30.0])))


def _drawn(case):
    return {k: v for k, v in case.items() if k != "name"}


def _lengths(case):
    """Tokens each row holds: spread evenly between the shortest and the longest."""
    b, n, lo = case["batch"], case["context"], case["shortest"]
    return [n if b == 1 else lo + (n - lo) * i // (b - 1) for i in range(b)]


def _counts(case):
    """New tokens of each row."""
    b, t = case["batch"], case["tokens"]
    return [t - (t * i // (2 * b) if case.get("ragged") else 0) for i in range(b)]


def _framework():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rust-llm-pager_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from pager_hf import page_table_cache, rotary

    return page_table_cache, rotary


class _Cache:
    """The buffers of a cache of pages, as PageTableCache names them."""

    def __init__(self, layers, pages, page, hkv, d, dtype):
        self.keys = torch.zeros(layers, pages, hkv, page, d, dtype=dtype, device="cuda")
        self.values = torch.zeros(layers, pages, hkv, page, d, dtype=dtype, device="cuda")


def _normal(g, dtype, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype) * scale


def _inv_freq(rotary):
    return (1.0 / 10000.0 ** (torch.arange(0, rotary, 2, dtype=torch.float64) / max(rotary, 1))).float().cuda()


def _weights(g, dtype, d):
    """A norm's weights: about 1."""
    return (1.0 + 0.25 * torch.randn(d, generator=g, device="cuda")).to(dtype)


def _parents(case, seed):
    """A tree for each row: -1 for a root, else an earlier token; long paths and short ones."""
    g = torch.Generator().manual_seed(seed)
    b, t = case["batch"], case["tokens"]
    at = torch.arange(t)
    back = 1 + (torch.rand(b, t, generator=g) ** 4 * 8).long()
    return (at - back).clamp(min=-1).int()


def _ancestors(parents):
    """(what each token sees among the drafted ones [B, T, T], its depth [B, T])."""
    b, t = parents.shape
    sees = torch.zeros(b, t, t, dtype=torch.bool)
    for i in range(t):
        for r in range(b):
            p = int(parents[r, i])
            if p >= 0:
                sees[r, i] = sees[r, p]
            sees[r, i, i] = True
    return sees, sees.sum(dim=-1).int() - 1


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, b, t, hq, hkv, d = (case[k] for k in ("kind", "batch", "tokens", "q_heads", "kv_heads", "head_dim"))
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if kind == "norm":
        # As a model's projections come: [batch, tokens, heads, head_dim], seen as [batch, heads, tokens, head_dim].
        s["q"] = _normal(g, dtype, b, t, hq, d, scale=2.0).transpose(1, 2)
        s["k"] = _normal(g, dtype, b, t, hkv, d, scale=2.0).transpose(1, 2)
        s["q_weight"], s["k_weight"] = _weights(g, dtype, d), _weights(g, dtype, d)
        s["positions"] = case["first"] + torch.arange(t, device="cuda").repeat(b, 1)
        s["inv_freq"] = _inv_freq(case["rotary"])
        return s

    # Rows' pages, scattered over the pool; entries behind a row's last page name none.
    page, lens, counts = case["page"], _lengths(case), _counts(case)
    need = [-(-(n + t) // page) for n in lens]
    pages = sum(need) + 1
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int()
    table, first = torch.full((b, max(need)), -1, dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[first: first + n]
        first += n
    s["table"] = table.cuda()
    s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda") if case.get("ragged") else None
    layers = case.get("layers", 1)
    if own:
        pt, _ = _framework()
        cache = pt.PageTableCache(layers, pages, page, hq, hkv, d, dtype, "cuda")
    else:
        cache = _Cache(layers, pages, page, hkv, d, dtype)
    cache.keys.copy_(_normal(g, dtype, layers, pages, hkv, page, d))
    cache.values.copy_(_normal(g, dtype, layers, pages, hkv, page, d))
    s["cache"] = cache
    if kind == "keep":
        # The path of a leaf of each row's tree: drafted tokens in order, -1 behind the last.
        sees, depth = _ancestors(_parents(case, seed))
        path = torch.full((b, t), -1, dtype=torch.int32)
        for i in range(b):
            leaf = int(depth[i].argmax()) if i % 4 else t - 1
            taken = sees[i, leaf].nonzero()[:, 0]
            path[i, : taken.numel()] = taken.int()
        s["path"] = path[:, : int((path >= 0).sum(dim=1).max())].contiguous().cuda()
        return s
    s["tree"] = s["sees"] = s["depths"] = None
    if case["tree"]:
        parents = _parents(case, seed)
        if own:  # made once a step, for all layers
            s["tree"] = pt.draft_tree(parents.cuda())
        else:
            sees, depth = _ancestors(parents)
            s["sees"], s["depths"] = sees.cuda(), depth.cuda()
    if kind == "append":
        # Views into one projection, as a model's fused q/k/v product gives them.
        qkv = _normal(g, dtype, b, t, (hq + 2 * hkv) * d)
        s["q"], s["k"], s["v"] = (x.unflatten(-1, (-1, d)).transpose(1, 2)
                                  for x in qkv.split([hq * d, hkv * d, hkv * d], dim=-1))
        s["inv_freq"] = _inv_freq(d)
        s["q_weight"] = _weights(g, dtype, d) if case["norm"] else None
        s["k_weight"] = _weights(g, dtype, d) if case["norm"] else None
        return s
    s["q"] = _normal(g, dtype, b, hq, t, d, scale=2.0)
    return s


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        _, rotary = _framework()
        if kind == "norm":
            return rotary.norm_rotary_embedding(s["q"], s["k"], s["positions"], s["inv_freq"], s["q_weight"],
                                                s["k_weight"], eps=EPS, interleaved=case["interleaved"])
        cache = s["cache"]
        if kind == "append":
            q = cache.append(0, s["q"], s["k"], s["v"], s["table"], s["lengths"], s["inv_freq"], counts=s["counts"],
                             tree=s["tree"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS)
            return [q, cache.keys, cache.values]
        if kind == "attend":
            return cache.attend(0, s["q"], s["table"], s["lengths"], counts=s["counts"], tree=s["tree"],
                                window=case["window"], softcap=case["softcap"])
        cache.keep(s["table"], s["lengths"], s["path"])
        return [cache.keys, cache.values]
    if kind == "norm":
        return tuple(_rotate(_norm(x, w), s["positions"][:, None], s["inv_freq"], case["interleaved"]).to(x.dtype)
                     for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))
    cache = s["cache"]
    if kind == "append":
        return [_append(s), cache.keys, cache.values]
    if kind == "attend":
        return _attend(s)
    _keep(s)
    return [cache.keys, cache.values]


# ---- plain forms ---------------------------------------------------------------------------------
def _norm(x, weight):
    f = x.float()
    return f * torch.rsqrt(f.square().mean(dim=-1, keepdim=True) + EPS) * weight.float()


def _rotate(f, positions, inv_freq, interleaved):
    """f [..., D] in 32 bits at positions [...]: angles in 64 bits, products in 32."""
    r = 2 * inv_freq.numel()
    angle = positions[..., None].double() * inv_freq.double()
    cos, sin = angle.cos().float(), angle.sin().float()
    if interleaved:
        a, b = f[..., 0:r:2], f[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = f[..., : r // 2], f[..., r // 2: r]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([y, f[..., r:]], dim=-1)


def _new_tokens(s):
    """Columns [T], which of them each row has [B, T]."""
    t = s["case"]["tokens"]
    at = torch.arange(t, device="cuda")
    has = torch.ones(s["case"]["batch"], t, dtype=torch.bool, device="cuda")
    return at, has if s["counts"] is None else at < s["counts"][:, None]


def _append(s):
    case, cache = s["case"], s["cache"]
    page = case["page"]
    at, has = _new_tokens(s)
    slot = s["lengths"].long()[:, None] + at
    positions = slot if s["depths"] is None else s["lengths"].long()[:, None] + s["depths"]
    turned = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        f = x.float() if w is None else _norm(x, w)
        turned.append(_rotate(f, positions[:, None], s["inv_freq"], False).to(x.dtype))
    where = s["table"].gather(1, slot // page).long()[has]
    cache.keys[0, where, :, (slot % page)[has]] = turned[1].transpose(1, 2)[has]
    cache.values[0, where, :, (slot % page)[has]] = s["v"].transpose(1, 2)[has]
    return turned[0] * has[:, None, :, None]


def _attend(s):
    case, cache, q = s["case"], s["cache"], s["q"]
    b, hq, t, d = q.shape
    hkv, page, window = case["kv_heads"], case["page"], case["window"]
    at, has = _new_tokens(s)
    n = s["table"].shape[1] * page
    out = torch.zeros(b, t, hq, d, dtype=q.dtype, device="cuda")
    for i in range(b):
        rows = s["table"][i].clamp(min=0).long()
        k = cache.keys[0, rows].transpose(0, 1).reshape(hkv, n, d).float()
        v = cache.values[0, rows].transpose(0, 1).reshape(hkv, n, d).float()
        col, length = torch.arange(n, device="cuda"), s["lengths"][i].long()
        new = (col - length).clamp(0, t - 1)
        depth = at if s["depths"] is None else s["depths"][i].long()
        among = at[:, None] >= new if s["sees"] is None else s["sees"][i][:, new]
        ok = (col < length) | ((col >= length) & (col - length < t) & among & has[i][new])
        if window > 0:
            position = torch.where(col < length, col, length + depth[new])
            ok = ok & (position > (length + depth)[:, None] - window)
        x = torch.matmul((q[i].float() / math.sqrt(d)).reshape(hkv, hq // hkv * t, d), k.transpose(1, 2).contiguous())
        x = x.view(hq, t, n)
        if case["softcap"] > 0:
            x = case["softcap"] * torch.tanh(x / case["softcap"])
        x = x.masked_fill(~ok, -math.inf)
        x = (x - x.amax(dim=-1, keepdim=True)).exp()  # (a token sees itself: none of those that count is empty)
        x = x / x.sum(dim=-1, keepdim=True)
        v = v.masked_fill((col >= length + t)[:, None], 0.0)
        y = torch.matmul(x.view(hkv, hq // hkv * t, n), v).view(hq, t, d)
        out[i] = torch.where(has[i][:, None], y, 0.0).transpose(0, 1).to(q.dtype)
    return out.transpose(1, 2)


def _keep(s):
    cache, page, path = s["cache"], s["case"]["page"], s["path"]
    moved = path >= 0
    old = s["lengths"].long()[:, None] + path.clamp(min=0)
    new = s["lengths"].long()[:, None] + torch.arange(path.shape[1], device="cuda")
    source, target = (s["table"].gather(1, x // page).long()[moved] for x in (old, new))
    for x in (cache.keys, cache.values):
        x[:, target, :, (new % page)[moved]] = x[:, source, :, (old % page)[moved]]


# ---- work and exact values -----------------------------------------------------------------------
def _visible(case):
    """(tokens read, pairs of a query and a token) of an attention, over all rows of one head. What a drafted
    token sees among the drafted ones is counted as half of them."""
    read = pairs = 0
    w = case["window"]
    for n, c in zip(_lengths(case), _counts(case)):
        if w <= 0:
            read += n + c
            pairs += c * n + c * (c + 1) // 2
        else:
            read += min(n, w - 1) + c
            pairs += sum(min(w, n + i + 1) for i in range(c))
    return read, pairs


def work(case):
    kind, b, t, hq, hkv, d = (case[k] for k in ("kind", "batch", "tokens", "q_heads", "kv_heads", "head_dim"))
    e = 4 if case["dtype"] == "float32" else 2
    if kind == "norm":
        n = b * t * (hq + hkv)
        return {"bytes": 2 * n * d * e + b * t * 8 + 2 * d * e + 2 * case["rotary"],
                "flops": n * (4 * d + 3 * case["rotary"])}
    if kind == "append":
        n = sum(_counts(case))
        return {"bytes": 2 * n * (hq + 2 * hkv) * d * e + 4 * n, "flops": n * (hq + hkv) * d * (7 if case["norm"] else 3)}
    if kind == "attend":
        read, pairs = _visible(case)
        return {"bytes": (2 * hkv * read + 2 * hq * sum(_counts(case))) * d * e, "flops": 4 * hq * pairs * d}
    # An accepted path takes about a third of the tree.
    return {"bytes": case["layers"] * b * max(1, t // 3) * hkv * d * e * 4, "flops": 1}


def _turned(x, positions, inv_freq, interleaved):
    """x as complex numbers times e^(i a), in 64 bits."""
    r = 2 * inv_freq.numel()
    y = x.double().clone()
    z = torch.complex(y[..., 0:r:2], y[..., 1:r:2]) if interleaved else torch.complex(y[..., : r // 2], y[..., r // 2: r])
    z = z * torch.exp(1j * (positions.double()[..., None] * inv_freq.double()))
    if interleaved:
        y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
    else:
        y[..., : r // 2], y[..., r // 2: r] = z.real, z.imag
    return y


def _unit(x, weight):
    """x over its root mean square, times the weight, in 64 bits."""
    y = x.double()
    return y / (torch.linalg.vector_norm(y, dim=-1, keepdim=True).square() / y.shape[-1] + EPS).sqrt() * weight.double()


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    kind, b, t, hq, hkv, d = (case[k] for k in ("kind", "batch", "tokens", "q_heads", "kv_heads", "head_dim"))
    rep = hq // hkv
    if kind == "norm":
        p = s["positions"][:, None, :]
        # A few heads at a time: 64-bit complex copies of the whole would not fit beside each other.
        return tuple(torch.cat([_turned(_unit(x[:, h: h + 4], w), p, s["inv_freq"], case["interleaved"])
                                for h in range(0, x.shape[1], 4)], dim=1)
                     for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))
    cache, page, lens, counts = s["cache"], case["page"], _lengths(case), _counts(case)
    table = s["table"].cpu()

    def cells(i, first, n):
        """Page and place of row i's tokens [first, first + n)."""
        at = torch.arange(first, first + n)
        return table[i, at // page].long().cuda(), (at % page).cuda()

    if kind == "keep":
        keys, values = cache.keys.clone(), cache.values.clone()
        for i in range(b):
            taken = [int(x) for x in s["path"][i].cpu() if x >= 0]
            for j, x in enumerate(taken):
                (sp, so), (tp, to) = cells(i, lens[i] + x, 1), cells(i, lens[i] + j, 1)
                keys[:, tp[0], :, to[0]] = cache.keys[:, sp[0], :, so[0]]
                values[:, tp[0], :, to[0]] = cache.values[:, sp[0], :, so[0]]
        return [keys.double(), values.double()]
    if kind == "append":
        q = torch.zeros(b, hq, t, d, dtype=torch.float64, device="cuda")
        keys, values = cache.keys.double(), cache.values.double()
        for i in range(b):
            n = counts[i]
            p = lens[i] + (torch.arange(t, device="cuda") if s["depths"] is None else s["depths"][i].long())[:n]
            x, y = s["q"][i, :, :n].double(), s["k"][i, :, :n].double()
            if s["q_weight"] is not None:
                x, y = _unit(x, s["q_weight"]), _unit(y, s["k_weight"])
            q[i, :, :n] = _turned(x, p[None], s["inv_freq"], False)
            pp, oo = cells(i, lens[i], n)
            keys[0, pp, :, oo] = _turned(y, p[None], s["inv_freq"], False).transpose(0, 1)
            values[0, pp, :, oo] = s["v"][i, :, :n].double().transpose(0, 1)
        return [q, keys, values]
    out = torch.zeros(b, hq, t, d, dtype=torch.float64, device="cuda")
    for i in range(b):
        length, n = lens[i], counts[i]
        pp, oo = cells(i, 0, length + n)
        sees = torch.ones(n, n, dtype=torch.bool, device="cuda").tril() if s["sees"] is None else s["sees"][i][:n, :n]
        depth = torch.arange(n, device="cuda") if s["depths"] is None else s["depths"][i][:n].long()
        hidden = torch.cat([torch.zeros(n, length, dtype=torch.bool, device="cuda"), ~sees], dim=1)
        if case["window"] > 0:
            position = torch.cat([torch.arange(length, device="cuda"), length + depth])
            hidden |= (length + depth)[:, None] - position >= case["window"]
        for h in range(hkv):
            k, v = cache.keys[0, pp, h, oo].double(), cache.values[0, pp, h, oo].double()
            for e in range(rep):
                x = s["q"][i, h * rep + e, :n].double() @ k.t() / math.sqrt(d)
                if case["softcap"] > 0:
                    x = case["softcap"] * torch.tanh(x / case["softcap"])
                out[i, h * rep + e, :n] = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1) @ v
    return out
