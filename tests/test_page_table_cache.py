"""The cache of pages and the normed rotary embedding: refusals and the oracle (CPU)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import _pgr_native as nat
from oracle import drafted_tokens as O
from pager_hf.page_table_cache import PageTableCache, draft_tree
from pager_hf.rotary import norm_rotary_embedding

INV, UNS, CAP = nat.PGR_ERR_INVALID, nat.PGR_ERR_UNSUPPORTED, nat.PGR_ERR_CAPACITY
S = (ctypes.c_int64 * 3)(1, 1, 1)
FAR = 1 << 30


def _cache(**over):
    fields = dict(keys=1 << 20, values=2 << 20, layers=2, pages=4, query_heads=4, kv_heads=2, page_tokens=16, head_dim=32,
                  dtype=0)
    return nat.PTCache(**{**fields, **over})


def _rows(**over):
    fields = dict(table=FAR, table_stride=3, width=3, lengths=FAR, counts=None, batch=1, tokens=4)
    return nat.PTRows(**{**fields, **over})


def _append(c=None, layer=0, r=None, q=FAR, k=FAR, v=FAR, q_out=8 << 20, positions=None, long=0, depths=None, inv=None,
            rotary=0, factor=1.0, qw=None, kw=None, f32=0, eps=1e-6, strides=S):
    return nat.load().pgr_pt_append(c or _cache(), layer, r or _rows(), q, strides, k, strides, v, strides, q_out, positions,
                                    long, S if positions else None, depths, inv, rotary, 0, factor, qw, kw, f32, eps, None)


def _attend(c=None, layer=0, r=None, q=FAR, out=8 << 20, masks=None, depths=None, window=0, scale=1.0, softcap=0.0,
            ws=16 << 20, nbytes=1 << 20, strides=S):
    return nat.load().pgr_pt_attend(c or _cache(), layer, r or _rows(), q, strides, out, masks, depths, window, scale, softcap,
                                    0, ws, nbytes, None)


def _keep(c=None, r=None, path=FAR):
    return nat.load().pgr_pt_keep(c or _cache(), r or _rows(), path, None)


BAD_CACHES = [
    (dict(query_heads=3), INV), (dict(query_heads=34), UNS), (dict(head_dim=48), UNS), (dict(dtype=2), UNS),
    (dict(page_tokens=8), UNS), (dict(page_tokens=48), UNS), (dict(page_tokens=512), UNS), (dict(layers=0), INV),
    (dict(pages=0), INV), (dict(pages=(1 << 30) + 1), INV), (dict(layers=65536), INV), (dict(keys=0), INV),
    (dict(values=(2 << 20) + 8), INV), (dict(kv_heads=0), INV), (dict(layers=65535, kv_heads=8192, query_heads=8192), INV),
]


@pytest.mark.parametrize("over,code", BAD_CACHES, ids=[str(x[0]) for x in BAD_CACHES])
def test_c_entries_refuse_a_bad_cache(over, code):
    c = _cache(**over)
    assert _append(c) == code and _attend(c) == code and _keep(c) == code
    assert nat.load().pgr_pt_attend_workspace_bytes(c, 1, 4, 3) == 0


BAD_ROWS = [dict(batch=-1), dict(tokens=-1), dict(width=-1), dict(batch=32768), dict(width=(1 << 26) + 1), dict(table=None),
            dict(lengths=None)]


@pytest.mark.parametrize("over", BAD_ROWS, ids=str)
def test_c_entries_refuse_bad_rows(over):
    r = _rows(**over)
    assert _append(r=r) == INV and _attend(r=r) == INV and _keep(r=r) == INV


def test_c_entries_refuse_bad_arguments():
    assert _append(layer=2) == INV and _append(layer=-1) == INV and _attend(layer=2) == INV
    for name in ("q", "k", "v", "q_out"):
        assert _append(**{name: None}) == INV, name
    assert _append(rotary=2) == INV  # no inv_freq
    assert _append(inv=FAR, rotary=34) == INV and _append(inv=FAR, rotary=3) == INV
    assert _append(factor=float("nan")) == INV
    assert _append(qw=FAR) == INV and _append(kw=FAR) == INV
    assert _append(qw=FAR, kw=FAR, eps=-1.0) == INV and _append(qw=FAR, kw=FAR, eps=float("inf")) == INV
    assert _append(r=_rows(tokens=1 << 26)) == INV
    assert _attend(q=None) == INV and _attend(out=None) == INV
    assert _attend(scale=0.0) == INV and _attend(softcap=float("nan")) == INV and _attend(window=-1) == INV
    assert _attend(masks=FAR) == INV and _attend(depths=FAR) == INV
    assert _attend(r=_rows(tokens=65), masks=FAR, depths=FAR) == UNS
    assert _attend(r=_rows(tokens=(1 << 19) + 1)) == INV
    assert _keep(path=None) == INV and _keep(r=_rows(tokens=65)) == UNS
    # Nothing to do.
    for r in (_rows(batch=0), _rows(tokens=0)):
        assert _append(r=r) == 0 and _attend(r=r) == 0 and _keep(r=r) == 0
    lib = nat.load()
    assert lib.pgr_draft_tree(None, 1, 4, FAR, FAR, None) == INV
    assert lib.pgr_draft_tree(FAR, 1, 65, FAR, FAR, None) == UNS
    assert lib.pgr_draft_tree(FAR, -1, 4, FAR, FAR, None) == INV
    assert lib.pgr_draft_tree(FAR, 1, 4, FAR, FAR + 4096, None) == INV  # masks over the parents
    assert lib.pgr_draft_tree(FAR, 1, 4, FAR + 4096, FAR + 4100, None) == INV
    assert lib.pgr_draft_tree(None, 0, 4, None, None, None) == 0


def test_workspace_of_an_attend_call():
    lib, c = nat.load(), _cache()
    r = _rows(width=1000)
    need = lib.pgr_pt_attend_workspace_bytes(c, 1, 4, 1000)
    assert need > 0
    assert _attend(r=r, nbytes=need - 1) == CAP and _attend(r=r, ws=None, nbytes=need) == CAP
    assert _attend(r=r, ws=(16 << 20) + 8, nbytes=need) == INV
    assert lib.pgr_pt_attend_workspace_bytes(c, 0, 4, 1000) == 0
    assert lib.pgr_pt_attend_workspace_bytes(c, 1, 0, 1000) == 0
    assert lib.pgr_pt_attend_workspace_bytes(c, 1, 1 << 20, 1000) == 0  # refused


# Where the buffers of _cache() begin and their bytes: 2 layers x 4 pages x 2 heads x 16 tokens x 32 dims.
BUFFERS = dict(keys=(1 << 20, 2 * 4 * 2 * 16 * 32 * 2), values=(2 << 20, 2 * 4 * 2 * 16 * 32 * 2))


@pytest.mark.parametrize("name", list(BUFFERS))
def test_c_entries_refuse_operands_in_the_cache(name):
    base, size = BUFFERS[name]

    def refused(rc):
        assert rc == INV and "own buffers" in nat.last_error()

    for at in (base, base + size - 4, base - 2):
        for x in ("q", "k", "v", "q_out"):
            refused(_append(**{x: at}))
        refused(_append(positions=at))
        refused(_append(positions=at, long=1))
        refused(_append(depths=at))
        refused(_append(inv=at, rotary=32))
        refused(_append(qw=at, kw=FAR))
        refused(_append(qw=FAR, kw=at, f32=1))
        for x in ("table", "lengths", "counts"):
            refused(_append(r=_rows(**{x: at})))
        refused(_attend(out=at))
        refused(_attend(r=_rows(width=1000), ws=at & ~15 if at > base else base - 16))
        refused(_keep(path=at))
        refused(_keep(r=_rows(table=at)))
        refused(_keep(r=_rows(lengths=at)))
    # One of the operand's rows reaches the buffer.
    far = (ctypes.c_int64 * 3)(1, (base - FAR) // 2, 1)
    refused(_append(k=FAR, strides=far))


def test_c_entries_refuse_outputs_over_their_inputs():
    out = 8 << 20
    size = 1 * 4 * 4 * 32 * 2

    def refused(rc):
        assert rc == INV and "overlap" in nat.last_error()

    for at in (out, out + size - 2, out - 2):
        for x in ("q", "k", "v"):
            refused(_append(**{x: at}))
        refused(_append(depths=at))
        refused(_append(positions=at))
        refused(_append(inv=at, rotary=32))
        refused(_append(qw=at, kw=FAR))
        refused(_attend(q=at))
        refused(_attend(masks=at, depths=FAR))
        refused(_attend(masks=FAR, depths=at))
        for x in ("table", "lengths", "counts"):
            refused(_append(r=_rows(**{x: at})))
            refused(_attend(r=_rows(**{x: at})))
    wide = _rows(width=1000)
    refused(_attend(r=wide, q=16 << 20))
    refused(_attend(r=wide, ws=out + size - 16))


def test_normed_rotary_refuses_before_any_launch():
    lib = nat.load()

    def call(q=FAR, q_out=8 << 20, q_heads=2, k=FAR, k_out=9 << 20, k_heads=1, qw=FAR, kw=FAR, f32=0, eps=1e-6, pos=FAR,
             inv=FAR, rotary=8, batch=1, tokens=4, d=16, dtype=0, factor=1.0):
        return lib.pgr_norm_rotary(q, S, q_out, q_heads, k, S, k_out, k_heads, qw, kw, f32, eps, pos, 0, S, inv, rotary, batch,
                                   tokens, d, dtype, 0, factor, None)

    assert call(batch=0) == 0 and call(tokens=0) == 0 and call(q_heads=0, k_heads=0) == 0
    for bad in (dict(q_heads=-1), dict(tokens=-1), dict(d=0), dict(dtype=3), dict(q=None), dict(k_out=None), dict(qw=None),
                dict(kw=None), dict(eps=-1.0), dict(eps=float("nan")), dict(pos=None), dict(inv=None), dict(rotary=7),
                dict(rotary=18), dict(factor=float("inf")), dict(tokens=1 << 26), dict(batch=1 << 25, tokens=4),
                dict(q_heads=40000)):
        assert call(**bad) == INV, bad
    # Outputs over inputs, and over each other.
    for bad in (dict(q_out=FAR), dict(k_out=FAR + 2), dict(qw=8 << 20), dict(kw=(9 << 20) + 2), dict(pos=8 << 20),
                dict(inv=9 << 20), dict(k_out=(8 << 20) + 2 * 4 * 16 * 2 - 2)):
        assert call(**bad) == INV and "overlap" in nat.last_error(), bad


def test_python_refusals_need_no_gpu():
    q, k, w = torch.zeros(1, 2, 4, 16), torch.zeros(1, 1, 4, 16), torch.ones(16)
    pos, inv = torch.zeros(1, 4, dtype=torch.int64), torch.ones(8)
    with pytest.raises(ValueError, match="CUDA"):
        norm_rotary_embedding(q, k, pos, inv, w, w)
    with pytest.raises(NotImplementedError, match="float64"):
        norm_rotary_embedding(q.double(), k.double(), pos, inv, w, w)
    with pytest.raises(TypeError, match="one dtype"):
        norm_rotary_embedding(q, k.half(), pos, inv, w, w)
    with pytest.raises(ValueError, match="does not match"):
        norm_rotary_embedding(q, k[:, :, :3], pos, inv, w, w)
    with pytest.raises(ValueError, match="together"):
        norm_rotary_embedding(q, None, pos, inv, w, w)
    with pytest.raises(ValueError, match="must be"):
        norm_rotary_embedding(q[0, 0], None, pos, inv, w, None)
    with pytest.raises(RuntimeError, match="gradient"):
        norm_rotary_embedding(q, k, pos, inv, w.clone().requires_grad_(), w)
    with pytest.raises(ValueError, match="CUDA"):
        draft_tree(torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(TypeError, match="int32"):
        draft_tree(torch.zeros(1, 4, dtype=torch.int64))
    with pytest.raises(ValueError, match="must be"):
        draft_tree(torch.zeros(4, dtype=torch.int32))

    def make(layers=1, pages=4, page=16, hq=4, hkv=2, d=32, dtype=torch.float16, device="cuda:0"):
        return PageTableCache(layers, pages, page, hq, hkv, d, dtype, device)

    for bad in (dict(layers=0), dict(pages=0), dict(hq=3), dict(device="cpu"), dict(pages=(1 << 30) + 1), dict(layers=65536)):
        with pytest.raises(ValueError):
            make(**bad)
    for bad in (dict(page=24), dict(page=8), dict(hq=34), dict(d=48), dict(dtype=torch.float32)):
        with pytest.raises(NotImplementedError):
            make(**bad)


# ---- oracle --------------------------------------------------------------------------------------
def test_oracle_tree():
    sees, depth = O.tree(np.array([[-1, 0, 1, 0, 9, 4]]))
    assert depth.tolist() == [[0, 1, 2, 1, 0, 1]]
    assert sees[0].astype(int).tolist() == [[1, 0, 0, 0, 0, 0], [1, 1, 0, 0, 0, 0], [1, 1, 1, 0, 0, 0], [1, 0, 0, 1, 0, 0],
                                            [0, 0, 0, 0, 1, 0], [0, 0, 0, 0, 1, 1]]


def test_oracle_norm_is_of_unit_size():
    x = np.random.default_rng(0).standard_normal((3, 64)) * 7
    y, bound = O.norm(x, np.ones(64), 0.0)
    np.testing.assert_allclose((y * y).mean(axis=-1), 1.0)
    assert np.all(bound > 0)


def test_oracle_cells():
    page, place = O.cells([5, -1, 2, 9], 16, 8, 14, 52)
    assert page[0] == 5 and place[0] == 14 and page[2] == -1 and page[18] == 2 and place[18] == 0
    assert page[34] == -1 and page[-1] == -1  # outside the pool, behind the table


def test_oracle_attention_of_a_chain_is_causal():
    rng = np.random.default_rng(1)
    q, k, v = rng.standard_normal((2, 3, 8)), rng.standard_normal((7, 8)), rng.standard_normal((7, 8))
    out, _ = O.attend_row(q, k, v, np.ones(7, bool), 4, 3, np.tril(np.ones((3, 3), bool)), np.arange(3), 0, 0.5, 0.0, 0, 0, 0)
    for t in range(3):
        s = q[:, t] @ k[: 5 + t].T * 0.5
        p = np.exp(s) / np.exp(s).sum(-1, keepdims=True)
        np.testing.assert_allclose(out[:, t], p @ v[: 5 + t])
    near, _ = O.attend_row(q, k, v, np.ones(7, bool), 4, 3, np.tril(np.ones((3, 3), bool)), np.arange(3), 1, 0.5, 0.0, 0, 0, 0)
    np.testing.assert_allclose(near, np.broadcast_to(v[4:], near.shape))
