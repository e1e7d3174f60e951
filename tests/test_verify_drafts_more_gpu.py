"""The operators of drafted tokens on the GPU, further: weights, depths, batches, softcaps, forms of a call, norms."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import drafted_tokens as O
from pager_hf import DraftTree
from pager_hf import _native as N
from test_verify_drafts_gpu import CACHE_TYPES, _check_attend, _filled, _int32, _order

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
