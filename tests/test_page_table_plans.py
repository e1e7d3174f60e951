"""How attend calls over pages are dealt out, by the workspace they ask for (CPU)."""
from __future__ import annotations

import pytest

import _pgr_native as nat


def _cache(query_heads=4, kv_heads=2, head_dim=32, page_tokens=16):
    return nat.PTCache(keys=1 << 20, values=2 << 20, layers=1, pages=4, query_heads=query_heads, kv_heads=kv_heads,
                       page_tokens=page_tokens, head_dim=head_dim, dtype=1)


def _bytes(batch, tokens, capacity, **geometry):
    c = _cache(**geometry)
    return nat.load().pgr_pt_attend_workspace_bytes(c, batch, tokens, -(-capacity // c.page_tokens))


MOST = 1 << 30  # tokens of a row


@pytest.mark.parametrize("batch,tokens,capacity,cut", [
    (1, 1, MOST, True), (31, 1, MOST, True), (32, 1, MOST, False), (64, 1, MOST, False), (256, 1, MOST, False),
    (65535, 1, MOST, False), (64, 64, MOST, False), (128, 64, MOST, False), (64, 1, MOST >> 1, False), (64, 1, MOST >> 2, True),
])
def test_rows_whose_tiles_pass_32_bits_stay_whole(batch, tokens, capacity, cut):
    """The rows' tiles (32 tokens; 64 with more than 32 rows a KV head) are added up in 32 bits on the device, so a batch
    of 2^30 of them or more is not cut into parts. (Rows may share a table's row, so such a call can be made.)"""
    assert (_bytes(batch, tokens, capacity, query_heads=4, kv_heads=1) > 0) == cut


@pytest.mark.parametrize("geometry", [dict(query_heads=16, kv_heads=1, head_dim=32), dict(query_heads=8, kv_heads=1, head_dim=128),
                                      dict(query_heads=32, kv_heads=8, head_dim=128), dict(query_heads=8, kv_heads=2, head_dim=256)],
                         ids=str)
@pytest.mark.parametrize("tokens", [1, 5, 64])
def test_large_batches_stay_whole(tokens, geometry):
    """Finding a part walks the batch, in every workgroup: not above 256 rows."""
    for batch in (257, 300, 520, 1025, 4097, 7000):
        assert _bytes(batch, tokens, 4096, **geometry) == 0, batch
    assert _bytes(2, tokens, 4096, **geometry) > 0


@pytest.mark.parametrize("tokens", [1, 5])
def test_large_batches_with_room_for_long_rows_are_cut(tokens):
    for batch in (257, 300, 1000, 2000):
        assert _bytes(batch, tokens, 32768, query_heads=16, kv_heads=1, head_dim=32) > 0
    assert _bytes(8193, tokens, 32768, query_heads=16, kv_heads=1, head_dim=32) == 0


GEOMETRIES = [(32, 8, 128), (28, 4, 128), (14, 2, 64), (16, 1, 32), (16, 16, 64), (8, 1, 256), (4, 2, 16)]
SIZES = sorted({max(1, (1 << k) + i) for k in range(0, 18) for i in (-1, 0, 1)})


@pytest.mark.parametrize("geometry", GEOMETRIES, ids=str)
def test_the_workspace_is_bounded_whatever_the_batch_and_the_prompt(geometry):
    """256 MiB of parts at most (and 1 KiB a buffer for its alignment, and the batch's own table of parts)."""
    hq, hkv, d = geometry
    for batch in (1, 2, 3, 31, 64, 65, 128, 255, 256, 257, 300, 2049):
        for tokens in SIZES:
            if tokens * (hq // hkv) > 1 << 20 or batch * hkv * tokens * (hq // hkv) > 1 << 27:
                continue
            for held in (0, 1000, 32768, 1 << 20):
                n = _bytes(batch, tokens, tokens + held, query_heads=hq, kv_heads=hkv, head_dim=d)
                assert n <= (256 << 20) + 4096 + 8 * batch, (batch, tokens, held, n)


@pytest.mark.parametrize("batch,tokens,held,geometry", [
    (1, 8192, 0, (32, 8, 128)), (1, 8193, 0, (32, 8, 128)), (1, 16385, 0, (32, 8, 128)), (1, 2049, 0, (32, 8, 128)),
    (1, 65537, 0, (32, 8, 128)), (9, 130, 900, (32, 4, 64)), (130, 40, 500, (8, 2, 128)),
])
def test_calls_whose_parts_cost_more_than_they_bring_stay_whole(batch, tokens, held, geometry):
    hq, hkv, d = geometry
    assert _bytes(batch, tokens, tokens + held, query_heads=hq, kv_heads=hkv, head_dim=d) == 0


@pytest.mark.parametrize("batch,tokens,held,geometry", [
    (1, 2100, 16384, (32, 8, 128)), (65, 1, 4096, (32, 8, 128)), (33, 64, 4096, (32, 8, 128)), (65, 5, 4000, (28, 4, 128)),
    (1, 1, 1000, (14, 2, 64)), (8, 64, 32768, (28, 4, 128)), (8, 13, 8191, (32, 4, 64)),
])
def test_calls_that_parts_make_faster_are_cut(batch, tokens, held, geometry):
    hq, hkv, d = geometry
    assert _bytes(batch, tokens, tokens + held, query_heads=hq, kv_heads=hkv, head_dim=d) > 0
