"""The bounded cache's refusals and its oracle (CPU)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import _pgr_native as nat
from oracle import bounded_cache as O
from pager_hf.heavy_hitter_cache import HeavyHitterCache, prompt_attention_weights


def _cache(**over):
    fields = dict(keys=256, values=256, weights=256, order=256, lengths=256, seen=256, batch=1, query_heads=4, kv_heads=2,
                  capacity=64, head_dim=32, dtype=0, keep_first=4, keep_recent=8)
    return nat.HHCache(**{**fields, **over})


BAD_CACHES = [
    (dict(batch=-1), nat.PGR_ERR_INVALID), (dict(query_heads=3), nat.PGR_ERR_INVALID),
    (dict(query_heads=34), nat.PGR_ERR_UNSUPPORTED), (dict(head_dim=48), nat.PGR_ERR_UNSUPPORTED),
    (dict(dtype=2), nat.PGR_ERR_UNSUPPORTED), (dict(capacity=0), nat.PGR_ERR_INVALID),
    (dict(capacity=(1 << 26) + 1), nat.PGR_ERR_INVALID), (dict(keep_first=-1), nat.PGR_ERR_INVALID),
    (dict(keep_recent=0), nat.PGR_ERR_INVALID), (dict(keep_first=60, keep_recent=5), nat.PGR_ERR_INVALID),
    (dict(seen=0), nat.PGR_ERR_INVALID), (dict(keys=264), nat.PGR_ERR_INVALID),
    (dict(batch=65536), nat.PGR_ERR_INVALID),
]


@pytest.mark.parametrize("over,code", BAD_CACHES)
def test_c_entries_refuse_a_bad_cache(over, code):
    lib, c = nat.load(), _cache(**over)
    s = (ctypes.c_int64 * 3)(1, 1, 1)
    assert lib.pgr_hh_append(c, 16, s, 16, s, 16, s, 16, None, 0, None, 0, 0, 1.0, None) == code
    assert lib.pgr_hh_attend(c, 16, s, 16, 1.0, 0.0, 256, 1 << 30, None) == code
    assert lib.pgr_hh_load_prompt(c, 16, s, 16, s, 16, None, 4, 256, 1 << 30, None) == code
    assert lib.pgr_hh_attend_workspace_bytes(c) == 0 and lib.pgr_hh_load_prompt_workspace_bytes(c, 4) == 0


def test_c_entries_refuse_bad_arguments():
    lib, c = nat.load(), _cache()
    s = (ctypes.c_int64 * 3)(1, 1, 1)
    inv, cap = nat.PGR_ERR_INVALID, nat.PGR_ERR_CAPACITY
    assert lib.pgr_hh_append(None, 16, s, 16, s, 16, s, 16, None, 0, None, 0, 0, 1.0, None) == inv
    assert lib.pgr_hh_append(c, 16, s, None, s, 16, s, 16, None, 0, None, 0, 0, 1.0, None) == inv
    assert lib.pgr_hh_append(c, None, s, 16, s, 16, s, 16, None, 0, None, 0, 0, 1.0, None) == inv
    assert lib.pgr_hh_append(c, 16, s, 16, s, 16, s, 16, None, 0, None, 2, 0, 1.0, None) == inv  # no inv_freq
    assert lib.pgr_hh_append(c, 16, s, 16, s, 16, s, 16, None, 0, 16, 34, 0, 1.0, None) == inv   # past the head
    assert lib.pgr_hh_append(c, 16, s, 16, s, 16, s, 16, None, 0, 16, 3, 0, 1.0, None) == inv    # odd
    assert lib.pgr_hh_attend_workspace_bytes(c) == 0  # a short row needs none
    long = _cache(capacity=4096)
    need = lib.pgr_hh_attend_workspace_bytes(long)
    assert need > 0
    assert lib.pgr_hh_attend(long, 16, s, 16, 1.0, 0.0, 256, need - 1, None) == cap
    assert lib.pgr_hh_attend(long, 16, s, 16, 1.0, 0.0, None, need, None) == cap
    assert lib.pgr_hh_attend(c, 16, s, None, 1.0, 0.0, 256, need, None) == inv
    assert lib.pgr_hh_attend(c, 16, s, 16, 0.0, 0.0, 256, need, None) == inv
    assert lib.pgr_hh_attend(c, 16, s, 16, 1.0, float("nan"), 256, need, None) == inv
    need = lib.pgr_hh_load_prompt_workspace_bytes(c, 4)
    assert lib.pgr_hh_load_prompt_workspace_bytes(c, -1) == 0
    assert need >= 2 * 64 * 4
    assert lib.pgr_hh_load_prompt(c, 16, s, 16, s, 16, None, -1, 256, need, None) == inv
    assert lib.pgr_hh_load_prompt(c, 16, s, 16, s, None, None, 4, 256, need, None) == inv
    assert lib.pgr_hh_load_prompt(c, 16, s, 16, s, 16, None, 4, 256, need - 1, None) == cap
    bytes_of = lib.pgr_hh_prompt_weights_workspace_bytes
    assert bytes_of(1, 4, 2, 100, 10, 32) > 0
    for bad in ((1, 4, 2, 8388481, 1, 32), (1, 32, 2, 200000, 131071, 32), (300, 32, 8, 1000000, 1, 32),
                (1, 4, 2, 100, 101, 32), (1, 4, 2, 100, -1, 32), (1, 3, 2, 100, 10, 32), (1, 4, 2, 100, 10, 40),
                (1, 34, 2, 100, 10, 32)):
        assert bytes_of(*bad) == 0
    run = lib.pgr_hh_prompt_weights
    assert run(16, s, 16, s, None, 16, 1, 4, 2, 100, 101, 32, 0, 1.0, 0.0, 256, 1 << 30, None) == inv
    assert run(16, s, 16, s, None, 16, 1, 4, 2, 100, 0, 32, 0, 1.0, 0.0, 256, 1 << 30, None) == inv
    assert run(16, s, 16, s, None, 16, 1, 4, 2, 100, 10, 32, 2, 1.0, 0.0, 256, 1 << 30, None) == nat.PGR_ERR_UNSUPPORTED
    assert run(16, s, 16, s, None, 16, 1, 4, 2, 100, 10, 32, 0, -1.0, 0.0, 256, 1 << 30, None) == inv
    assert run(16, s, 16, s, None, 16, 1, 4, 2, 100, 10, 32, 0, 1.0, 0.0, 256, 16, None) == cap
    wide = (ctypes.c_int64 * 3)(1, 1 << 31, 1)
    assert run(16, wide, 16, s, None, 16, 1, 4, 2, 100, 10, 32, 0, 1.0, 0.0, 256, 1 << 30, None) == inv
    assert run(None, s, 16, s, None, 16, 1, 4, 2, 100, 10, 32, 0, 1.0, 0.0, 256, 1 << 30, None) == inv
    assert run(16, s, 16, s, None, 16, 1, 4, 2, 0, 0, 32, 0, 1.0, 0.0, None, 0, None) == 0  # nothing to do


def test_c_entries_refuse_operands_in_the_cache():
    """keys, values and weights at addresses of their own: 1 x 2 rows of 64 slots, 32 dims."""
    lib, inv = nat.load(), nat.PGR_ERR_INVALID
    c = _cache(keys=1 << 20, values=2 << 20, weights=3 << 20, order=4 << 20, lengths=5 << 20, seen=6 << 20)
    s = (ctypes.c_int64 * 3)(1, 1, 1)
    kv = 2 * 64 * 32 * 2
    for at in (1 << 20, (1 << 20) + kv - 2, (2 << 20) + 64, (3 << 20) + 4):
        assert lib.pgr_hh_append(c, 16, s, at, s, 16, s, None, None, 0, None, 0, 0, 1.0, None) == inv
        assert lib.pgr_hh_append(c, 16, s, 16, s, at, s, None, None, 0, None, 0, 0, 1.0, None) == inv
        assert lib.pgr_hh_load_prompt(c, at, s, 16, s, 16, None, 4, 256, 1 << 30, None) == inv
        assert lib.pgr_hh_load_prompt(c, 16, s, at, s, 16, None, 4, 256, 1 << 30, None) == inv
        assert lib.pgr_hh_load_prompt(c, 16, s, 16, s, at, None, 4, 256, 1 << 30, None) == inv
        assert lib.pgr_hh_attend(c, at, s, 16, 1.0, 0.0, None, 0, None) == inv
        assert "own buffers" in nat.last_error()


# The same cache: where each of its buffers begins and how many bytes it has.
BUFFERS = dict(keys=(1 << 20, 8192), values=(2 << 20, 8192), weights=(3 << 20, 512), order=(4 << 20, 512),
               lengths=(5 << 20, 8), seen=(6 << 20, 8))


@pytest.mark.parametrize("name", list(BUFFERS))
def test_c_entries_refuse_every_operand_in_every_buffer(name):
    """Operands that begin in a buffer, end in it, or reach it with one of their rows; the index operands too,
    which the workgroups of other rows read while a row's own workgroup changes the buffer."""
    lib, inv = nat.load(), nat.PGR_ERR_INVALID
    c = _cache(**{n: at for n, (at, _) in BUFFERS.items()})
    s, far = (ctypes.c_int64 * 3)(1, 1, 1), 1 << 30
    base, size = BUFFERS[name]

    def append(q=far, k=far, v=far, q_out=far, positions=None, inv_freq=None, long=0, strides=s):
        return lib.pgr_hh_append(c, q, strides, k, strides, v, strides, q_out, positions, long, inv_freq,
                                 32 if inv_freq else 0, 0, 1.0, None)

    def load(k=far, v=far, weights=far, lo=None, strides=s):
        return lib.pgr_hh_load_prompt(c, k, strides, v, strides, weights, lo, 4, 256, 1 << 30, None)

    def attend(q=far, out=far, strides=s):
        return lib.pgr_hh_attend(c, q, strides, out, 1.0, 0.0, None, 0, None)

    refused = []

    def refuse(rc):
        refused.append(rc == inv and "own buffers" in nat.last_error())

    for at in (base, base + size - 4, base - 2):  # (every operand has more than two bytes)
        refuse(append(k=at))
        refuse(append(v=at))
        refuse(append(q=at))
        refuse(append(q_out=at))
        refuse(append(positions=at))
        refuse(append(positions=at, long=1))
        refuse(append(inv_freq=at))
        refuse(load(k=at))
        refuse(load(v=at))
        refuse(load(weights=at))
        refuse(load(lo=at))
        refuse(attend(q=at))
        refuse(attend(out=at))
    # The second head's row, 4096 elements behind or before the first.
    for step in (4096, -4096):
        apart = (ctypes.c_int64 * 3)(1, step, 1)
        refuse(append(k=base - 2 * step, strides=apart))
        refuse(load(v=base - 2 * step, strides=apart))
        refuse(attend(q=base - 2 * step, strides=apart))
    assert all(refused), refused


def test_c_entries_take_operands_around_the_buffers():
    """Rows whose gaps span the cache, operands that end where a buffer begins: past the checks of the operands,
    so another error than theirs (no device here), or none."""
    if torch.cuda.is_available():
        pytest.skip("addresses without memory behind them: for hosts without a GPU")
    lib, s = nat.load(), (ctypes.c_int64 * 3)(1, 1, 1)
    c = _cache(**{n: at for n, (at, _) in BUFFERS.items()})
    far = 1 << 30
    spans = (ctypes.c_int64 * 3)(1, 8 << 20, 1)  # rows at 64 KB and, 16 MB on, past every buffer
    for rc in (lib.pgr_hh_append(c, far, s, 1 << 16, spans, far, s, None, None, 0, None, 0, 0, 1.0, None),
               lib.pgr_hh_append(c, far, s, far, s, far, s, None, (6 << 20) - 8, 1, None, 0, 0, 1.0, None),
               lib.pgr_hh_load_prompt(c, 1 << 16, spans, far, s, far, (6 << 20) + 8, 4, 256, 1 << 30, None),
               lib.pgr_hh_attend(c, far, s, (1 << 20) - 4 * 32 * 2, 1.0, 0.0, None, 0, None)):
        assert rc not in (0, nat.PGR_ERR_INVALID)


def test_c_entries_refuse_outputs_over_their_inputs():
    """append's threads read the partner of the element they write, and other heads' workgroups the rest; attend
    in place (the same contiguous layout) reads before it writes."""
    if torch.cuda.is_available():
        pytest.skip("addresses without memory behind them: for hosts without a GPU")
    lib, inv = nat.load(), nat.PGR_ERR_INVALID
    c = _cache(**{n: at for n, (at, _) in BUFFERS.items()})
    s, dense = (ctypes.c_int64 * 3)(1, 1, 1), (ctypes.c_int64 * 2)(128, 32)  # 4 query heads of 32
    far, out = 1 << 30, 1 << 29

    def append(q=far, k=far, v=far, positions=None, inv_freq=None, strides=dense):
        return lib.pgr_hh_append(c, q, strides, k, s, v, s, out, positions, 0, inv_freq, 32 if inv_freq else 0, 0, 1.0, None)

    for at in (out, out + 254, out - 2):
        for rc in (append(q=at), append(k=at), append(v=at), append(positions=at), append(inv_freq=at, q=far)):
            assert rc == inv and "overlap" in nat.last_error(), at
    assert append(q=out - 256) not in (0, inv) and append(q=out + 256) not in (0, inv)
    attend = lambda q, strides: lib.pgr_hh_attend(c, q, strides, out, 1.0, 0.0, None, 0, None)
    for q, strides in ((out + 64, dense), (out - 64, dense), (out, (ctypes.c_int64 * 2)(128, 64))):
        assert attend(q, strides) == inv and "overlap" in nat.last_error()
    assert attend(out, dense) not in (0, inv) and attend(out + 256, dense) not in (0, inv)


def test_prompt_weights_refuse_an_output_over_the_inputs():
    """Workgroups write their keys' weights while others still read q, k and lo."""
    if torch.cuda.is_available():
        pytest.skip("addresses without memory behind them: for hosts without a GPU")
    lib, inv = nat.load(), nat.PGR_ERR_INVALID
    s, far, out = (ctypes.c_int64 * 3)(1, 1, 1), 1 << 30, 1 << 29  # out: 2 heads of 100 floats

    def run(q=far, k=far, lo=None):
        return lib.pgr_hh_prompt_weights(q, s, k, s, lo, out, 1, 4, 2, 100, 10, 32, 0, 1.0, 0.0, 256, 1 << 30, None)

    for at in (out, out + 798, out - 2):
        assert run(q=at) == inv and "overlap" in nat.last_error()
        assert run(k=at) == inv and "overlap" in nat.last_error()
        assert run(lo=at) == inv and "overlap" in nat.last_error()
    assert run(q=out + 800, k=out - 1024, lo=out - 4) not in (0, inv)


def test_python_refusals_need_no_gpu():
    def make(**over):
        a = dict(batch=1, num_query_heads=4, num_kv_heads=2, capacity=64, head_dim=32, dtype=torch.float16, device="cuda")
        return HeavyHitterCache(**{**a, **over})

    with pytest.raises(ValueError, match="CUDA"):
        make(device="cpu")
    with pytest.raises(NotImplementedError, match="float32"):
        make(dtype=torch.float32)
    with pytest.raises(NotImplementedError, match="head_dim"):
        make(head_dim=80)
    with pytest.raises(NotImplementedError, match="16"):
        make(num_query_heads=34)
    with pytest.raises(ValueError, match="multiple"):
        make(num_query_heads=5)
    with pytest.raises(ValueError, match="keep_recent"):
        make(keep_recent=0)
    with pytest.raises(ValueError, match="capacity"):
        make(keep_first=40, keep_recent=25)
    with pytest.raises(ValueError, match="dimension"):
        make(capacity=0)
    q, k = torch.zeros(1, 4, 8, 32).half(), torch.zeros(1, 2, 16, 32).half()
    with pytest.raises(ValueError, match="CUDA"):
        prompt_attention_weights(q, k)
    with pytest.raises(NotImplementedError, match="float32"):
        prompt_attention_weights(q.float(), k.float())
    with pytest.raises(TypeError, match="one dtype"):
        prompt_attention_weights(q, k.bfloat16())
    with pytest.raises(ValueError, match="does not match"):
        prompt_attention_weights(q, k[..., :16])
    with pytest.raises(RuntimeError, match="gradient"):
        prompt_attention_weights(q, k.requires_grad_())


# ---- the oracle itself ---------------------------------------------------------------------------
def test_oracle_keeps_what_the_rule_says():
    w = np.array([0.0, 5.0, 1.0, 3.0, 3.0, np.nan, 0.5, 3.0, 9.0, 0.1])
    assert O.kept_columns(w, 0, 10, 1, 1).tolist() == list(range(10))
    assert O.kept_columns(w, 4, 6, 1, 1).tolist() == [4, 5, 6, 7, 8, 9]
    # first 1, last 2; then NaN, 5, and the first of the threes
    assert O.kept_columns(w, 0, 6, 1, 2).tolist() == [0, 1, 3, 5, 8, 9]
    assert O.kept_columns(w, 0, 7, 1, 2).tolist() == [0, 1, 3, 4, 5, 8, 9]
    assert O.kept_columns(w, 0, 3, 1, 2).tolist() == [0, 8, 9]


def test_oracle_slot_of_an_append():
    w = np.array([0.0, 2.0, -0.0, np.nan, 2.0, 0.0])
    order = np.array([0, 1, 7, 3, 9, 5])
    assert O.append_slot(4, 10, w, order, 6, 1, 2) == 4       # room left
    assert O.append_slot(6, 10, w, order, 6, 1, 2) == 2       # order 0 and 9 stay; -0 equals 0: the lower slot
    assert O.append_slot(6, 10, w, order, 6, 1, 4) == 5       # 7 and 9 are recent
    assert O.append_slot(6, 10, w, order, 6, 0, 1) == 0


def test_oracle_prompt_weights_sum_to_the_queries():
    rng = np.random.default_rng(0)
    q, k = rng.standard_normal((3, 5, 16)), rng.standard_normal((9, 16))
    w, _ = O.prompt_weights(q, k, 2, 0.25, 0.0)
    assert abs(w.sum() - 15) < 1e-12 and not w[:2].any()
    w, _ = O.prompt_weights(q, k, 6, 0.25, 30.0)  # queries at columns 4, 5 are padding
    assert abs(w.sum() - 9) < 1e-12 and not w[:6].any()
    w, _ = O.prompt_weights(q, k, 9, 0.25, 0.0)
    assert not w.any()
