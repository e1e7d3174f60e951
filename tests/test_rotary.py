"""Rotary positions: the frequencies against their formulas, the kernel against 64 bits."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import _pgr_native as nat
from oracle import bounded_cache as O
from pager_hf.rotary import rotary_embedding, rotary_frequencies

gpu = pytest.mark.gpu
STEP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}


def _np(t):
    return t.detach().cpu().double().numpy()


# ---- frequencies (CPU) ---------------------------------------------------------------------------
def test_default_frequencies():
    inv, factor = rotary_frequencies(64, 10000.0)
    want = 10000.0 ** (-np.arange(0, 64, 2) / 64)
    np.testing.assert_allclose(inv.double().numpy(), want, rtol=2.0**-23)
    assert factor == 1.0 and inv.dtype == torch.float32


def test_scaled_frequencies_follow_their_formulas():
    base = 10000.0 ** (-np.arange(0, 128, 2) / 128)
    inv, _ = rotary_frequencies(128, scaling={"rope_type": "linear", "factor": 4.0})
    np.testing.assert_allclose(inv.double().numpy(), base / 4, rtol=2.0**-23)
    inv, _ = rotary_frequencies(128, scaling={"type": "ntk", "factor": 8.0})
    # The fastest pair stays, the slowest is stretched by the factor.
    assert inv[0] == 1.0
    np.testing.assert_allclose(inv[-1].double().item(), base[-1] / 8, rtol=1e-6)
    cfg = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
           "original_max_position_embeddings": 8192}
    inv, _ = rotary_frequencies(128, 500000.0, cfg)
    freq = 500000.0 ** (-np.arange(0, 128, 2) / 128)
    for f, got in zip(freq, inv.double().numpy()):
        wavelength = 2 * math.pi / f
        if wavelength < 8192 / 4:
            want = f
        elif wavelength > 8192:
            want = f / 8
        else:
            smooth = (8192 / wavelength - 1) / 3
            want = (1 - smooth) * f / 8 + smooth * f
        assert abs(got - want) <= 2.0**-23 * want
    cfg = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    inv, factor = rotary_frequencies(128, 1000000.0, cfg)
    freq = 1000000.0 ** (-np.arange(0, 128, 2) / 128)
    turns = 32768 * freq / (2 * math.pi)
    got = inv.double().numpy()
    np.testing.assert_allclose(got[turns > 64], freq[turns > 64], rtol=2.0**-23)  # whole ramp steps past the borders
    np.testing.assert_allclose(got[turns < 0.5], freq[turns < 0.5] / 4, rtol=2.0**-23)
    assert np.all(got <= freq * (1 + 2.0**-23)) and np.all(got >= freq / 4 * (1 - 2.0**-23))
    assert abs(factor - (0.1 * math.log(4.0) + 1)) < 1e-15


def test_frequencies_match_the_models_own():
    rope = pytest.importorskip("transformers.modeling_rope_utils")
    from transformers import LlamaConfig

    settings = [
        {"rope_type": "linear", "factor": 4.0},
        {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 2048},
        {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
         "original_max_position_embeddings": 2048},
    ]
    for s in settings:
        cfg = LlamaConfig(hidden_size=512, num_attention_heads=8, max_position_embeddings=8192,
                          rope_parameters=dict(s, rope_theta=10000.0))
        want, factor = rope.ROPE_INIT_FUNCTIONS[s["rope_type"]](cfg, torch.device("cpu"))
        inv, got = rotary_frequencies(64, 10000.0, s)
        # (the model's are float32 throughout: base, power, quotient and blend, a few roundings each)
        np.testing.assert_allclose(inv.double().numpy(), want.double().numpy(), rtol=2.0**-19)
        assert abs(factor - got) < 1e-12


def test_base_comes_from_the_settings():
    """A config's rope_parameters hold the base as rope_theta."""
    llama3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
              "original_max_position_embeddings": 8192}
    yarn = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    for s in ({"rope_type": "default"}, {"rope_type": "linear", "factor": 2.0}, {"rope_type": "ntk", "factor": 2.0}, llama3,
              yarn):
        want = rotary_frequencies(128, 500000.0, s)
        for got in (rotary_frequencies(128, scaling=dict(s, rope_theta=500000)),
                    rotary_frequencies(128, 500000.0, dict(s, rope_theta=500000.0))):
            assert torch.equal(got[0], want[0]) and got[1] == want[1]
        assert torch.equal(rotary_frequencies(128, scaling=s)[0], rotary_frequencies(128, 10000.0, s)[0])
        with pytest.raises(ValueError, match="rope_theta"):
            rotary_frequencies(128, 10000.0, dict(s, rope_theta=500000.0))
    with pytest.raises(ValueError, match="rope_theta"):
        rotary_frequencies(128, scaling={"rope_type": "default", "rope_theta": -1.0})


def test_base_of_a_models_own_settings():
    rope = pytest.importorskip("transformers.modeling_rope_utils")
    from transformers import LlamaConfig

    cfg = LlamaConfig(hidden_size=512, num_attention_heads=8, max_position_embeddings=8192,
                      rope_parameters={"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                                       "original_max_position_embeddings": 2048, "rope_theta": 500000.0})
    want, factor = rope.ROPE_INIT_FUNCTIONS["llama3"](cfg, torch.device("cpu"))
    inv, got = rotary_frequencies(64, scaling=cfg.rope_parameters)
    # (the model's are float32 throughout: base, power, quotient and blend, a few roundings each)
    np.testing.assert_allclose(inv.double().numpy(), want.double().numpy(), rtol=2.0**-19)
    assert factor == got == 1.0


@pytest.mark.parametrize("mscale,all_dim", [(1.0, 1.0), (0.707, 0.707), (1.0, 0.8), (0.5, 1.25)])
@pytest.mark.parametrize("factor", [40.0, 4.0, 1.0])
def test_yarn_factor_of_two_scales(mscale, all_dim, factor):
    """cos and sin are scaled by (0.1 mscale ln(factor) + 1) / (0.1 mscale_all_dim ln(factor) + 1)."""
    cfg = {"rope_type": "yarn", "factor": factor, "original_max_position_embeddings": 4096, "mscale": mscale,
           "mscale_all_dim": all_dim}
    inv, got = rotary_frequencies(64, 10000.0, cfg)
    want = (0.1 * mscale * math.log(factor) + 1) / (0.1 * all_dim * math.log(factor) + 1)
    assert abs(got - want) < 1e-12
    assert torch.equal(inv, rotary_frequencies(64, 10000.0, {k: v for k, v in cfg.items() if "mscale" not in k})[0])
    assert rotary_frequencies(64, 10000.0, dict(cfg, attention_factor=1.5))[1] == 1.5
    rope = pytest.importorskip("transformers.modeling_rope_utils")
    from transformers import LlamaConfig

    model = LlamaConfig(hidden_size=512, num_attention_heads=8, max_position_embeddings=8192,
                        rope_parameters=dict(cfg, rope_theta=10000.0))
    assert abs(rope.ROPE_INIT_FUNCTIONS["yarn"](model, torch.device("cpu"))[1] - got) < 1e-12


def test_yarn_scale_refusals():
    cfg = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}
    for name in ("mscale", "mscale_all_dim"):
        with pytest.raises(ValueError, match="mscale"):
            rotary_frequencies(64, scaling=dict(cfg, **{name: 0.7}))
        with pytest.raises(ValueError, match="positive"):
            rotary_frequencies(64, scaling=dict({**cfg, "mscale": 1.0, "mscale_all_dim": 1.0}, **{name: -1.0}))


def test_settings_that_are_not_read_are_refused():
    """An entry that would change a model's angles and that no supported rope type reads."""
    for s in ({"rope_type": "default", "mrope_section": [16, 24, 24]},
              {"rope_type": "linear", "factor": 2.0, "short_factor": [1.0]},
              {"full_attention": {"rope_type": "default", "rope_theta": 1e6}, "sliding_attention": {"rope_type": "default"}}):
        with pytest.raises(NotImplementedError, match="mrope_section|short_factor|full_attention"):
            rotary_frequencies(128, scaling=s)
    # rotary_dim is the part that turns: whether the share is in it already cannot be seen here.
    with pytest.raises(NotImplementedError, match="partial_rotary_factor"):
        rotary_frequencies(128, scaling={"rope_type": "default", "partial_rotary_factor": 0.5})
    # Entries that change nothing: absent ones, a whole share, what another rope type reads.
    want = rotary_frequencies(128, 10000.0)[0]
    for s in ({"rope_type": "default", "partial_rotary_factor": 1.0, "rope_theta": 10000.0},
              {"rope_type": "default", "mrope_section": None, "factor": 4.0, "original_max_position_embeddings": 4096}):
        assert torch.equal(rotary_frequencies(128, scaling=s)[0], want)


def test_frequency_refusals():
    with pytest.raises(ValueError, match="even"):
        rotary_frequencies(63)
    with pytest.raises(ValueError, match="even"):
        rotary_frequencies(0)
    with pytest.raises(ValueError, match="base"):
        rotary_frequencies(64, -1.0)
    with pytest.raises(NotImplementedError, match="longrope"):
        rotary_frequencies(64, scaling={"rope_type": "longrope"})
    with pytest.raises(ValueError, match="factor"):
        rotary_frequencies(64, scaling={"rope_type": "linear"})
    with pytest.raises(ValueError, match="factor"):
        rotary_frequencies(64, scaling={"rope_type": "linear", "factor": 0.0})
    with pytest.raises(ValueError, match="4 or more"):
        rotary_frequencies(2, scaling={"rope_type": "ntk", "factor": 2.0})


def test_c_entry_refuses_before_any_launch():
    lib = nat.load()

    def call(q_heads=2, k_heads=1, rotary=8, batch=1, tokens=4, d=16, dtype=0, factor=1.0):
        return lib.pgr_rotary(None, None, None, q_heads, None, None, None, k_heads, None, 0, None, None, rotary, batch,
                              tokens, d, dtype, 0, factor, 0, None)

    assert call(rotary=0, batch=0) == 0 and call(rotary=0, tokens=0) == 0 and call(rotary=0, q_heads=0, k_heads=0) == 0
    for bad in (dict(q_heads=-1), dict(tokens=-1), dict(d=0), dict(dtype=3), dict(), dict(rotary=0),
                dict(rotary=0, factor=float("nan")), dict(rotary=0, batch=1 << 31), dict(rotary=0, q_heads=70000)):
        assert call(**bad) == nat.PGR_ERR_INVALID, bad


def test_c_entry_refuses_a_grid_that_wraps():
    """A grid dimension of 2^32 threads runs none without an error: the last sizes below it round up to that."""
    lib = nat.load()

    def call(tokens, d):
        rc = lib.pgr_rotary(None, None, None, 1, None, None, None, 0, None, 0, None, None, 0, 1, tokens, d, 0, 0, 1.0, 0, None)
        assert rc == nat.PGR_ERR_INVALID
        return "limits" in nat.last_error()

    for d in (4, 12, 65, 100, 4097):
        most = ((1 << 32) - 256) // d
        assert call(most + 1, d), d
        assert not call(most, d), d  # (refused for its null pointers)


def test_python_refusals_need_no_gpu():
    q, k = torch.zeros(1, 2, 4, 16), torch.zeros(1, 1, 4, 16)
    pos, inv = torch.zeros(1, 4, dtype=torch.int64), torch.ones(8)
    with pytest.raises(ValueError, match="CUDA"):
        rotary_embedding(q, k, pos, inv)
    with pytest.raises(NotImplementedError, match="float64"):
        rotary_embedding(q.double(), k.double(), pos, inv)
    with pytest.raises(TypeError, match="one dtype"):
        rotary_embedding(q, k.half(), pos, inv)
    with pytest.raises(ValueError, match="does not match"):
        rotary_embedding(q, k[:, :, :3], pos, inv)
    with pytest.raises(ValueError, match="must be"):
        rotary_embedding(q[0, 0], None, pos, inv)
    with pytest.raises(RuntimeError, match="gradient"):
        rotary_embedding(q.requires_grad_(), k, pos, inv)


def test_forward_tangents_are_refused():
    from torch.autograd import forward_ad

    from pager_hf.heavy_hitter_cache import prompt_attention_weights

    q, k = torch.zeros(1, 2, 4, 16), torch.zeros(1, 1, 4, 16)
    pos, inv = torch.zeros(1, 4, dtype=torch.int64), torch.ones(8)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for mode in (torch.enable_grad, torch.no_grad):
            with mode():
                for bad in (lambda: rotary_embedding(dual(q), k, pos, inv), lambda: rotary_embedding(q, dual(k), pos, inv),
                            lambda: rotary_embedding(q, k, pos, dual(inv)),
                            lambda: rotary_embedding(dual(q[:, :, 0]), None, pos[:, 0], inv),
                            lambda: prompt_attention_weights(dual(q.half()), k.half())):
                    with pytest.raises(RuntimeError, match="gradient"):
                        bad()
        with pytest.raises(ValueError, match="CUDA"):
            rotary_embedding(q, k, pos, inv)


# ---- kernel --------------------------------------------------------------------------------------
def _check(got, x, ref, inv_freq, factor, interleaved):
    """Half a step of the output type, and of the float32 steps before it: cos and sin within 2 steps
    (4 halves), their scale, the two products and the sum."""
    half = len(inv_freq)
    size = np.abs(x).copy()
    if interleaved:
        pair = size[..., 0:2 * half:2] + size[..., 1:2 * half:2]
        size[..., 0:2 * half:2] = size[..., 1:2 * half:2] = pair
    else:
        size[..., half:2 * half] = size[..., :half] = size[..., :half] + size[..., half:2 * half]
    step = STEP[got.dtype]
    tol = step * np.abs(ref) + 8 * O.U32 * abs(factor) * size
    tol[..., 2 * half:] = 0.0
    if got.dtype == torch.float16:
        tol[..., :2 * half] += 2.0**-25  # half of the smallest subnormal
    err = np.abs(_np(got) - ref)
    assert np.all(err <= tol), float((err - tol).max())


CASES = [
    # batch, q heads, k heads, tokens, head dim, rotary dims
    (1, 14, 2, 1, 64, 64),
    (3, 4, 2, 5, 128, 64),
    (2, 3, 1, 17, 80, 32),
    (1, 2, 2, 3, 10, 6),
    (2, 1, 1, 7, 2, 2),
    (1, 8, 1, 129, 256, 256),
    (5, 32, 8, 33, 128, 128),
    (1, 1, 1, 1, 65, 2),
]


@gpu
@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_against_64_bits(case, dtype, interleaved):
    b, hq, hk, t, d, r = case
    g = torch.Generator().manual_seed(hash(case) % 1000)
    # Projection layout: [B, T, H, D] seen as [B, H, T, D].
    q = torch.randn(b, t, hq, d, generator=g).to(dtype).cuda().transpose(1, 2)
    k = torch.randn(b, t, hk, d, generator=g).to(dtype).cuda().transpose(1, 2)
    inv, _ = rotary_frequencies(r, device="cuda")
    pos = torch.randint(0, 1 << 20, (b, t), generator=g)
    pos[0, 0] = 0
    factor = 1.25
    for inverse in (False, True):
        for p in (pos, pos.int()):
            qo, ko = rotary_embedding(q, k, p.cuda(), inv, interleaved=interleaved, factor=factor, inverse=inverse)
            assert qo.is_contiguous() and qo.shape == q.shape and ko.shape == k.shape
            for x, y in ((q, qo), (k, ko)):
                ref = O.rotate(_np(x), pos.numpy()[:, None], _np(inv), interleaved=interleaved, factor=factor,
                               inverse=inverse)
                _check(y, _np(x), ref, _np(inv), factor, interleaved)


@gpu
def test_forms_of_the_arguments():
    g = torch.Generator().manual_seed(5)
    q = torch.randn(2, 4, 6, 64, generator=g).half().cuda()
    k = torch.randn(2, 2, 6, 64, generator=g).half().cuda()
    inv, _ = rotary_frequencies(64, device="cuda")
    pos = torch.arange(6, device="cuda").unsqueeze(0)
    a, b = rotary_embedding(q, k, pos, inv)
    # One row of positions for all, its expansion, strided positions, no k, a view at an odd offset.
    a2, b2 = rotary_embedding(q, k, pos.expand(2, 6), inv)
    a3, none = rotary_embedding(q, None, torch.stack([pos[0]] * 2, dim=-1).repeat(2, 1, 1)[..., 1], inv)
    flat = torch.cat([q.flatten()[:1], q.flatten()])[1:].view(q.shape)
    a4, _ = rotary_embedding(flat, None, pos, inv)
    a5, _ = rotary_embedding(q.permute(3, 1, 2, 0).contiguous().permute(3, 1, 2, 0), None, pos, inv)
    assert none is None and torch.equal(b, b2)
    for x in (a2, a3, a4, a5):
        assert torch.equal(a, x)
    # One token per row.
    s, t = rotary_embedding(q[:, :, 3], k[:, :, 3], pos[0, 3].repeat(2), inv)
    assert torch.equal(s, a[:, :, 3]) and torch.equal(t, b[:, :, 3])
    # Nothing to do.
    e, f = rotary_embedding(q[:, :, :0], k[:, :, :0], pos[:, :0], inv)
    assert e.shape == (2, 4, 0, 64) and f.shape == (2, 2, 0, 64)
    for bad in (lambda: rotary_embedding(q, k, pos[:, :5], inv), lambda: rotary_embedding(q, k, pos.float(), inv),
                lambda: rotary_embedding(q, k, pos, inv.half()), lambda: rotary_embedding(q, k, pos, inv.repeat(2)),
                lambda: rotary_embedding(q, k, pos.cpu(), inv), lambda: rotary_embedding(q, k, pos, inv.cpu()),
                lambda: rotary_embedding(q, k, pos, inv, factor=float("inf"))):
        with pytest.raises((ValueError, TypeError)):
            bad()


@gpu
def test_inverse_is_the_gradient():
    """The map is linear: <g, R x> = <R' g, x>, and R' agrees with differences of <g, R x>."""
    gen = torch.Generator().manual_seed(9)
    x = torch.randn(1, 2, 5, 32, generator=gen).cuda()
    g = torch.randn(1, 2, 5, 32, generator=gen).cuda()
    inv, _ = rotary_frequencies(16, device="cuda")
    pos = torch.tensor([[0, 1, 77, 4096, 131071]], device="cuda")
    for interleaved in (False, True):
        y, _ = rotary_embedding(x, None, pos, inv, interleaved=interleaved, factor=1.5)
        back, _ = rotary_embedding(g, None, pos, inv, interleaved=interleaved, factor=1.5, inverse=True)
        lhs, rhs = (g.double() * y.double()).sum(), (back.double() * x.double()).sum()
        # Each turned element is off by at most 8 halves of a step of 1.5 times its pair's size.
        size = 1.5 * 2 * (g.double().abs().sum() * x.abs().max() + x.double().abs().sum() * g.abs().max())
        assert abs(lhs - rhs) <= 8 * O.U32 * size
        for at in ((0, 0, 2, 3), (0, 1, 4, 9), (0, 1, 3, 20)):
            e = torch.zeros_like(x)
            e[at] = 1.0
            d, _ = rotary_embedding(e, None, pos, inv, interleaved=interleaved, factor=1.5)
            assert abs((g.double() * d.double()).sum() - back[at].double()) <= 16 * O.U32 * g[0, at[1], at[2]].abs().sum()


@gpu
def test_replays_and_other_streams():
    g = torch.Generator().manual_seed(2)
    q = torch.randn(3, 4, 9, 128, generator=g).bfloat16().cuda()
    k = torch.randn(3, 2, 9, 128, generator=g).bfloat16().cuda()
    inv, _ = rotary_frequencies(128, device="cuda")
    pos = torch.arange(9, device="cuda").unsqueeze(0)
    rotary_embedding(q, k, pos, inv)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo, ko = rotary_embedding(q, k, pos, inv)
    for n in range(3):
        q.copy_(torch.randn(q.shape, generator=g))
        pos.add_(n * 1000)
        graph.replay()
        a, b = rotary_embedding(q, k, pos, inv)
        assert torch.equal(a, qo) and torch.equal(b, ko)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c, _ = rotary_embedding(q, k, pos, inv)
    side.synchronize()
    assert torch.equal(c, a)
