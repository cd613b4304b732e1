"""What the sequence operators promise beside their values, as far as it shows without a GPU: the C entry points check before they launch, the Python ones look at the device last."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from genefaceplusplus_amd import _lib
from genefaceplusplus_amd._lib import GfppError
from genefaceplusplus_amd.radnerfs import RotaryEncoder, WindowCache, layer_norm, rotary_embed, sequence, window_attention, window_attention_step

# ---- the C entry points: every bad call returns its code before a launch (the pointers are never followed) ------------------------------------------------------
P, EINVAL = 4096, -1


def strides(n, value=8):
    return (ctypes.c_int64 * n)(*[value] * n)


def attention_forward(B, Tq, Tk, Hq, Hk, D=8):
    return _lib.lib().gfpp_window_attn_forward(P, P, P, P, None, None, strides(12), B, Tq, Tk, Hq, Hk, D, 3, 0, 0, 0, None, 1.0, 0, None)


def attention_backward(B, Tq, Tk, Hq, Hk, D=8, left=3, sinks=0):
    return _lib.lib().gfpp_window_attn_backward(P, P, P, P, None, P, P, P, P, P, P, strides(24), B, Tq, Tk, Hq, Hk, D, left, 0, sinks, 0, None, 1.0, 0, None)


def step(B, Hq, Hk, slots, D=8, scratch=P):
    return _lib.lib().gfpp_window_attn_step(P, P, P, P, P, P, 0, P, strides(14), B, Hq, Hk, D, slots, 0, 1.0, 0, scratch, None)


def rotary(B, T, heads, D, sections):
    return _lib.lib().gfpp_rotary(P, strides(3), heads, P, None, None, 0, None, P, 0, 0, P, (ctypes.c_uint32 * len(sections))(*sections), len(sections), B, T, D, 0, 0, 0, None)


def test_launches_beyond_a_grid_are_refused():
    """A launch of 2^32 threads along an axis or more would wrap and leave outputs unwritten: it is an error."""
    most = 2 ** 24                       # workgroups of 256 threads
    for call in (lambda: attention_forward(2 ** 20, 8, 8, 16, 1), lambda: attention_forward(1, 2 ** 29, 8, 4, 4), lambda: attention_forward(2 ** 29, 2 ** 29, 1, 2 ** 29, 1),
                 lambda: attention_backward(2 ** 20, 8, 8, 16, 1), lambda: attention_backward(2, 4, 2 ** 29, 1, 1), lambda: attention_backward(1, 2, 64, most, most),
                 lambda: rotary(most, 1, 1, 1024, (512,)), lambda: rotary(2 ** 31, 2 ** 31, 1, 2, (1,)),
                 lambda: step(most, 1, 1, 100), lambda: step(2 ** 20, 16, 16, 100), lambda: step(2 ** 29, 2 ** 29, 2 ** 29, 1), lambda: step(2 ** 19, 64, 1, 1536)):
        assert call() == EINVAL and b"grid_fits" in _lib.lib().gfpp_last_error()


def test_scratch_of_the_backward_pass_is_bounded():
    """Beside one float per query and head, the sinks' partial sums: 4 096 slices of 64 keys' dk and dv at most, however many sinks, heads and queries there are."""
    floats = _lib.lib().gfpp_window_attn_backward_scratch_floats
    for B, T, H, D, left, sinks in ((1, 13000, 8, 128, 128, 1000), (1, 500000, 8, 128, 64, 400000), (1, 500000, 1, 128, 0, 500000), (64, 4096, 8, 64, 127, 4), (1, 300, 65540, 2, 40, 3),
                                    (2000, 1000, 32, 128, 10, 1), (1, 100000, 1, 64, 100, 64)):
        partial = floats(B, T, T, H, H, D, left, 0, sinks, 0, 0) - B * H * T
        assert 0 <= partial <= 4096 * 2 * 64 * D, (B, T, H, partial)
        tiles = -(-sinks // 64) * B * H
        assert partial % (tiles * 2 * 64 * D) == 0 and (partial > 0) == (tiles <= 2048)


# ---- the Python side ---------------------------------------------------------------------------------------------------------------------------------------
def test_a_cache_moves_the_running_streams_alone(monkeypatch):
    """The position of a stream that rests (negative) stays; the step itself is stubbed out here."""
    monkeypatch.setattr(sequence, "window_attention_step", lambda q, *rest: q)
    cache = WindowCache(4, 1, 8, 4, 1, dtype=torch.float32, device="cpu")
    kept = cache.positions
    cache.positions.copy_(torch.tensor([-1, 5, 0, -2 ** 31]))
    x = torch.zeros(4, 1, 8)
    for t in range(1, 4):
        cache.step(x, x, x)
        assert cache.positions.tolist() == [-1, 5 + t, t, -2 ** 31] and cache.positions.dtype == torch.int32
    assert cache.positions is kept


def test_fill_moves_and_casts_nothing():
    """Keys, values or lengths on another device, lengths that are no whole numbers."""
    x, here = torch.zeros(2, 3, 1, 8), WindowCache(2, 1, 8, 4, 1, dtype=torch.float32, device="cpu")
    away = WindowCache(2, 1, 8, 4, 1, dtype=torch.float32, device="meta")
    for cache, k, v in ((away, x, x), (here, x, x.to("meta")), (here, x.to("meta"), x)):
        with pytest.raises(GfppError, match="k, v must be on"):
            cache.fill(k, v)
    for lengths in (torch.tensor([1.5, 2.0]), torch.tensor([True, False]), torch.tensor([1, 2], device="meta"), torch.tensor([1, 2], dtype=torch.int16)):
        with pytest.raises(GfppError, match="lengths must be"):
            here.fill(x, x, lengths)
    for lengths in (torch.tensor([1, 9]), torch.tensor([1, 3], dtype=torch.int32)):
        here.fill(x, x, lengths)
        assert here.positions.tolist() == [1, 3]


def sequence_calls():
    """One call of every operator without fault (but for the device), and the tensors of floating point that it takes, by argument."""
    z = lambda *shape: torch.zeros(*shape)  # noqa: E731
    x, q, t = z(3, 8), z(2, 5, 4, 8), z(2, 4, 8)
    return [(layer_norm, dict(x=x, weight=z(8), bias=z(8)), ("x", "weight", "bias")),
            (rotary_embed, dict(x=q, positions=z(5, 1), frequencies=z(4).double(), sections=(4,)), ("x", "positions", "frequencies")),
            (lambda k, **how: rotary_embed((q, k), **how), dict(k=z(2, 5, 1, 8), positions=z(5, 1), frequencies=z(4).double(), sections=(4,)), ("k",)),
            (window_attention, dict(q=q, k=q, v=q), ("q", "k", "v")),
            (window_attention_step, dict(q=t, k=t, v=t, cache_k=z(2, 6, 4, 8), cache_v=z(2, 6, 4, 8), positions=torch.zeros(2, dtype=torch.int32)), ("q", "k", "v", "cache_k", "cache_v"))]


def test_tangents_are_refused():
    """A dual tensor does not ask for a gradient: without a check its tangent would be dropped in silence."""
    for call, args, names in sequence_calls():
        with pytest.raises(GfppError, match="must be on the GPU"):
            call(**args)
        for name in names:
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
                assert not dual.requires_grad
                with pytest.raises(GfppError, match="forward mode"):
                    call(**{**args, name: dual})
                with torch.no_grad(), pytest.raises(GfppError, match="forward mode"):
                    call(**{**args, name: dual})
        with pytest.raises(GfppError, match="must be on the GPU"):
            call(**args)


def test_tracing_is_refused():
    """A tracer would record the outputs' allocation alone, and replay that."""
    for call, args, names in sequence_calls():
        def of(t):
            out = call(**{**args, names[0]: t})
            return out if isinstance(out, torch.Tensor) else out[0]
        with pytest.raises(GfppError, match="traced"):
            torch.jit.trace(of, (args[names[0]],), check_trace=False)
        with pytest.raises(GfppError, match="traced"):
            make_fx(of)(args[names[0]])
        with pytest.raises(GfppError, match="must be on the GPU"):
            call(**args)


def test_encoder_keeps_ordinary_frequencies(monkeypatch):
    """Whatever mode the encoder is made or first called in, its frequencies can be kept for a backward pass; a move takes them along, a change of type leaves them as they are."""
    meta = torch.device("meta")
    with torch.inference_mode():
        encoder = RotaryEncoder(16, (3, 5))
        encoder.frequencies(meta)
    for device in (meta, torch.device("cpu")):
        kept = encoder.frequencies(device)
        assert not kept.is_inference() and kept.dtype == torch.float64 and kept.shape == (8,) and kept.device == device
        assert encoder.frequencies(device) is kept
    with torch.device("meta"):
        assert torch.equal(RotaryEncoder(16, (3, 5)).frequencies(torch.device("cpu")), encoder.frequencies(torch.device("cpu")))
    moved = RotaryEncoder(16, (8,)).to("meta").half()
    assert moved._on[meta].dtype == torch.float64
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(GfppError, match="captured"):
        RotaryEncoder(16, (8,)).frequencies(torch.device("cuda", 0))
    assert moved.frequencies(meta) is moved._on[meta]
