"""Sequence operators of the conditioning stage: layer norm, attention with a sliding window and visible first tokens, and its single-token step over a rolling cache.

The reference smooths its conditioning over windows of 1 .. 16 frames (AudioNet / AudioAttNet, modules/radnerfs/cond_encoder.py:98-180).  These are the operators of
a conditioning network over whole clips (thousands of frames, forward and backward) and over live streams (one token at a time); the rotary positions that go with
them are in encoders.py.  Hand-written HIP kernels through the C ABI (csrc/layer_norm.hip, window_attn*.hip); float32, float16 and bfloat16, sums in float32.

Tensors live on one GPU, nothing is moved silently; kernels run on torch's current stream of that GPU.  Gradients are first derivatives only, summed in a fixed
order (the same bits every time); tangents of forward mode and tracers (torch.jit.trace, make_fx), which would not see the kernels, are refused.  Argument checks,
allocation and the autograd nodes are compiled (csrc/sequence_torch.cpp)."""
import ctypes
import importlib
import os

import torch
import torch.nn as nn

from .. import _lib
from .._lib import GfppError

_p, _u32, _i32, _i64, _u64, _f, _i = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_int32, ctypes.c_int64, ctypes.c_uint64, ctypes.c_float, ctypes.c_int
_strides = ctypes.POINTER(ctypes.c_int64)
_lib.register("gfpp_layer_norm_forward", [_p, _i64, _p, _p, _i, _u64, _u32, _f, _i, _p, _p, _p, _p])
_lib.register("gfpp_layer_norm_backward", [_p, _i64, _p, _i64, _p, _i, _p, _p, _u64, _u32, _i, _p, _p, _p, _p, _p])
_lib.register("gfpp_layer_norm_backward_scratch_floats", [_u64, _u32], restype=ctypes.c_uint64)
_lib.register("gfpp_rotary", [_p, _strides, _u32, _p] * 2 + [_p, _i, _i64, _p, ctypes.POINTER(_u32)] + [_u32] * 4 + [_i] * 3 + [_p])
_lib.register("gfpp_window_attn_two_part", [_u32] + [_i32] * 3 + [_i])
_lib.register("gfpp_window_attn_forward", [_p] * 6 + [_strides] + [_u32] * 6 + [_i32] * 4 + [_p, _f, _i, _p])
_lib.register("gfpp_window_attn_backward", [_p] * 11 + [_strides] + [_u32] * 6 + [_i32] * 4 + [_p, _f, _i, _p])
_lib.register("gfpp_window_attn_backward_scratch_floats", [_u32] * 6 + [_i32] * 4 + [_i], restype=ctypes.c_uint64)
_lib.register("gfpp_window_attn_step", [_p] * 6 + [_i, _p, _strides] + [_u32] * 6 + [_f, _i, _p, _p])
_lib.register("gfpp_window_attn_step_scratch_floats", [_u32] * 5, restype=ctypes.c_uint64)
_SYMBOLS = ("gfpp_last_error", "gfpp_layer_norm_forward", "gfpp_layer_norm_backward", "gfpp_layer_norm_backward_scratch_floats", "gfpp_rotary", "gfpp_window_attn_two_part",
            "gfpp_window_attn_forward", "gfpp_window_attn_backward", "gfpp_window_attn_backward_scratch_floats", "gfpp_window_attn_step",
            "gfpp_window_attn_step_scratch_floats")
_ops = None


def ops():
    """The compiled binding (csrc/sequence_torch.cpp), given the entry points of the library that _lib has loaded.  Raises if it has not been built."""
    global _ops
    if _ops is None:
        library = _lib.lib()
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "_sequence.so")
        if not os.path.exists(path):
            raise GfppError(f"{path} is missing: run `python -c 'import __graft_entry__ as g; g.build()'` (or `make -C genefaceplusplus_amd/csrc`). There is no fallback.")
        module = importlib.import_module("genefaceplusplus_amd._sequence")
        module.bind({name: ctypes.cast(getattr(library, name), ctypes.c_void_p).value for name in _SYMBOLS})
        _ops = module
    return _ops


# ---- layer norm ------------------------------------------------------------------------------------------------------------------------------------------
def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x [..., N]; differentiable in x, weight and bias.

    weight, bias: [N], float32 or x's type (both the same), or None.  The output has x's type; statistics and sums are float32."""
    return (_ops or ops()).layer_norm(x, weight, bias, eps)


class LayerNorm(nn.Module):
    """Layer norm over the last axis, parameters named as in torch's (``weight``, ``bias``)."""

    def __init__(self, dim, eps=1e-5, affine=True):
        super().__init__()
        self.dim, self.eps = dim, eps
        self.weight = nn.Parameter(torch.ones(dim)) if affine else None
        self.bias = nn.Parameter(torch.zeros(dim)) if affine else None

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)


# ---- attention with a sliding window and sinks ---------------------------------------------------------------------------------------------------------------
def window_attention(q, k, v, left=None, right=0, sinks=0, lengths=None, scale=None, q_start=None):
    """softmax(scale q k^T) v over the keys that each query sees; differentiable in q, k and v.

    q [B, Tq, Hq, D], k and v [B, Tk, Hk, D], Hq a multiple of Hk (query head h reads key head h // (Hq // Hk)), D up to 128 -> [B, Tq, Hq, D].
    The query at position p = q_start + i sees key j iff ``j <= p + right and (j >= p - left or j < sinks)``; left / right None: no end on that side.  Queries are tokens of
    the sequence: one at p >= Tk is behind its end and sees nothing.  q_start: Tk - Tq by default (the queries are the last tokens).  lengths: [B] int32 / int64 on the GPU, tokens of every sequence: what lies behind is neither
    read nor seen, its output rows and gradients are zero, as are those of a query that sees nothing.  Within its length a sequence has to be finite.
    scale: D ** -0.5 by default."""
    return (_ops or ops()).window_attention(q, k, v, left, right, sinks, lengths, scale, q_start)


def window_attention_step(q, k, v, cache_k, cache_v, positions, sinks=0, scale=None):
    """One new token of every stream: k and v are written into the rolling cache (in place), the attention of q over what it then holds is returned.

    q [B, Hq, D], k and v [B, Hk, D] -> [B, Hq, D]; cache_k, cache_v [B, slots, Hk, D] (any strides with a dense last axis) hold a stream's first `sinks` tokens
    and its last W = slots - sinks ones, the token at position n in slot ``n if n < sinks else sinks + (n - sinks) % W``.  positions: [B] int32 / int64 on the GPU, the
    new tokens' positions; a negative one leaves its stream as it is (output zeros).  The result is row n of window_attention(left=W - 1, right=0, sinks=sinks)
    over the whole stream.  No two slots may share memory, and q, k, v may not lie in the caches.  Serving only: no gradients; the caches count as modified in place (a
    backward pass that has kept them raises).  Positions and caches are read on the GPU, so a captured graph of steps can be replayed."""
    return (_ops or ops()).window_attention_step(q, k, v, cache_k, cache_v, positions, sinks, scale)


class WindowCache:
    """The rolling cache of one layer for `batch` streams: keys and values [batch, sinks + window, kv_heads, dim] and the streams' next positions [batch] int32."""

    def __init__(self, batch, kv_heads, dim, window, sinks=0, dtype=torch.bfloat16, device="cuda"):
        if window < 1 or sinks < 0:
            raise GfppError(f"WindowCache: window {window} must be at least 1, sinks {sinks} at least 0")
        self.window, self.sinks = int(window), int(sinks)
        shape = (batch, self.sinks + self.window, kv_heads, dim)
        self.k, self.v = torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)
        self.positions = torch.zeros(batch, dtype=torch.int32, device=device)

    @torch.no_grad()
    def fill(self, k, v, lengths=None):
        """What a stream's steps would have left after the tokens k, v [batch, T, kv_heads, dim] (the first lengths[b] of each), in place of what the cache held."""
        B, T = k.shape[:2]
        if tuple(k.shape) != tuple(v.shape) or (B, *k.shape[2:]) != (self.k.shape[0], *self.k.shape[2:]):
            raise GfppError(f"WindowCache.fill: k, v must be [{self.k.shape[0]}, T, {self.k.shape[2]}, {self.k.shape[3]}], got {tuple(k.shape)}, {tuple(v.shape)}")
        if k.dtype != self.k.dtype or v.dtype != self.k.dtype:
            raise GfppError(f"WindowCache.fill: k, v must be {self.k.dtype}, got {k.dtype}, {v.dtype}")
        if k.device != self.k.device or v.device != self.k.device:
            raise GfppError(f"WindowCache.fill: k, v must be on {self.k.device}, got {k.device}, {v.device}")
        if lengths is not None and (tuple(lengths.shape) != (B,) or lengths.dtype not in (torch.int32, torch.int64) or lengths.device != self.k.device):
            raise GfppError(f"WindowCache.fill: lengths must be an int32 or int64 tensor [{B}] on {self.k.device}, got {lengths.dtype} {tuple(lengths.shape)} on {lengths.device}")
        n = torch.full((B, 1), T, device=k.device) if lengths is None else lengths.to(torch.int64).clamp(0, T).view(B, 1)
        slot = torch.arange(self.sinks + self.window, device=k.device).view(1, -1)
        # the newest token of every ring slot: the last one before n whose distance from the first ring token leaves the slot's remainder
        newest = slot + torch.div(n - 1 - slot, self.window, rounding_mode="floor").clamp(min=0) * self.window
        token = torch.where(slot < self.sinks, slot, newest)
        held = (token < n)[..., None, None]
        if T == 0:
            self.k.zero_(), self.v.zero_()
        else:
            rows = torch.arange(B, device=k.device).view(B, 1)
            at = token.clamp(max=T - 1)
            self.k.copy_(torch.where(held, k[rows, at], torch.zeros((), dtype=k.dtype, device=k.device)))
            self.v.copy_(torch.where(held, v[rows, at], torch.zeros((), dtype=v.dtype, device=v.device)))
        self.positions.copy_(n.view(B))

    def step(self, q, k, v, scale=None):
        """window_attention_step at every stream's next position, which moves on by one.  A stream whose position has been set to a negative number rests: its output is
        zeros, its rows and its position stay until it is given one that is not."""
        out = window_attention_step(q, k, v, self.k, self.v, self.positions, self.sinks, scale)
        self.positions += self.positions >= 0
        return out
