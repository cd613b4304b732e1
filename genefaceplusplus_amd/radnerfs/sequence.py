"""Sequence operators of the conditioning stage: layer norm, attention with a sliding window and visible first tokens, and its single-token step over a rolling cache.

The reference smooths its conditioning over windows of 1 .. 16 frames (AudioNet / AudioAttNet, modules/radnerfs/cond_encoder.py:98-180).  These are the operators of
a conditioning network over whole clips (thousands of frames, forward and backward) and over live streams (one token at a time); the rotary positions that go with
them are in encoders.py.  Hand-written HIP kernels through the C ABI (csrc/layer_norm.hip, window_attn*.hip); float32, float16 and bfloat16, sums in float32.

Tensors live on one GPU, nothing is moved silently; kernels run on torch's current stream of that GPU.  Gradients are first derivatives only, summed in a fixed
order (the same bits every time)."""
import ctypes

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import _lib
from .._lib import GfppError

_p, _u32, _i32, _i64, _u64, _f, _i = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_int32, ctypes.c_int64, ctypes.c_uint64, ctypes.c_float, ctypes.c_int
_strides = ctypes.POINTER(ctypes.c_int64)
_lib.register("gfpp_layer_norm_forward", [_p, _i64, _p, _p, _i, _u64, _u32, _f, _i, _p, _p, _p, _p])
_lib.register("gfpp_layer_norm_backward", [_p, _i64, _p, _i64, _p, _i, _p, _p, _u64, _u32, _i, _p, _p, _p, _p, _p])
_lib.register("gfpp_layer_norm_backward_scratch_floats", [_u64, _u32], restype=ctypes.c_uint64)
_lib.register("gfpp_window_attn_forward", [_p, _p, _p, _p, _p, _strides] + [_u32] * 6 + [_i32] * 4 + [_p, _f, _i, _p])
_lib.register("gfpp_window_attn_backward", [_p] * 10 + [_strides] + [_u32] * 6 + [_i32] * 4 + [_p, _f, _i, _p])
_lib.register("gfpp_window_attn_backward_scratch_floats", [_u32] * 6 + [_i32] * 3, restype=ctypes.c_uint64)
_lib.register("gfpp_window_attn_step", [_p] * 6 + [_i, _p, _strides] + [_u32] * 6 + [_f, _i, _p, _p])
_lib.register("gfpp_window_attn_step_scratch_floats", [_u32] * 5, restype=ctypes.c_uint64)

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
#: a window side without an end
_FAR = 1 << 29


def launch(device, name, *args):
    """One entry point on `device` and torch's current stream there, whatever the current device is."""
    if device.index == torch.cuda.current_device():
        _lib.call(name, *args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, torch.cuda.current_stream().cuda_stream)


def scratch_floats(device, name, *args):
    """The library's answer goes by the device's compute units."""
    if device.index == torch.cuda.current_device():
        return int(getattr(_lib.lib(), name)(*args))
    with torch.cuda.device(device):
        return int(getattr(_lib.lib(), name)(*args))


def check_tensors(what, like, **tensors):
    """Every given tensor on the GPU of `like` (the first one), of a supported type."""
    if not like.is_cuda:
        raise GfppError(f"{what}: tensors must be on the GPU (no CPU path)")
    if like.dtype not in DTYPES:
        raise GfppError(f"{what}: float32, float16 or bfloat16 expected, got {like.dtype}")
    for name, t in tensors.items():
        if t is not None and t.device != like.device:
            raise GfppError(f"{what}: {name} is on {t.device}, expected {like.device}")


def wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---- layer norm ------------------------------------------------------------------------------------------------------------------------------------------
def _rows(t, N):
    """t as [M, N] rows of one pitch: a view where the layout has one, a copy otherwise."""
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= 0:
        return t
    return t.contiguous().view(-1, N)


def _layer_norm_forward(x, weight, bias, eps, keep):
    N = x.shape[-1]
    rows = _rows(x, N)
    M = rows.shape[0]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty(2, M, dtype=torch.float32, device=x.device) if keep else None
    param = weight if weight is not None else bias
    launch(x.device, "gfpp_layer_norm_forward", rows.data_ptr(), rows.stride(0), _ptr(weight), _ptr(bias), DTYPES[param.dtype] if param is not None else 0, M, N,
           float(eps), DTYPES[x.dtype], y.data_ptr(), stats.data_ptr() if keep else None, stats[1].data_ptr() if keep else None)
    return y, rows, stats


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, rows, stats = _layer_norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(rows, weight, bias, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        rows, weight, bias, stats = ctx.saved_tensors
        M, N = rows.shape
        dev = rows.device
        dyr = _rows(dy, N)
        param = weight if weight is not None else bias
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        dx = torch.empty(dy.shape, dtype=rows.dtype, device=dev) if want_x else None
        dw, db = torch.empty_like(weight) if want_w else None, torch.empty_like(bias) if want_b else None
        scratch = None
        if want_w or want_b:
            scratch = torch.empty(scratch_floats(dev, "gfpp_layer_norm_backward_scratch_floats", M, N), dtype=torch.float32, device=dev)
        launch(dev, "gfpp_layer_norm_backward", dyr.data_ptr(), dyr.stride(0), rows.data_ptr(), rows.stride(0), _ptr(weight),
               DTYPES[param.dtype] if param is not None else 0, stats.data_ptr(), stats[1].data_ptr(), M, N, DTYPES[rows.dtype], _ptr(dx), _ptr(dw), _ptr(db),
               _ptr(scratch))
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x [..., N]; differentiable in x, weight and bias.

    weight, bias: [N], float32 or x's type (both the same), or None.  The output has x's type; statistics and sums are float32."""
    check_tensors("layer_norm", x, weight=weight, bias=bias)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise GfppError(f"layer_norm: the last axis must not be empty, got {tuple(x.shape)}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if tuple(p.shape) != (x.shape[-1],) or not p.is_contiguous():
            raise GfppError(f"layer_norm: {name} must be a contiguous [{x.shape[-1]}], got {tuple(p.shape)}")
        if p.dtype not in (torch.float32, x.dtype):
            raise GfppError(f"layer_norm: {name} must be float32 or {x.dtype}, got {p.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise GfppError(f"layer_norm: weight is {weight.dtype}, bias {bias.dtype}")
    if not eps >= 0:
        raise GfppError(f"layer_norm: eps must not be negative, got {eps}")
    if wants_grad(x, weight, bias):
        return _LayerNormFn.apply(x, weight, bias, eps)
    return _layer_norm_forward(x, weight, bias, eps, False)[0]


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
def _heads(t):
    """t [B, T, H, D] with a dense last axis."""
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _token_strides(*tensors):
    flat = [s for t in tensors for s in t.stride()[:3]]
    return (ctypes.c_int64 * len(flat))(*flat)


def _window_forward(q, k, v, window, lengths, scale, keep):
    B, Tq, Hq, D = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    out = torch.empty(B, Tq, Hq, D, dtype=q.dtype, device=q.device)
    lse = torch.empty(B, Hq, Tq, dtype=torch.float32, device=q.device) if keep else None
    launch(q.device, "gfpp_window_attn_forward", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(lse), _token_strides(q, k, v, out), B, Tq, Tk, Hq, Hk,
           D, *window, _ptr(lengths), scale, DTYPES[q.dtype])
    return out, lse


class _WindowAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, lengths, scale):
        out, lse = _window_forward(q, k, v, window, lengths, scale, True)
        ctx.save_for_backward(q, k, v, out, lse, lengths)
        ctx.window, ctx.scale = window, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, lengths = ctx.saved_tensors
        B, Tq, Hq, D = q.shape
        Tk, Hk = k.shape[1], k.shape[2]
        dev = q.device
        dout = _heads(dout)
        dq = torch.empty(q.shape, dtype=q.dtype, device=dev)
        dk, dv = torch.empty(k.shape, dtype=k.dtype, device=dev), torch.empty(v.shape, dtype=v.dtype, device=dev)
        left, right, sinks, start = ctx.window
        scratch = torch.empty(scratch_floats(dev, "gfpp_window_attn_backward_scratch_floats", B, Tq, Tk, Hq, Hk, D, left, sinks, start), dtype=torch.float32, device=dev)
        launch(dev, "gfpp_window_attn_backward", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(), lse.data_ptr(), dq.data_ptr(),
               dk.data_ptr(), dv.data_ptr(), scratch.data_ptr(), _token_strides(q, k, v, out, dout, dq, dk, dv), B, Tq, Tk, Hq, Hk, D, *ctx.window, _ptr(lengths),
               ctx.scale, DTYPES[q.dtype])
        return dq, dk, dv, None, None, None


def _check_heads(what, q, k, v, axes):
    check_tensors(what, q, k=k, v=v)
    if q.dim() != axes or k.dim() != axes or tuple(k.shape) != tuple(v.shape):
        raise GfppError(f"{what}: q, k, v must have {axes} axes and k the shape of v, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise GfppError(f"{what}: q, k, v must have one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    if q.shape[0] != k.shape[0] or q.shape[-1] != k.shape[-1]:
        raise GfppError(f"{what}: q and k differ in batch or head width: {tuple(q.shape)}, {tuple(k.shape)}")
    Hq, Hk, D = q.shape[-2], k.shape[-2], q.shape[-1]
    if Hk < 1 or Hq < 1 or Hq % Hk:
        raise GfppError(f"{what}: {Hq} query heads are no multiple of {Hk} key heads")
    if not 1 <= D <= 128:
        raise GfppError(f"{what}: head width {D} (1 .. 128 are supported)")


def _scale(what, scale, D):
    scale = float(D) ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise GfppError(f"{what}: scale must be positive, got {scale}")
    return scale


def window_attention(q, k, v, left=None, right=0, sinks=0, lengths=None, scale=None, q_start=None):
    """softmax(scale q k^T) v over the keys that each query sees; differentiable in q, k and v.

    q [B, Tq, Hq, D], k and v [B, Tk, Hk, D], Hq a multiple of Hk (query head h reads key head h // (Hq // Hk)), D up to 128 -> [B, Tq, Hq, D].
    The query at position p = q_start + i sees key j iff ``j <= p + right and (j >= p - left or j < sinks)``; left / right None: no end on that side.
    q_start: Tk - Tq by default (the queries are the last tokens).  lengths: [B] int32 / int64 on the GPU, tokens of every sequence: what lies behind is neither
    read nor seen, its output rows and gradients are zero, as are those of a query that sees nothing.  Within its length a sequence has to be finite.
    scale: D ** -0.5 by default."""
    what = "window_attention"
    _check_heads(what, q, k, v, 4)
    B, Tq, Tk = q.shape[0], q.shape[1], k.shape[1]
    for name, n in (("left", left), ("right", right), ("sinks", sinks)):
        if n is not None and (n != int(n) or n < 0):
            raise GfppError(f"{what}: {name} must be a whole number from 0, got {n}")
    if max(Tq, Tk, B) > _FAR:
        raise GfppError(f"{what}: more than 2^29 tokens or sequences")
    q_start = Tk - Tq if q_start is None else int(q_start)
    if not 0 <= q_start <= _FAR:
        raise GfppError(f"{what}: q_start {q_start} must be 0 .. 2^29 (more queries than keys need it given)")
    if lengths is not None:
        if not torch.is_tensor(lengths) or tuple(lengths.shape) != (B,) or lengths.dtype not in (torch.int32, torch.int64):
            raise GfppError(f"{what}: lengths must be an int32 or int64 tensor [{B}]")
        check_tensors(what, q, lengths=lengths)
        lengths = lengths.clamp(0, Tk).to(torch.int32) if lengths.dtype == torch.int64 else lengths.contiguous()
    window = (_FAR if left is None else min(int(left), _FAR), _FAR if right is None else min(int(right), _FAR), min(int(sinks or 0), _FAR), q_start)
    scale = _scale(what, scale, q.shape[3])
    q, k, v = _heads(q), _heads(k), _heads(v)
    if wants_grad(q, k, v):
        return _WindowAttentionFn.apply(q, k, v, window, lengths, scale)
    return _window_forward(q, k, v, window, lengths, scale, False)[0]


def window_attention_step(q, k, v, cache_k, cache_v, positions, sinks=0, scale=None):
    """One new token of every stream: k and v are written into the rolling cache (in place), the attention of q over what it then holds is returned.

    q [B, Hq, D], k and v [B, Hk, D] -> [B, Hq, D]; cache_k, cache_v [B, slots, Hk, D] (any strides with a dense last axis) hold a stream's first `sinks` tokens
    and its last W = slots - sinks ones, the token at position n in slot ``n if n < sinks else sinks + (n - sinks) % W``.  positions: [B] int32 / int64 on the GPU, the
    new tokens' positions; a negative one leaves its stream as it is (output zeros).  The result is row n of window_attention(left=W - 1, right=0, sinks=sinks)
    over the whole stream.  Serving only: no gradients.  Positions and caches are read on the GPU, so a captured graph of steps can be replayed."""
    what = "window_attention_step"
    _check_heads(what, q, k, v, 3)
    B, Hq, D = q.shape
    Hk = k.shape[1]
    check_tensors(what, q, cache_k=cache_k, cache_v=cache_v, positions=positions)
    for name, c in (("cache_k", cache_k), ("cache_v", cache_v)):
        if c.dim() != 4 or (c.shape[0], c.shape[2], c.shape[3]) != (B, Hk, D) or tuple(c.shape) != tuple(cache_k.shape):
            raise GfppError(f"{what}: {name} must be [{B}, slots, {Hk}, {D}] like the other, got {tuple(c.shape)}")
        if c.dtype != q.dtype:
            raise GfppError(f"{what}: {name} must be {q.dtype}, got {c.dtype}")
        if (D > 1 and c.stride(3) != 1) or any(s <= 0 and n > 1 for s, n in zip(c.stride(), c.shape)):
            raise GfppError(f"{what}: {name} needs a dense last axis and rows of its own (strides {c.stride()}): it is written in place")
    slots = cache_k.shape[1]
    if sinks != int(sinks) or not 0 <= sinks < slots:
        raise GfppError(f"{what}: sinks {sinks} must be 0 .. slots - 1 ({slots} slots)")
    if slots > _FAR:
        raise GfppError(f"{what}: more than 2^29 slots")
    if tuple(positions.shape) != (B,) or positions.dtype not in (torch.int32, torch.int64) or not positions.is_contiguous():
        raise GfppError(f"{what}: positions must be a contiguous int32 or int64 tensor [{B}]")
    if wants_grad(q, k, v, cache_k, cache_v):
        raise GfppError(f"{what}: no gradients (call it under torch.no_grad(); window_attention is the differentiable form)")
    scale = _scale(what, scale, D)
    q, k, v = (t if t.stride(2) == 1 or D == 1 else t.contiguous() for t in (q, k, v))
    out = torch.empty(B, Hq, D, dtype=q.dtype, device=q.device)
    n = scratch_floats(q.device, "gfpp_window_attn_step_scratch_floats", B, Hq, Hk, D, slots)
    scratch = torch.empty(n, dtype=torch.float32, device=q.device) if n else None
    strides = (ctypes.c_int64 * 14)(*q.stride()[:2], *k.stride()[:2], *v.stride()[:2], *cache_k.stride()[:3], *cache_v.stride()[:3], *out.stride()[:2])
    launch(q.device, "gfpp_window_attn_step", q.data_ptr(), k.data_ptr(), v.data_ptr(), cache_k.data_ptr(), cache_v.data_ptr(), positions.data_ptr(),
           int(positions.dtype == torch.int64), out.data_ptr(), strides, B, Hq, Hk, D, slots, int(sinks), scale, DTYPES[q.dtype], _ptr(scratch))
    return out


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
        if lengths is not None and tuple(lengths.shape) != (B,):
            raise GfppError(f"WindowCache.fill: lengths must be [{B}], got {tuple(lengths.shape)}")
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
        """window_attention_step at every stream's next position, which moves on by one."""
        out = window_attention_step(q, k, v, self.k, self.v, self.positions, self.sinks, scale)
        self.positions += 1
        return out
