"""What the sequence operators promise beside their values: state that belongs to others, streams that rest, calls at the edges of what is allowed."""
import ctypes
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import sequence_reference as ref
from genefaceplusplus_amd import _lib
from genefaceplusplus_amd._lib import GfppError
from genefaceplusplus_amd.radnerfs import RotaryEncoder, WindowCache, layer_norm, window_attention, window_attention_step

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


# ---- the step and what autograd keeps ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("view", [False, True])
def test_step_marks_its_caches_as_changed(view):
    """Keys and values that a backward pass still needs are not changed behind its back: as with any in-place operation of torch, the backward pass raises."""
    cache = WindowCache(2, 2, 32, window=6, sinks=1, dtype=torch.float32)
    cache.fill(rand(0, 2, 7, 2, 32), rand(1, 2, 7, 2, 32))
    q = rand(2, 2, 3, 4, 32).requires_grad_(True)
    for changed in (cache.k, cache.v):
        k, v = (cache.k[:, 1:], cache.v[:, 1:]) if view else (cache.k, cache.v)
        out = window_attention(q, k, v)
        before = changed._version
        with torch.no_grad():
            cache.step(rand(3, 2, 4, 32), rand(4, 2, 2, 32), rand(5, 2, 2, 32))
        assert changed._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()
    # nothing in between: the gradient is there
    window_attention(q, cache.k, cache.v).sum().backward()
    assert torch.isfinite(q.grad).all()
    with torch.inference_mode():                              # (tensors without a version)
        live = WindowCache(2, 2, 32, window=6, sinks=1, dtype=torch.float32)
        live.step(rand(3, 2, 4, 32), rand(4, 2, 2, 32), rand(5, 2, 2, 32))
        assert live.positions.tolist() == [1, 1]


# ---- streams that rest -----------------------------------------------------------------------------------------------------------------------------------
def test_parked_streams_stay():
    """A stream at a negative position: neither its rows nor its position move, however many steps the others take; put back, it goes on where it was."""
    B, T, Hq, Hk, D, window, sinks = 3, 12, 4, 2, 32, 5, 2
    q, k, v = rand(0, B, T, Hq, D), rand(1, B, T, Hk, D), rand(2, B, T, Hk, D)
    parked, free = (WindowCache(B, Hk, D, window, sinks, dtype=torch.float32) for _ in range(2))
    for t in range(4):
        parked.step(q[:, t], k[:, t], v[:, t]), free.step(q[:, t], k[:, t], v[:, t])
    held, rows = parked.positions[1].clone(), parked.k[1].clone()
    parked.positions[1] = -1
    for t in range(4, 9):
        out, want = parked.step(q[:, t], k[:, t], v[:, t]), free.step(q[:, t], k[:, t], v[:, t])
        assert not out[1].any() and torch.equal(out[::2], want[::2])
        assert parked.positions.tolist() == [t + 1, -1, t + 1] and torch.equal(parked.k[1], rows)
    parked.positions[1] = held
    alone = WindowCache(1, Hk, D, window, sinks, dtype=torch.float32)
    for t in (0, 1, 2, 3, 9, 10):
        want = alone.step(q[1:2, t], k[1:2, t], v[1:2, t])
        if t >= 9:
            assert torch.equal(parked.step(q[:, t], k[:, t], v[:, t])[1:2], want)


def test_parked_streams_stay_in_a_graph():
    cache = WindowCache(2, 1, 16, 4, 1, dtype=torch.float32)
    q, k = rand(0, 2, 2, 16), rand(1, 2, 1, 16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.step(q, k, k)
    torch.cuda.current_stream().wait_stream(side)
    cache.positions.copy_(torch.tensor([3, -5]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.step(q, k, k)
    rows = cache.k[1].clone()
    for t in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert cache.positions.tolist() == [4 + t, -5] and torch.equal(cache.k[1], rows)


@pytest.mark.parametrize("sinks", [0, 2])
def test_step_at_the_last_position(sinks):
    """The largest position that 64 bits hold: a wrapped stream like any other."""
    slots, last = 7, 2 ** 63 - 1
    window = slots - sinks
    near = sinks + (last - sinks) % window + 3 * window        # the same slot, a smaller number
    q, k, v = rand(0, 1, 2, 16), rand(1, 1, 1, 16), rand(2, 1, 1, 16)
    outs = []
    for n in (near, last, last - window):
        ck, cv = rand(3, 1, slots, 1, 16), rand(4, 1, slots, 1, 16)
        outs.append((window_attention_step(q, k, v, ck, cv, torch.tensor([n]).cuda(), sinks), ck, cv))
    for got in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got, outs[0]))
    assert outs[0][0].any()


# ---- memory ------------------------------------------------------------------------------------------------------------------------------------------------
def test_caches_of_one_memory_are_refused():
    """Slots that lie in one another, within a cache or between the two, would be written twice; halves of one allocation are apart."""
    B, slots, Hk, D = 2, 6, 2, 16
    q, k = rand(0, B, 4, D), rand(1, B, Hk, D)
    pos = torch.tensor([3, 9]).cuda()
    room = torch.zeros(4096, device="cuda")
    dense = (slots * Hk * D, Hk * D, D, 1)
    at = lambda offset, strides=dense: torch.as_strided(room, (B, slots, Hk, D), strides, offset)  # noqa: E731
    for ck, cv in ((at(0), at(0)), (at(0), at(D)), (at(0), at(dense[0])), (at(D // 2), at(0)), (at(0, (slots * Hk * D, Hk * D, D - 4, 1)), at(2048)), (at(0), at(1024, (64, Hk * D, D, 1))),
                   (at(0), at(dense[0] // 2, (slots * Hk * D, D, slots * D, 1)))):
        with pytest.raises(GfppError, match="one memory"):
            window_attention_step(q, k, k, ck, cv, pos)
    assert not room.any()
    want = window_attention_step(q, k, k, torch.zeros(B, slots, Hk, D, device="cuda"), torch.zeros(B, slots, Hk, D, device="cuda"), pos)
    tokens = torch.zeros(B, slots, 2, Hk, D, device="cuda")
    heads = torch.zeros(B, slots, Hk, 2, D, device="cuda")
    streams = torch.zeros(B, 2, slots, Hk, D, device="cuda")
    whole = torch.zeros(2, B, slots, Hk, D, device="cuda")
    swapped = torch.zeros(2, B, Hk, slots, D, device="cuda").transpose(2, 3)
    blocks = torch.zeros(B, 2, slots * Hk * D, device="cuda")
    for ck, cv in ((tokens[:, :, 0], tokens[:, :, 1]), (tokens[:, :, 1], tokens[:, :, 0]), (heads[..., 0, :], heads[..., 1, :]), (streams[:, 0], streams[:, 1]), (whole[0], whole[1]),
                   (swapped[0], swapped[1]), (blocks[:, 0].view(B, Hk, slots, D).transpose(1, 2), blocks[:, 1].view(B, slots, Hk, D)),
                   (blocks[:, 1].view(B, slots, Hk, D), blocks[:, 0].view(B, Hk, slots, D).transpose(1, 2))):
        ck.zero_(), cv.zero_()
        assert torch.equal(window_attention_step(q, k, k, ck, cv, pos), want)


# ---- transforms that see no kernel ---------------------------------------------------------------------------------------------------------------------------
def test_transforms_do_not_pass_unseen():
    x, w = rand(0, 3, 4, 2, 16), rand(1, 16)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: layer_norm(t, w))(x)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: layer_norm(t, w).sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: layer_norm(t, w), (x,), (x,))
    with forward_ad.dual_level(), pytest.raises(GfppError, match="forward mode"):
        layer_norm(forward_ad.make_dual(x, x), w)
    with pytest.raises(GfppError, match="traced"):
        torch.jit.trace(lambda t: layer_norm(t, w), (x,), check_trace=False)
    for call in (lambda t: layer_norm(t, w), lambda t: window_attention(t, t, t), lambda t: RotaryEncoder(16, (8,))(t, torch.arange(4.0, device="cuda")[:, None])):
        leaf = x.clone().requires_grad_(True)
        y = call(leaf)
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(lambda g: torch.autograd.grad(y, leaf, g, retain_graph=True))(x)
        assert torch.isfinite(torch.autograd.grad(y, leaf, x)[0]).all()
    assert not torch.isnan(layer_norm(x, w)).any()


# ---- the rotary encoder's frequencies ------------------------------------------------------------------------------------------------------------------------
def test_encoder_serves_first_and_trains_later():
    """A first call under inference_mode leaves nothing that a later training pass cannot use."""
    pos = torch.arange(5).cuda()[:, None]
    x = rand(0, 2, 5, 3, 16)
    served, fresh = RotaryEncoder(16, (8,)), RotaryEncoder(16, (8,))
    with torch.inference_mode():
        served(x, pos)
    leaf = x.clone().requires_grad_(True)
    y = served(leaf, pos)
    assert torch.equal(y, fresh(x, pos))
    (dx,) = torch.autograd.grad(y, leaf, x)
    ref.close(dx, ref.rotary(x.cpu(), pos.cpu(), 10000.0 ** (-torch.arange(8, dtype=torch.float64) / 8), (8,), backward=True), "dx")


def test_encoder_moved_to_the_gpu_can_be_captured():
    """Module.to / .cuda() brings the frequencies along (unrounded by .half()), so that the first call may be a captured one; without it capture is refused before it is broken."""
    pos = torch.arange(6).cuda()[:, None]
    x = rand(0, 1, 6, 2, 32, dtype=torch.float16)
    want = RotaryEncoder(32, (16,))(x, pos)
    moved = RotaryEncoder(32, (16,)).cuda().half()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = moved(x, pos)
        with pytest.raises(GfppError, match="captur"):
            RotaryEncoder(32, (16,))(x, pos)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


# ---- sizes at the edges ----------------------------------------------------------------------------------------------------------------------------------------
def test_backward_of_very_many_heads_with_sinks():
    """More (sequence, key head) pairs than a grid's second axis holds, long enough for the sinks' tile to be taken in slices: every head has the same data and the same gradients."""
    T, H, D = 300, 65540, 2
    q, k, v, dout = (rand(s, 1, T, 1, D) for s in range(4))
    how = dict(left=40, right=0, sinks=3)
    want = ref.attention(*(t.cpu() for t in (q, k, v, dout)), **how)
    leaves = [t.expand(1, T, H, D).detach().requires_grad_(True) for t in (q, k, v)]
    out = window_attention(*leaves, **how)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, dout.expand(1, T, H, D)))):
        assert torch.equal(got, got[:, :, :1].expand_as(got)), name
        ref.close(got[:, :, :1], want[name], name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_backward_of_many_sinks(dtype):
    """Many tiles of sinks of many heads: fewer slices than queries would make, so that their partial sums stay bounded; the same bits every time."""
    B, T, H, D, lengths = 2, 1100, 64, 16, (1100, 801)
    q, k, v, dout = (rand(s, B, T, H, D, dtype=dtype) for s in range(4))
    how = dict(left=20, right=3, sinks=1000)
    want = ref.attention(q, k, v, dout, lengths=lengths, **how)
    runs = []
    for _ in range(2):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = window_attention(*leaves, lengths=torch.tensor(lengths).cuda(), **how)
        runs.append((out, *torch.autograd.grad(out, leaves, dout)))
    for name, got, again in zip(("out", "dq", "dk", "dv"), *runs):
        ref.close(got, want[name], name)
        assert torch.equal(got, again), name


def test_layer_norm_of_very_wide_rows():
    """More columns than 2^16 workgroups of the column sums take side by side, more than 2^32 threads of the last launch."""
    N = 2 ** 26 + 35
    x, w, b, dy = rand(0, 1, N), rand(1, N), rand(2, N), rand(3, 1, N)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(db, dy[0])
    want = ref.layer_norm(x.detach(), w.detach(), b.detach(), 1e-5, dy)
    for name, got in (("y", y), ("dx", dx), ("dweight", dw)):
        value, bound = want[name]
        assert ((got.detach().double() - value).abs() <= bound).all(), name


@pytest.mark.parametrize("N", [8, 1000, 5000, 20000])
@pytest.mark.parametrize("dtype", [0, 2])
def test_layer_norm_backward_without_rows_from_c(dtype, N):
    """No rows, an address for dx all the same: the parameters' gradients are zeros."""
    lib = _lib.lib()
    size = 4 if dtype == 0 else 2
    room = torch.full((8, N), 7.0, device="cuda")
    scratch = torch.full((int(lib.gfpp_layer_norm_backward_scratch_floats(0, N)),), math.nan, device="cuda")
    p = [ctypes.c_void_p(room[i].data_ptr()) for i in range(8)]
    torch.cuda.synchronize()
    assert N * size % 16 == 0
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.gfpp_layer_norm_backward(p[0], N, p[1], N, p[2], 0, p[3], p[4], 0, N, dtype, p[5], p[6], p[7], ctypes.c_void_p(scratch.data_ptr()), stream) == 0, lib.gfpp_last_error()
    assert not room[6:].any() and (room[:6] == 7.0).all()


# ---- arguments in company --------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("Tq,Tk,start,left,right,sinks,lengths", [(70, 200, 100, 30, 0, 3, (200, 120, 0)), (64, 150, 60, 20, 10, 0, (61, 150, 124)), (90, 64, 10, None, 0, 2, (64, 11, 40)),
                                                                  (300, 330, 30, 70, 0, 5, (330, 200, 31))])
def test_chunks_of_padded_streams(Tq, Tk, start, left, right, sinks, lengths, dtype):
    """Queries that are some of the tokens of sequences of several lengths."""
    B, Hq, Hk, D = 3, 4, 2, 40
    q, k, v, dout = (rand(s, B, t, h, D, dtype=dtype) for s, (t, h) in enumerate(((Tq, Hq), (Tk, Hk), (Tk, Hk), (Tq, Hq))))
    how = dict(left=left, right=right, sinks=sinks, q_start=start)
    want = ref.attention(*(t.cpu() for t in (q, k, v, dout)), lengths=lengths, **how)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = window_attention(*leaves, lengths=torch.tensor(lengths).cuda(), **how)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, dout))):
        ref.close(got, want[name], name)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_step_of_strided_tokens(dtype):
    """Queries, keys and values out of one projection, every other head, one head for all, features apart."""
    B, Hq, Hk, D, slots, sinks = 3, 4, 2, 32, 40, 2
    q, k, v = rand(0, B, Hq, D, dtype=dtype), rand(1, B, Hk, D, dtype=dtype), rand(2, B, Hk, D, dtype=dtype)
    pos = torch.tensor([5, 100, 39], dtype=torch.int32).cuda()
    fresh = lambda: (rand(3, B, slots, Hk, D, dtype=dtype), rand(4, B, slots, Hk, D, dtype=dtype))  # noqa: E731
    ck, cv = fresh()
    want = (window_attention_step(q, k, v, ck, cv, pos, sinks), ck, cv)
    packed = torch.cat((q, k, v), 1)
    apart = [torch.stack((t, t), 2).view(B, -1, D)[:, ::2] for t in (q, k, v)]
    odd = [torch.nn.functional.pad(t, (1, 2))[..., 1:1 + D] for t in (q, k, v)]
    features = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    for a, b, c in ((packed[:, :Hq], packed[:, Hq:Hq + Hk], packed[:, Hq + Hk:]), apart, odd, features):
        assert torch.equal(a, q) and torch.equal(b, k) and torch.equal(c, v)
        ck, cv = fresh()
        got = (window_attention_step(a, b, c, ck, cv, pos, sinks), ck, cv)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    one = q[:, :1].expand(B, Hq, D)
    ck, cv = fresh()
    out = window_attention_step(one, k, v, ck, cv, pos, sinks)
    ck, cv = fresh()
    assert torch.equal(out, window_attention_step(one.contiguous(), k, v, ck, cv, pos, sinks))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("B,Tq,Tk", [(2, 5, 0), (2, 0, 9), (0, 5, 9), (2, 0, 0)])
@pytest.mark.parametrize("D,sinks", [(64, 0), (64, 3), (5, 1)])
def test_attention_of_nothing(dtype, B, Tq, Tk, D, sinks):
    """No keys, no queries, no sequences: outputs and gradients of the right shapes, all zeros."""
    q, k, v, dout = (rand(s, B, t, h, D, dtype=dtype) for s, (t, h) in enumerate(((Tq, 4), (Tk, 2), (Tk, 2), (Tq, 4))))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    for lengths in (None, torch.full((B,), Tk).cuda()):
        out = window_attention(*leaves, left=3, sinks=sinks, lengths=lengths, q_start=0)
        for t, like in zip((out, *torch.autograd.grad(out, leaves, dout)), (q, q, k, v)):
            assert t.shape == like.shape and t.dtype == dtype and not t.any()


def test_lengths_of_a_captured_pass_are_read_at_every_replay():
    """Lengths that change between the replays, in either type; what lies behind them stays zero."""
    B, T, H, D = 3, 90, 2, 32
    q, k, v, dout = (rand(s, B, T, H, D) for s in range(4))
    for kind in (torch.int32, torch.int64):
        lengths = torch.tensor((90, 17, 0), dtype=kind).cuda()
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]

        def run():
            out = window_attention(*leaves, left=20, right=2, sinks=1, lengths=lengths)
            return (out.detach(), *torch.autograd.grad(out, leaves, dout))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = run()
        for now in ((90, 17, 0), (0, 90, 33), (5, 64, 89), (200, -3, 1)):
            lengths.copy_(torch.tensor(now))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in kept]
            for a, b in zip(got, run()):
                assert torch.equal(a, b), now
