"""The sequence operators (csrc/layer_norm.hip, rotary.hip, window_attn*.hip) against their definitions in 64 bits, within the bounds of sequence_reference.py."""
import math

import pytest
import torch

import sequence_reference as ref
from genefaceplusplus_amd._lib import GfppError
from genefaceplusplus_amd.radnerfs import LayerNorm, RotaryEncoder, WindowCache, get_encoder, layer_norm, rotary_embed, window_attention, window_attention_step

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


def rand(gen, *shape, dtype=torch.float32, scale=1.0, mean=0.0):
    return (torch.randn(*shape, generator=gen) * scale + mean).to(dtype)


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


# ---- layer norm ------------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,N", [(1, 1), (3, 2), (5, 7), (1, 64), (2, 204), (9, 256), (4, 512), (7, 513), (3, 1000), (6, 1024), (2, 1025), (3, 2048), (2, 2049), (2, 4096),
                                 (3, 5000), (2, 8192), (2, 8200), (2, 20001), (4099, 40), (1500, 96)])
def test_layer_norm(dtype, M, N):
    g = gen(M * 31 + N)
    x = (rand(g, M, N, scale=3.0) + rand(g, N)).to(dtype)
    w, b, dy = rand(g, N, scale=0.3, mean=1.0), rand(g, N, scale=0.3), rand(g, M, N, dtype=dtype)
    for params in {torch.float32, dtype}:
        wp, bp = w.to(params), b.to(params)
        want = ref.layer_norm(x, wp, bp, 1e-5, dy, params)
        xg, wg, bg = (t.cuda().requires_grad_(True) for t in (x, wp, bp))
        y = layer_norm(xg, wg, bg)
        ref.close(y, want["y"], "y")
        for name, got in zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, (xg, wg, bg), dy.cuda())):
            assert got.dtype == (dtype if name == "dx" else params)
            ref.close(got, want[name], name)
        with torch.no_grad():
            assert torch.equal(layer_norm(xg, wg, bg), y)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_layer_norm_layouts_and_parts(dtype):
    g = gen(5)
    big, dy = rand(g, 6, 3, 130, dtype=dtype), rand(g, 6, 64, dtype=dtype)
    for x in (big[:, 1, 3:67], big[:, 0, :64], big[:, 2, 64:128], big[:, 1, ::2][:, :64], big[:1, 1, :64].expand(6, 64)):
        assert x.shape == (6, 64)
        want = ref.layer_norm(x, None, None, 1e-3, dy)
        whole = big.cuda()
        xg = torch.as_strided(whole, x.size(), x.stride(), x.storage_offset()).requires_grad_(True)
        y = layer_norm(xg, eps=1e-3)
        ref.close(y, want["y"], "y")
        ref.close(torch.autograd.grad(y, xg, dy.cuda())[0], want["dx"], "dx")
        # gradients of every layout: strided, one value for all rows
        on = dy.cuda()
        for d in (torch.stack((on, on), 2)[:, :, 1], on[:, :1].expand(6, 64), on[:1].expand(6, 64), torch.nn.functional.pad(on, (1, 2))[:, 1:65]):
            y = layer_norm(xg, eps=1e-3)
            ref.close(torch.autograd.grad(y, xg, d)[0], ref.layer_norm(x, None, None, 1e-3, d.cpu())["dx"], "dx")
    # one parameter without the other, gradients of one input alone
    x, w = big[:, 0, :64], rand(g, 64)
    y = layer_norm(x.cuda(), None, w.cuda().requires_grad_(True))
    ref.close(y, ref.layer_norm(x, None, w, 1e-5)["y"], "bias alone")
    wg = w.cuda().requires_grad_(True)
    y = layer_norm(x.cuda(), wg)
    ref.close(torch.autograd.grad(y, wg, dy.cuda())[0], ref.layer_norm(x, w, None, 1e-5, dy)["dweight"], "dweight alone")
    # no rows
    xg, wg, bg = torch.empty(0, 4, 8, device="cuda", dtype=dtype, requires_grad=True), torch.ones(8, device="cuda", requires_grad=True), torch.ones(8, device="cuda", requires_grad=True)
    y = layer_norm(xg, wg, bg)
    dx, dw, db = torch.autograd.grad(y, (xg, wg, bg), torch.empty_like(y))
    assert y.shape == dx.shape == (0, 4, 8) and not dw.any() and not db.any()
    # a row without spread: y = bias, no gradient but rstd's bound
    y = layer_norm(torch.full((2, 204), 7.0, device="cuda", dtype=dtype), torch.ones(204, device="cuda"), torch.full((204,), 0.5, device="cuda"))
    assert torch.equal(y, torch.full_like(y, 0.5))
    m = LayerNorm(64).cuda()
    ref.close(m(x.cuda()), ref.layer_norm(x, torch.ones(64), torch.zeros(64), 1e-5)["y"], "module")


def test_layer_norm_large_offset_keeps_its_spread():
    """mean 10^4, spread 1: the centred variance keeps what E x^2 - mean^2 would lose."""
    x = rand(gen(1), 5, 1024, mean=1.0e4)
    ref.close(layer_norm(x.cuda()), ref.layer_norm(x, None, None, 1e-5)["y"], "y")


@pytest.mark.parametrize("dtype,N", [(torch.float32, 204), (torch.float32, 300), (torch.bfloat16, 1000), (torch.float16, 24), (torch.float16, 31)])
def test_layer_norm_many_rows(dtype, N):
    """Rows for every wavefront of the chip: several rows of a wavefront in flight, a last share that is not whole."""
    M = 64 * torch.cuda.get_device_properties(0).multi_processor_count + 3
    g = gen(N)
    x, w, b, dy = (rand(g, M, N, scale=2.0) + 1.0).to(dtype), rand(g, N, mean=1.0), rand(g, N), rand(g, M, N, dtype=dtype)
    want = ref.layer_norm(x, w, b, 1e-5, dy)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves)
    ref.close(y, want["y"], "y")
    for name, got in zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, leaves, dy.cuda())):
        ref.close(got, want[name], name)


@pytest.mark.parametrize("dtype,N", [(torch.float32, 100), (torch.bfloat16, 200), (torch.bfloat16, 8)])
def test_layer_norm_many_short_rows(dtype, N):
    """Four rows of a wavefront at a time, the last of them not whole."""
    test_layer_norm_many_rows(dtype, N)


# ---- rotary positions ------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,Hq,Hk,D,sections", [(1, 1, 1, 1, 2, (1,)), (2, 5, 3, 1, 64, (32,)), (1, 33, 2, 2, 40, (5, 11)), (3, 7, 4, 2, 128, (16, 24, 24)), (2, 9, 1, 3, 20, (3,)),
                                                  (1, 3, 2, 1, 96, (8, 8, 8, 8)), (2, 3, 1, 1, 33, (4, 0, 5)), (1, 2, 1, 1, 1040, (512,)), (1, 700, 2, 1, 16, (8,))])
def test_rotary(dtype, interleaved, B, T, Hq, Hk, D, sections):
    g = gen(T + D)
    q, k = rand(g, B, T, Hq, D, dtype=dtype), rand(g, B, T, Hk, D, dtype=dtype)
    A = len(sections)
    freq = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) for n in sections])
    for pos in (torch.randint(0, 4000000, (B, T, A), generator=g), torch.randint(-50, 50, (T, A), generator=g, dtype=torch.int32), rand(g, B, T, A, scale=100.0)):
        qg, kg = q.cuda().requires_grad_(True), k.cuda().requires_grad_(True)
        yq, yk = rotary_embed((qg, kg), pos.cuda(), freq.cuda(), sections, interleaved)
        ref.close(yq, ref.rotary(q, pos, freq, sections, interleaved), "q")
        ref.close(yk, ref.rotary(k, pos, freq, sections, interleaved), "k")
        dq, dk = torch.autograd.grad((yq, yk), (qg, kg), (q.cuda().flip(1), k.cuda().flip(1)))
        ref.close(dq, ref.rotary(q.flip(1), pos, freq, sections, interleaved, True), "dq")
        ref.close(dk, ref.rotary(k.flip(1), pos, freq, sections, interleaved, True), "dk")
        assert torch.equal(rotary_embed(qg.detach(), pos.cuda(), freq.cuda(), sections, interleaved), yq)
    # one of the pair alone
    yq, yk = rotary_embed((qg, kg.detach()), pos.cuda(), freq.cuda(), sections, interleaved)
    ref.close(torch.autograd.grad(yq, qg, q.cuda())[0], ref.rotary(q, pos, freq, sections, interleaved, True), "dq alone")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_rotary_layouts_and_encoder(dtype):
    g = gen(3)
    packed = rand(g, 2, 6, 5, 66, dtype=dtype)
    enc = RotaryEncoder(64, (8, 24))
    freq = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / n) for n in (8, 24)])
    pos = torch.randint(0, 1000, (6, 2), generator=g)
    dev = packed.cuda()
    for sl in ((slice(None), slice(None), slice(0, 3), slice(0, 64)), (slice(None), slice(None), slice(1, 4), slice(1, 65)), (slice(None), slice(None), slice(2, 5), slice(2, 66))):
        ref.close(enc(dev[sl], pos.cuda()), ref.rotary(packed[sl], pos, freq, (8, 24)), "slice")
    heads_first = packed[..., :64].permute(0, 2, 1, 3).contiguous()
    ref.close(enc(heads_first.cuda().permute(0, 2, 1, 3), pos.cuda()), ref.rotary(packed[..., :64], pos, freq, (8, 24)), "heads first")
    one = packed[:, :, :1, :64].expand(2, 6, 4, 64)
    ref.close(enc(one.cuda(), pos.cuda()), ref.rotary(one, pos, freq, (8, 24)), "expanded")
    assert rotary_embed(dev[:, :0, :, :64], pos[:0].cuda(), freq.cuda(), (8, 24)).shape == (2, 0, 5, 64)
    joint = RotaryEncoder(64, (8, 24), theta=500.0, joint=True, interleaved=True).half()
    ref.close(joint(dev[..., :64], pos.cuda()), ref.rotary(packed[..., :64], pos, 500.0 ** (-torch.arange(32, dtype=torch.float64) / 32), (8, 24), True), "joint")
    e, width = get_encoder("rotary", input_dim=3, dim=64)
    assert e.sections == (10, 10, 10) and width == 64


# ---- attention ---------------------------------------------------------------------------------------------------------------------------------------
CASES = [
    # B, T, Hq, Hk, D, left, right, sinks, lengths
    (1, 1, 1, 1, 1, None, 0, 0, None), (2, 1, 4, 2, 32, 0, 0, 0, None), (1, 2, 2, 1, 3, None, None, 0, None), (1, 31, 1, 1, 64, 3, 0, 0, None),
    (1, 33, 2, 2, 20, 0, 0, 0, None), (2, 64, 2, 1, 33, 5, 2, 1, None), (1, 127, 3, 1, 40, None, 0, 0, None), (1, 129, 2, 2, 128, 64, 64, 0, None),
    (2, 130, 4, 2, 100, 40, 0, 7, None), (1, 296, 4, 4, 16, 4, 3, 0, None), (3, 200, 2, 1, 64, 20, 10, 3, (200, 77, 0)), (2, 190, 6, 3, 40, None, 5, 0, (1, 190)),
    (1, 300, 2, 1, 64, 10, 0, 150, None), (1, 140, 1, 1, 48, 7, 0, 500, None), (1, 260, 5, 1, 96, 90, None, 2, (259,)), (2, 150, 2, 2, 64, 149, 149, 4, (150, 3)),
    (1, 520, 2, 1, 128, 130, 0, 4, None), (1, 257, 2, 2, 8, 0, 256, 1, None),
]


def attention_inputs(seed, B, Tq, Tk, Hq, Hk, D, dtype):
    g = gen(seed)
    return rand(g, B, Tq, Hq, D, dtype=dtype), rand(g, B, Tk, Hk, D, dtype=dtype), rand(g, B, Tk, Hk, D, dtype=dtype), rand(g, B, Tq, Hq, D, dtype=dtype)


def run_attention(q, k, v, dout, **how):
    """Forward and gradients of GPU tensors; the form without gradients has to give the same bits."""
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = window_attention(*leaves, **how)
    grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        assert torch.equal(window_attention(q, k, v, **how), out)
    return dict(zip(("out", "dq", "dk", "dv"), (out, *grads)))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("case", CASES, ids=[f"{c[1]}x{c[4]}h{c[2]}_{c[3]}w{c[5]}_{c[6]}s{c[7]}{'r' if c[8] else ''}" for c in CASES])
def test_attention(case, dtype):
    B, T, Hq, Hk, D, left, right, sinks, lengths = case
    q, k, v, dout = attention_inputs(T + D, B, T, T, Hq, Hk, D, dtype)
    how = dict(left=left, right=right, sinks=sinks)
    want = ref.attention(q, k, v, dout, lengths=lengths, **how)
    got = run_attention(*(t.cuda() for t in (q, k, v, dout)), lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32).cuda(), **how)
    for n in got:
        ref.close(got[n], want[n], n)
    for b, n in enumerate(lengths or ()):
        for t in got.values():
            assert not t[b, n:].any(), "rows behind the sequence are zero"


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("Tq,Tk,start,left,right,sinks", [(40, 200, None, 50, 0, 4), (1, 300, None, 100, 0, 2), (70, 100, 10, 20, 5, 0), (130, 64, 0, 10, 0, 0), (5, 140, 3, None, 0, 0),
                                                          (64, 64, 40, 16, 0, 1), (3, 2, 0, 0, 0, 0)])
def test_attention_chunks(Tq, Tk, start, left, right, sinks, dtype):
    """Queries that are some of the tokens: a chunk of a stream against all its keys, queries behind the keys' end."""
    q, k, v, dout = attention_inputs(Tq + Tk, 2, Tq, Tk, 4, 2, 64, dtype)
    how = dict(left=left, right=right, sinks=sinks, q_start=start)
    want = ref.attention(q, k, v, dout, **how)
    got = run_attention(*(t.cuda() for t in (q, k, v, dout)), **how)
    for n in got:
        ref.close(got[n], want[n], n)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("D", [64, 40, 12])
def test_attention_layouts(D, dtype):
    """Packed projections, heads before tokens, rows that start anywhere, one key head for all batches: the same values as dense tensors, bit for bit."""
    B, T, Hq, Hk = 2, 150, 4, 2
    q, k, v, dout = (t.cuda() for t in attention_inputs(D, B, T, T, Hq, Hk, D, dtype))
    how = dict(left=30, right=3, sinks=2)
    want = run_attention(q, k, v, dout, **how)
    packed = torch.cat((q, k, v), 2)
    swapped = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (q, k, v)]
    odd = []
    for t in (q, k, v):
        room = torch.full((t.numel() + 1,), math.nan, device="cuda", dtype=dtype)
        room[1:] = t.flatten()
        odd.append(room[1:].view(t.shape))
    wide = [torch.nn.functional.pad(t, (3, 2), value=math.nan)[..., 3:3 + D] for t in (q, k, v)]
    for views in ((packed[:, :, :Hq], packed[:, :, Hq:Hq + Hk], packed[:, :, Hq + Hk:]), swapped, odd, wide, [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)]):
        for d in (dout, torch.stack((dout, dout), -1)[..., 0], torch.nn.functional.pad(dout, (1, 1))[..., 1:1 + D]):
            got = run_attention(*views, d, **how)
            for n in want:
                assert torch.equal(got[n], want[n]), n
    shared = [t[:1, :, :1].expand(B, T, Hk, D) for t in (k, v)]
    got, dense = run_attention(q, *shared, dout, **how), run_attention(q, *(t.contiguous() for t in shared), dout, **how)
    for n in want:
        assert torch.equal(got[n], dense[n]), n
    one = run_attention(q, k, v, dout[:, :1, :1, :1].expand_as(dout), **how)
    same = run_attention(q, k, v, dout[:, :1, :1, :1].expand_as(dout).contiguous(), **how)
    for n in want:
        assert torch.equal(one[n], same[n]), n


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_attention_padding_may_hold_anything(dtype):
    B, T, lengths = 4, 170, (170, 65, 1, 0)
    q, k, v, dout = attention_inputs(9, B, T, T, 4, 2, 64, dtype)
    lens = torch.tensor(lengths, dtype=torch.int64).cuda()
    how = dict(left=60, right=4, sinks=3, lengths=lens)
    want = run_attention(*(t.cuda() for t in (q, k, v, dout)), **how)
    for junk in (math.nan, math.inf, -math.inf, torch.finfo(dtype).min):
        dirty = []
        for t in (q, k, v, dout):
            t = t.clone()
            for b, n in enumerate(lengths):
                t[b, n:] = junk
            dirty.append(t.cuda())
        got = run_attention(*dirty, **how)
        for n in want:
            assert torch.equal(got[n], want[n]), (junk, n)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_attention_large_scores_and_scale(dtype):
    """Scores of some hundreds (one key takes all), a scale of one's own, rows whose first visible tiles are far below their later ones (the maximum grows)."""
    q, k, v, dout = attention_inputs(4, 1, 200, 200, 2, 1, 64, dtype)
    ramp = torch.linspace(0.1, 6.0, 200).view(1, 200, 1, 1)
    k = (k.float() * ramp).to(dtype)
    for scale in (0.9, 0.02):
        want = ref.attention(q, k, v, dout, left=None, right=None, scale=scale)
        got = run_attention(*(t.cuda() for t in (q, k, v, dout)), left=None, right=None, scale=scale)
        for n in got:
            ref.close(got[n], want[n], n)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_attention_alone_has_no_score_gradient(dtype):
    """A query that sees one key copies its value; its score's gradient is exactly zero."""
    q, k, v, dout = (t.cuda() for t in attention_inputs(2, 2, 100, 100, 4, 2, 72, dtype))
    got = run_attention(q, k, v, dout, left=0, right=0)
    assert torch.equal(got["out"], v.repeat_interleave(2, 2)) and not got["dq"].any() and not got["dk"].any()


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float32, 32), (torch.float16, 128)])
def test_attention_sinks_of_a_long_sequence(dtype, D):
    """Long enough for the sinks' tiles to be taken in slices; the same bits every time."""
    T = 2100
    q, k, v, dout = attention_inputs(7, 1, T, T, 2, 1, D, dtype)
    for sinks in (5, 200):
        how = dict(left=70, right=0, sinks=sinks)
        want = ref.attention(q, k, v, dout, **how)
        dev = [t.cuda() for t in (q, k, v, dout)]
        got = run_attention(*dev, **how)
        for n in got:
            ref.close(got[n], want[n], n)
        again = run_attention(*dev, **how)
        for n in got:
            assert torch.equal(got[n], again[n]), n


@pytest.mark.parametrize("dtype,B,Hq,Hk,D,left,right,sinks", [
    (torch.bfloat16, 4, 16, 4, 128, 150, 20, 3),           # two heads of a group a workgroup
    (torch.float16, 4, 16, 16, 120, 90, 0, 2),             # 128 keys a workgroup in the backward pass
    (torch.bfloat16, 4, 16, 16, 64, 300, 0, 0), (torch.float32, 4, 16, 16, 40, 100, 10, 1), (torch.float32, 4, 16, 16, 96, 100, 10, 1),
    (torch.bfloat16, 4, 16, 2, 64, 20, 11, 2), (torch.float16, 4, 16, 8, 33, 10, 0, 0), (torch.float32, 4, 16, 4, 32, 7, 8, 4)])      # few keys and a large grid
def test_attention_grids_that_fill_the_chip(dtype, B, Hq, Hk, D, left, right, sinks):
    """The variants that large grids take; the definition in 64 bits is computed on the GPU here."""
    T = 1100
    q, k, v, dout = (t.cuda() for t in attention_inputs(D, B, T, T, Hq, Hk, D, dtype))
    assert -(-T // 128) * Hq * B >= 2 * torch.cuda.get_device_properties(0).multi_processor_count
    lengths = (T, T - 1, 700, 5)
    how = dict(left=left, right=right, sinks=sinks)
    want = ref.attention(q, k, v, dout, lengths=lengths, **how)
    got = run_attention(q, k, v, dout, lengths=torch.tensor(lengths, dtype=torch.int32).cuda(), **how)
    for n in got:
        ref.close(got[n], want[n], n)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_attention_far_offsets(dtype):
    """A view into a batch whose heads lie more than 2^31 elements apart, and rows so far apart that 64 of them span more than 2^31 bytes."""
    T, D = 40, 64
    q, k, v, dout = attention_inputs(5, 1, T, T, 2, 2, D, dtype)
    want = run_attention(*(t.cuda() for t in (q, k, v, dout)), left=9)
    room = torch.empty(2 ** 31 + 2 ** 22, dtype=dtype, device="cuda")
    apart = torch.as_strided(room, (1, T, 2, D), (0, 2 * D, 2 ** 31 + 64, 1))
    apart.copy_(k.cuda())
    rows = torch.as_strided(room, (1, T, 2, D), (0, 2 ** 25, D, 1), 2 ** 21)
    got = run_attention(q.cuda(), apart, v.cuda(), dout.cuda(), left=9)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    rows.copy_(v.cuda())
    got = run_attention(q.cuda(), k.cuda(), rows, dout.cuda(), left=9)
    for n in want:
        assert torch.equal(got[n], want[n]), n


def test_other_device():
    """Tensors of another GPU than the current one."""
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    q, k, v, dout = attention_inputs(1, 1, 50, 50, 2, 1, 32, torch.bfloat16)
    want = run_attention(*(t.cuda() for t in (q, k, v, dout)), left=9)
    got = run_attention(*(t.to("cuda:1") for t in (q, k, v, dout)), left=9)
    assert torch.cuda.current_device() == 0
    for n in want:
        assert torch.equal(got[n].cpu(), want[n].cpu()), n


def test_attention_gradient_against_differences():
    """Directional derivatives of the 64-bit forward pass, central differences: sum(dout . out) moves by h grad . direction, up to h^2 third derivatives (h = 1e-5: below 1e-8)."""
    q, k, v, dout = attention_inputs(11, 2, 90, 90, 4, 2, 24, torch.float32)
    how = dict(left=30, right=2, sinks=2, lengths=(90, 41))
    got = run_attention(*(t.cuda() for t in (q, k, v, dout)), **{**how, "lengths": torch.tensor(how["lengths"], dtype=torch.int32).cuda()})
    g = gen(12)
    for at, (name, t) in enumerate((("dq", q), ("dk", k), ("dv", v))):
        d = rand(g, *t.shape).double()
        def loss(h):
            args = [x.double() for x in (q, k, v)]
            args[at] = args[at] + h * d
            return (ref.attention(*args, **how)["out"][0] * dout.double()).sum()
        change = (loss(1e-5) - loss(-1e-5)) / 2e-5
        mine = (got[name].double().cpu() * d).sum()
        # the kernel's 32 bits: its elementwise bound, summed
        slack = (ref.attention(q, k, v, dout, **how)[name][1] * d.abs()).sum() + 1e-6 * (1 + change.abs())
        assert (mine - change).abs() <= slack, (name, mine, change)


# ---- the step over a rolling cache -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("Hq,Hk,D,window,sinks,T", [(1, 1, 64, 1, 0, 4), (4, 2, 64, 5, 2, 19), (3, 1, 40, 40, 0, 70), (8, 2, 128, 33, 4, 80), (33, 1, 16, 9, 1, 25), (2, 2, 5, 3, 3, 12)])
def test_step_streams_the_offline_rows(Hq, Hk, D, window, sinks, T, dtype):
    """Token by token from an empty cache, past its wrap: every output is the row of the attention over the whole stream."""
    B = 3
    q, k, v, _ = attention_inputs(T, B, T, T, Hq, Hk, D, dtype)
    value, bound = ref.attention(q, k, v, left=window - 1, right=0, sinks=sinks)["out"]
    cache = WindowCache(B, Hk, D, window, sinks, dtype=dtype)
    qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
    for t in range(T):
        out = cache.step(qd[:, t], kd[:, t], vd[:, t])
        ref.close(out, (value[:, t], bound[:, t]), f"token {t}")
    assert cache.positions.tolist() == [T] * B
    other = WindowCache(B, Hk, D, window, sinks, dtype=dtype)
    other.fill(kd, vd)
    assert torch.equal(other.k, cache.k) and torch.equal(other.v, cache.v) and torch.equal(other.positions, cache.positions)


def test_cache_fill_of_ragged_streams():
    lengths = (0, 1, 6, 23, 40)
    g = gen(8)
    k, v = rand(g, 5, 40, 2, 8).cuda(), rand(g, 5, 40, 2, 8).cuda()
    cache = WindowCache(5, 2, 8, 7, 3, dtype=torch.float32)
    cache.fill(k, v, torch.tensor(lengths).cuda())
    for b, n in enumerate(lengths):
        alone = WindowCache(1, 2, 8, 7, 3, dtype=torch.float32)
        for t in range(n):
            alone.step(k[b:b + 1, t], k[b:b + 1, t], v[b:b + 1, t])
        assert torch.equal(alone.k[0], cache.k[b]) and torch.equal(alone.v[0], cache.v[b]) and int(cache.positions[b]) == n
    cache.fill(k[:, :0], v[:, :0])
    assert not cache.k.any() and not cache.positions.any()


def step_reference(q, k, v, cache_k, cache_v, positions, sinks):
    """Caches after the step and (value, bound) of its output, through the attention over the filled slots (any order: the softmax has none)."""
    ck, cv = cache_k.clone(), cache_v.clone()
    B, slots = ck.shape[:2]
    value, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b, n in enumerate(positions.tolist()):
        if n < 0:
            continue
        at = n if n < sinks else sinks + (n - sinks) % (slots - sinks)
        ck[b, at], cv[b, at] = k[b], v[b]
        m = min(n + 1, slots)
        value[b:b + 1, None], bound[b:b + 1, None] = ref.attention(q[b:b + 1, None], ck[b:b + 1, :m], cv[b:b + 1, :m])["out"]
    return ck, cv, (value, bound)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("B,Hq,Hk,D,slots,sinks", [(1, 8, 2, 64, 260, 4), (5, 4, 2, 128, 700, 4), (2, 6, 3, 40, 1025, 0), (1, 1, 1, 128, 3000, 1), (7, 70, 2, 32, 130, 7), (3, 2, 1, 33, 513, 2)])
def test_step(B, Hq, Hk, D, slots, sinks, dtype):
    """Young, full and wrapped streams, a stream that is left alone, caches of every layout; whatever an unfilled slot holds is not read."""
    g = gen(slots)
    q, k, v = rand(g, B, Hq, D, dtype=dtype), rand(g, B, Hk, D, dtype=dtype), rand(g, B, Hk, D, dtype=dtype)
    ck, cv = rand(g, B, slots, Hk, D, dtype=dtype), rand(g, B, slots, Hk, D, dtype=dtype)
    pos = torch.tensor([(10 * slots + 3, slots // 2, -1, 0, slots - 1, slots, 3 * 10 ** 9)[b % 7] for b in range(B)])
    for b, n in enumerate(pos.tolist()):
        ck[b, max(0, n):], cv[b, max(0, n):] = math.nan, math.nan
    wk, wv, want = step_reference(q, k, v, ck, cv, pos, sinks)
    for layout in ("dense", "heads", "layers", "odd"):
        if layout == "dense":
            dk, dv = ck.cuda(), cv.cuda()
        elif layout == "heads":
            dk, dv = (c.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3) for c in (ck, cv))
        elif layout == "layers":
            both = torch.stack((ck, cv), 1).cuda()
            dk, dv = both[:, 0], both[:, 1]
        else:
            dk, dv = (torch.nn.functional.pad(c, (1, 2)).cuda()[..., 1:1 + D] for c in (ck, cv))
        for p in (pos, pos.clamp(max=2 ** 31 - 1).to(torch.int32) if layout == "odd" and int(pos.max()) < 2 ** 31 else pos):
            out = window_attention_step(q.cuda(), k.cuda(), v.cuda(), dk, dv, p.cuda(), sinks)
            ref.close(out, want, layout)
            same = lambda a, b: torch.equal(a.cpu().nan_to_num(nan=9.0), b.nan_to_num(nan=9.0))  # noqa: E731
            assert same(dk, wk) and same(dv, wv), f"{layout}: one slot of every running stream is written, nothing else"


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("D,slots,sinks", [(16, 3901, 4), (40, 1570, 0), (64, 767, 1)])
def test_step_grids_that_fill_the_chip(D, slots, sinks, dtype):
    """Streams in five, two and one stretches, and key heads turned against the streams: young, full and wrapped ones, the last stretch not whole."""
    Hk = 8
    B = torch.cuda.get_device_properties(0).multi_processor_count // 2 // Hk + 1
    g = gen(slots)
    q, k, v = rand(g, B, 2 * Hk, D, dtype=dtype), rand(g, B, Hk, D, dtype=dtype), rand(g, B, Hk, D, dtype=dtype)
    ck, cv = rand(g, B, slots, Hk, D, dtype=dtype), rand(g, B, slots, Hk, D, dtype=dtype)
    pos = torch.tensor([(7 * slots + 900, slots // 5, -1, slots - 1, slots + 31, 795, 0)[b % 7] for b in range(B)])
    wk, wv, want = step_reference(q, k, v, ck, cv, pos, sinks)
    dk, dv = ck.cuda(), cv.cuda()
    ref.close(window_attention_step(q.cuda(), k.cuda(), v.cuda(), dk, dv, pos.cuda(), sinks), want, "out")
    assert torch.equal(dk.cpu(), wk) and torch.equal(dv.cpu(), wv)


@pytest.mark.parametrize("slots", [640, 1028, 4100])
def test_step_of_one_stream_in_stretches(slots):
    g = gen(slots)
    q, k, v = rand(g, 1, 8, 32, dtype=torch.bfloat16), rand(g, 1, 2, 32, dtype=torch.bfloat16), rand(g, 1, 2, 32, dtype=torch.bfloat16)
    ck, cv = rand(g, 1, slots, 2, 32, dtype=torch.bfloat16), rand(g, 1, slots, 2, 32, dtype=torch.bfloat16)
    for n in (slots - 2, slots // 2, 5 * slots + 1):
        pos = torch.tensor([n])
        wk, wv, want = step_reference(q, k, v, ck, cv, pos, 4)
        dk, dv = ck.cuda(), cv.cuda()
        ref.close(window_attention_step(q.cuda(), k.cuda(), v.cuda(), dk, dv, pos.cuda(), 4), want, n)
        assert torch.equal(dk.cpu(), wk) and torch.equal(dv.cpu(), wv)


# ---- streams, graphs, the run of them together ---------------------------------------------------------------------------------------------------------------
def test_other_stream():
    q, k, v, dout = (t.cuda() for t in attention_inputs(1, 1, 300, 300, 4, 2, 64, torch.bfloat16))
    x = rand(gen(2), 300, 256).cuda()
    want, want_n = run_attention(q, k, v, dout, left=50, sinks=2), layer_norm(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, got_n = run_attention(q, k, v, dout, left=50, sinks=2), layer_norm(x)
    side.synchronize()
    for n in want:
        assert torch.equal(got[n], want[n]), n
    assert torch.equal(got_n, want_n)


def test_captured_training_pass():
    """Norm, rotary, attention and their gradients in one graph, replayed on new inputs: the eager bits every time."""
    B, T, H, D = 2, 1100, 2, 64
    enc = RotaryEncoder(D, (32,))
    pos = torch.arange(T, device="cuda")[:, None]
    g = gen(4)
    static = [rand(g, B, T, H * D).cuda().requires_grad_(True), rand(g, H * D, scale=0.1, mean=1.0).cuda().requires_grad_(True), rand(g, H * D).cuda().requires_grad_(True)]
    dout = rand(g, B, T, H, D).cuda()

    def run(x, w, b):
        y = layer_norm(x, w, b).view(B, T, H, D)
        q, k = enc((y, y.flip(1)), pos)
        o = window_attention(q, k, y, left=64, sinks=3)
        return (o.detach(), *torch.autograd.grad(o, (x, w, b), dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = run(*static)
    for seed in range(4):
        with torch.no_grad():
            static[0].copy_(rand(gen(50 + seed), B, T, H * D))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in kept]
        want = run(*[t.detach().clone().requires_grad_(True) for t in static])
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_captured_steps():
    """A graph of one step, replayed past the cache's wrap; two graphs whose workspaces do not meet."""
    T, Hq, Hk, D, window, sinks = 30, 4, 1, 64, 600, 2
    q, k, v, _ = attention_inputs(3, 1, T, T, Hq, Hk, D, torch.bfloat16)
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    caches = [WindowCache(1, Hk, D, window, sinks) for _ in range(2)]
    old = rand(gen(6), 1, window + sinks - 10, Hk, D, dtype=torch.bfloat16).cuda()
    eager = WindowCache(1, Hk, D, window, sinks)
    for c in caches + [eager]:
        c.fill(old, old.flip(1))
    ins = [torch.zeros_like(t[:, 0]) for t in (q, k, v)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        caches[0].step(*ins)                                  # warm
    torch.cuda.current_stream().wait_stream(side)
    caches[0].fill(old, old.flip(1))
    graphs, outs = [], []
    for c in caches:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(c.step(*ins))
    for t in range(T):
        for x, src in zip(ins, (q, k, v)):
            x.copy_(src[:, t])
        for g in graphs:
            g.replay()
        want = eager.step(q[:, t], k[:, t], v[:, t])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want), t
    assert torch.equal(caches[0].k, eager.k) and torch.equal(caches[1].v, eager.v)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_block_offline_and_live(dtype):
    """A pre-norm attention block over a clip, with its gradients, and the same block fed token by token."""
    B, T, Hq, Hk, D, window, sinks = 2, 70, 4, 2, 32, 24, 2
    C = Hq * D
    g = gen(21)
    norm = LayerNorm(C).cuda()
    enc = RotaryEncoder(D, (6, 10))
    wqkv = (rand(g, (Hq + 2 * Hk) * D, C, dtype=dtype, scale=C ** -0.5)).cuda().requires_grad_(True)
    x = rand(g, B, T, C, dtype=dtype).cuda().requires_grad_(True)
    pos = torch.stack((torch.arange(T), torch.arange(T) % 9), -1).cuda()

    def project(h):
        return (h @ wqkv.t()).view(B, -1, Hq + 2 * Hk, D).split((Hq, Hk, Hk), 2)

    q, k, v = project(norm(x))
    qr, kr = enc((q, k), pos)
    out = window_attention(qr, kr, v, left=window - 1, right=0, sinks=sinks)
    dout = rand(g, B, T, Hq, D, dtype=dtype).cuda()
    grads = torch.autograd.grad(out, (x, wqkv, norm.weight, norm.bias), dout)
    assert all(torch.isfinite(t).all() and t.any() for t in grads)
    # every stage on what the stage before it gave
    want_q, want_k = (ref.rotary(t.detach().cpu(), pos.cpu(), enc.frequencies(x.device).cpu(), enc.sections) for t in (q, k))
    ref.close(qr, want_q, "q"), ref.close(kr, want_k, "k")
    ref.close(out, ref.attention(qr.detach().cpu(), kr.detach().cpu(), v.detach().cpu(), left=window - 1, right=0, sinks=sinks)["out"], "out")
    value, bound = ref.attention(qr.detach().cpu(), kr.detach().cpu(), v.detach().cpu(), left=window - 1, right=0, sinks=sinks)["out"]
    cache = WindowCache(B, Hk, D, window, sinks, dtype=dtype)
    with torch.no_grad():
        for t in range(T):
            live = cache.step(qr[:, t], kr[:, t], v[:, t])
            ref.close(live, (value[:, t], bound[:, t]), f"token {t}")


# ---- refusals on the GPU -----------------------------------------------------------------------------------------------------------------------------------
def test_refusals_leave_the_device_usable():
    x = torch.zeros(2, 4, 2, 8, device="cuda")
    with pytest.raises(GfppError, match="is on cpu"):
        layer_norm(x, torch.ones(8))
    with pytest.raises(GfppError, match="is on cpu"):
        window_attention(x, x, x.cpu())
    with pytest.raises(GfppError, match="no gradients"):
        window_attention_step(x[:, 0].requires_grad_(True), x[:, 0], x[:, 0], x, x.clone(), torch.zeros(2, dtype=torch.int32, device="cuda"))
    y = layer_norm(x.requires_grad_(True))
    (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    assert not layer_norm(x.detach()).any()
