"""The sequence operators in 64 bits, with bounds on how far an implementation in 32 bits (operands of its matrix products and outputs rounded to `dtype`) may be off.

u(dtype) = eps / 2 is the relative error of one rounding.  Bounds are first-order: every rounding of a value x adds u |x| there and travels with the absolute values
of what it is multiplied by; sums in 32 bits add at most (terms + a few) 2^-24 of the sum of their absolute values."""
import math

import torch

F32 = 2.0 ** -24


def u(dtype):
    return torch.finfo(dtype).eps / 2


def visible(n_q, n_k, q_start, left, right, sinks, n, device="cpu"):
    """[n_q, n_k] bool: what query i (position q_start + i) of a sequence of n tokens sees; None: no end."""
    p, j = q_start + torch.arange(n_q, device=device)[:, None], torch.arange(n_k, device=device)[None, :]
    near = torch.ones(n_q, n_k, dtype=torch.bool, device=device) if left is None else (j >= p - left)
    ahead = torch.ones(n_q, n_k, dtype=torch.bool, device=device) if right is None else (j <= p + right)
    return ahead & (near | (j < sinks)) & (j < n) & (p < n)


def attention(q, k, v, dout=None, left=None, right=0, sinks=0, lengths=None, scale=None, q_start=None):
    """{name: (value, bound)} of out and, with dout, dq, dk, dv; inputs [B, T, H, D] of any type; computed where they are."""
    dtype = q.dtype
    r = u(dtype) if dtype != torch.float32 else 0.0            # (32 bits: the matrix products take their operands as they are)
    ro = u(dtype)
    q, k, v = q.double(), k.double(), v.double()
    B, Tq, Hq, D = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    G = Hq // Hk
    scale = D ** -0.5 if scale is None else scale
    q_start = Tk - Tq if q_start is None else q_start
    names = ("out",) if dout is None else ("out", "dq", "dk", "dv")
    val = {n: torch.zeros_like(t) for n, t in zip(("out", "dq", "dk", "dv"), (q, q, k, v))}
    bnd = {n: torch.zeros_like(t) for n, t in val.items()}
    for b in range(B):
        n = Tk if lengths is None else max(0, min(int(lengths[b]), Tk))
        see = visible(Tq, Tk, q_start, left, right, sinks, n, q.device)
        inside_q, inside_k = ((start + torch.arange(t, device=q.device) < n)[:, None] for start, t in ((q_start, Tq), (0, Tk)))
        rows = see.any(1)
        for h in range(Hq):
            # what lies behind the sequence may hold anything: it is not part of the definition
            qh = torch.where(inside_q, q[b, :, h], 0.0)
            kh, vh = (torch.where(inside_k, t[b, :, h // G], 0.0) for t in (k, v))
            s = (qh @ kh.T) * scale
            P = torch.softmax(torch.where(see, s, -math.inf), 1)
            P = torch.where(rows[:, None], P, 0.0)
            # relative error of a probability: its score's (D products and sums, the scaling) and the largest score's of the row, the exponentials', the sum's
            es = (D + 8) * F32 * ((qh.abs() @ kh.abs().T) * scale + 1)
            ep = es + (es * see).amax(1, keepdim=True) + (Tk + 16) * F32
            o = P @ vh
            # an operand below the type's smallest normal number is rounded in steps of its own: by tiny(dtype) / 2 at most, whatever its size (half: 2^-25).  The
            # forward pass rounds exp(s - running maximum), at most 2^8 sizes above or below the final one
            least = tiny(dtype) / 2 if dtype != torch.float32 else 0.0
            eo = ((r + ep) * P) @ vh.abs() + 256 * least * (see.double() @ vh.abs()) + (Tk + 8) * F32 * (P @ vh.abs())
            val["out"][b, :, h], bnd["out"][b, :, h] = o, ro * o.abs() + eo * (1 + ro)
            if dout is None:
                continue
            g = torch.where(inside_q, dout[b, :, h].double(), 0.0)
            dP = g @ vh.T
            delta = (g * o).sum(1, keepdim=True)
            dS = P * (dP - delta)
            ga = g.abs()
            e_dp = (D + 4) * F32 * (ga @ vh.abs().T)
            e_delta = (ga * (ro * o.abs() + eo * (1 + ro))).sum(1, keepdim=True) + (D + 4) * F32 * (ga * o.abs()).sum(1, keepdim=True)
            e_ds = (r + ep + 4 * F32) * dS.abs() + P * (1 + ep) * (e_dp + e_delta) + least * see
            def product(m, e_m, x):
                return m @ x, e_m @ x.abs() + (m.shape[1] * G + 8) * F32 * (m.abs() @ x.abs())
            w, e = product(dS, e_ds, kh)
            val["dq"][b, :, h], bnd["dq"][b, :, h] = scale * w, scale * e + ro * (scale * w).abs()
            w, e = product(dS.T, e_ds.T, qh)
            val["dk"][b, :, h // G] += scale * w
            bnd["dk"][b, :, h // G] += scale * e
            w, e = product(P.T, ((r + ep) * P + least * see).T, g)
            val["dv"][b, :, h // G] += w
            bnd["dv"][b, :, h // G] += e
    for n in ("dk", "dv"):
        bnd[n] += ro * val[n].abs()
    return {n: (val[n], bnd[n] * 1.01 + 1e-30 + tiny(dtype)) for n in names}


def tiny(dtype):
    """Half a step at the small end of a type: what a rounding may be off where relative steps end."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps


def layer_norm(x, weight, bias, eps, dy=None, param_dtype=torch.float32):
    """{name: (value, bound)} of y and, with dy, dx, dweight, dbias; x [M, N]."""
    dtype = x.dtype
    x = x.double()
    M, N = x.shape
    w = torch.ones(N, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(N, dtype=torch.float64) if bias is None else bias.double()
    mean = x.mean(1, keepdim=True)
    rstd = ((x - mean).pow(2).mean(1, keepdim=True) + eps).rsqrt()
    xh = (x - mean) * rstd
    # sums: at most 8 192 / 256 terms in a row by one thread, then a tree (long rows: N / 256 terms)
    chain = 40 + N / 256
    e_mean = chain * F32 * x.abs().mean(1, keepdim=True)
    # rstd: half the variance's relative error; a wrong mean enters the variance squared and, doubled, as its product with the (zero-sum) centred values
    e_rstd = rstd * (chain * F32 + (e_mean * rstd).pow(2) + 4 * F32)
    e_xh = (e_mean + F32 * (x.abs() + mean.abs())) * rstd + xh.abs() * (e_rstd / rstd + 2 * F32)
    y = xh * w + b
    out = {"y": (y, u(dtype) * y.abs() + (e_xh * w.abs() + 2 * F32 * (y.abs() + (xh * w).abs())) * 1.01 + tiny(dtype))}
    if dy is None:
        return out
    dy = dy.double()
    g = dy * w
    m0, m1 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = rstd * (g - m0 - xh * m1)
    e_m0 = (chain + 2) * F32 * g.abs().mean(1, keepdim=True)
    e_m1 = (chain + 2) * F32 * (g * xh).abs().mean(1, keepdim=True) + (g.abs() * e_xh).mean(1, keepdim=True)
    e = rstd * (4 * F32 * (g.abs() + m0.abs() + (xh * m1).abs()) + e_m0 + e_xh * m1.abs() + xh.abs() * e_m1) + (e_rstd / rstd) * dx.abs()
    out["dx"] = (dx, u(dtype) * dx.abs() + e * 1.01 + tiny(dtype))
    terms = 64 + M / 64
    dw, db = (dy * xh).sum(0), dy.sum(0)
    out["dweight"] = (dw, u(param_dtype) * dw.abs() + (dy.abs() * e_xh).sum(0) * 1.01 + terms * F32 * (dy * xh).abs().sum(0) + tiny(param_dtype))
    out["dbias"] = (db, u(param_dtype) * db.abs() + terms * F32 * dy.abs().sum(0) + tiny(param_dtype))
    return out


def rotary(x, positions, frequencies, sections, interleaved=False, backward=False):
    """(value, bound) of x [B, T, H, D] turned; positions [T or B, T, axes]."""
    dtype = x.dtype
    x = x.double()
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    t = positions.double()[..., axis] * frequencies
    t = (t if t.dim() == 3 else t[None])[:, :, None, :] * (-1.0 if backward else 1.0)
    P = int(axis.numel())
    i0, i1 = (torch.arange(0, 2 * P, 2), torch.arange(1, 2 * P, 2)) if interleaved else (torch.arange(P), torch.arange(P, 2 * P))
    a, b = x[..., i0], x[..., i1]
    y, e = x.clone(), torch.zeros_like(x)
    y[..., i0], y[..., i1] = a * t.cos() - b * t.sin(), a * t.sin() + b * t.cos()
    # a fraction of a turn below 1/2, narrowed: 2 pi 2^-26; sine and cosine to 2 ulp; two products and their sum.  The position's own product in 64 bits: 2^-52 t
    e[..., i0] = e[..., i1] = (2 * math.pi * 2.0 ** -26 + 5 * F32 + 2.0 ** -51 * t.abs()) * (a.abs() + b.abs())
    e += u(dtype) * y.abs() + tiny(dtype)
    e[..., 2 * P:] = 0.0
    return y, e


def close(got, value_bound, name):
    value, bound = value_bound
    got = got.detach().double().to(value.device)
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    off = (got - value).abs() - bound
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 0.0, f"{name}: off by {(got - value).abs().max().item():.3g}, {worst:.3g} over the bound at {divmod(int(off.argmax()), off.shape[-1])}"
