"""Plain 64-bit statements of the gated feed-forward operators (RMS norm with the residual's addition, gated unit, 8-bit
checkpoints) for the tests, and the tolerances the tests derive from the kernels' arithmetic."""
import math

import torch

GROUP = 32
U32 = 2.0 ** -24  # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the smallest step of a type (its subnormals')."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def two(k):
    """2^k in 64 bits for whole k, from its bits."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def q8(x):
    """(value bytes as float64, scale bytes) of [rows, columns]; non-finite elements are NaN and leave the scale alone."""
    x = x.double()
    rows, cols = x.shape
    ngr = -(-cols // GROUP)
    scale = torch.empty(rows, ngr, dtype=torch.uint8, device=x.device)
    out = torch.empty_like(x)
    for k in range(ngr):
        g = x[:, k * GROUP:(k + 1) * GROUP]
        a = torch.where(torch.isfinite(g), g.abs(), torch.zeros_like(g)).amax(1)
        e = torch.full_like(a, -126.0)
        nz = a > 0
        e[nz] = torch.clamp(torch.ceil(torch.log2(a[nz] / 448.0)), min=-126.0)
        # (log2 in 64 bits can sit on the wrong side of a border: settle it by the definition)
        e = torch.where(a > 448.0 * two(e), e + 1, e)
        e = torch.where((e > -126) & (a <= 448.0 * two(e - 1)), e - 1, e)
        scale[:, k] = (e + 127).to(torch.uint8)
        v = g / two(e)[:, None]
        _, ex = torch.frexp(v)
        step = two(torch.clamp(ex - 1, min=-6) - 3)
        r = torch.round(v / step) * step
        out[:, k * GROUP:(k + 1) * GROUP] = torch.where(torch.isfinite(g), r, torch.full_like(r, math.nan))
    return out, scale


def q8_value(values, scale):
    """What (values, scale bytes) stand for, in 64 bits."""
    v = values.double()
    v2, s2 = v.reshape(-1, v.shape[-1]), scale.reshape(-1, scale.shape[-1])
    col = torch.arange(v2.shape[1], device=v.device) // GROUP
    s = two(s2.long() - 127)
    s = torch.where(s2 == 255, torch.full_like(s, math.nan), s)
    return (v2 * s[:, col]).reshape(v.shape)


def act(name, g):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu":
        return 0.5 * g * (1 + torch.erf(g / math.sqrt(2)))
    if name == "relu":
        return torch.clamp(g, min=0)
    return g


def act_grad(name, g):
    if name == "silu":
        s = torch.sigmoid(g)
        return s * (1 + g * (1 - s))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(g / math.sqrt(2))) + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if name == "relu":
        return (g > 0).double()
    return torch.ones_like(g)


def norm_fwd(x, w, eps, r=None):
    s = x.double() if r is None else x.double() + r.double()
    rstd = (s.square().mean(-1) + eps) ** -0.5
    return s, rstd, s * rstd[:, None] * w.double()


def norm_bwd(dy, s, rstd, w, dres=None):
    """dx, dw, and the sums of magnitudes their fp32 rounding errors scale with."""
    dy, s, rstd, w = dy.double(), s.double(), rstd.double()[:, None], w.double()
    n, g = s * rstd, dy * w
    dx = rstd * (g - n * (g * n).mean(-1, keepdim=True))
    size = rstd * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True))
    if dres is not None:
        dx = dx + dres.double()
        size = size + dres.double().abs()
    return dx, (dy * n).sum(0), size, (dy * n).abs().sum(0)


def gated_fwd(x, w, name, bias=None):
    gu = x.double() @ w.double().t()
    if bias is not None:
        gu = gu + bias.double()
    f = gu.shape[1] // 2
    return gu, act(name, gu[:, :f]) * gu[:, f:]


def gated_bwd(dh, gu, x, w, name):
    dh, gu, x, w = dh.double(), gu.double(), x.double(), w.double()
    f = dh.shape[1]
    g, u = gu[:, :f], gu[:, f:]
    a = act(name, g)
    dgu = torch.cat([dh * u * act_grad(name, g), dh * a], 1)
    return {"h": a * u, "dgu": dgu, "dx": dgu @ w, "dw": dgu.t() @ x, "db": dgu.sum(0)}
