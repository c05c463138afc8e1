"""The operators of a gated feed-forward block as they are measured: RMS norm with the residual's addition, the gated
unit (both projections, activation, product), and 8-bit activation checkpoints, forward and backward.

Shapes: widths 256 (mask decoder), 768 / 1024 / 1280 (the ViT encoders), gated widths of 8/3 of those rounded to a
multiple of 8, rows from one token to four images of 64 x 64 patches; odd sizes in between."""
import math

import torch

own = False

EPS = 1e-6
GROUP = 32  # columns that share a scale
_T = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one token through the norm of a ViT-H wide block: latency
        {"name": "norm_token", "op": "norm_fwd", "rows": 1, "d": 1280, "type": "bf16", "residual": True, "q8": False},
        # the norm in front of a block at training size, its output kept in 8 bits for the backward pass and read back
        {"name": "norm_train_q8", "op": "norm_fwd", "rows": 16384, "d": 1024, "type": "bf16", "residual": True, "q8": True},
        # its backward, the residual's gradient added
        {"name": "norm_back", "op": "norm_bwd", "rows": 16384, "d": 1280, "type": "bf16", "residual": True, "q8": False},
        # the prompt tokens of a decoder (147 prompts x 7 tokens), an odd width, fp32, from an 8-bit checkpoint
        {"name": "norm_back_odd", "op": "norm_bwd", "rows": 1029, "d": 251, "type": "f32", "residual": False, "q8": True},
        # one token through the gated unit: the weights' reading is the time
        {"name": "gated_token", "op": "gated_fwd", "rows": 1, "d": 1280, "f": 3416, "type": "bf16", "act": "silu", "save": "none"},
        # prompt tokens, a ragged number of rows, fp16, the projections kept in 16 bits
        {"name": "gated_prompts", "op": "gated_fwd", "rows": 1029, "d": 256, "f": 688, "type": "f16", "act": "gelu", "save": "16"},
        # four images of 4096 patches, the projections kept in 8 bits and read back
        {"name": "gated_train_q8", "op": "gated_fwd", "rows": 16384, "d": 1024, "f": 2736, "type": "bf16", "act": "silu", "save": "8"},
        # the backward pass of the prompt tokens
        {"name": "gated_back_prompts", "op": "gated_bwd", "rows": 1029, "d": 256, "f": 688, "type": "f16", "act": "gelu", "save": "16"},
        # the backward pass of a ViT-L wide block from 8-bit checkpoints, the product recomputed for the layer behind it
        {"name": "gated_back_q8", "op": "gated_bwd", "rows": 16384, "d": 1024, "f": 2736, "type": "bf16", "act": "silu", "save": "8"},
        # the largest: a ViT-H wide block from 16-bit projections
        {"name": "gated_back_large", "op": "gated_bwd", "rows": 16384, "d": 1280, "f": 3416, "type": "bf16", "act": "gelu", "save": "16"},
        # a checkpoint of the patches of one image: written and read
        {"name": "q8_image", "op": "q8", "rows": 4096, "d": 768, "type": "f16"},
        # a checkpoint of a batch's gated product
        {"name": "q8_batch", "op": "q8", "rows": 16384, "d": 2736, "type": "bf16"},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "gated_fwd", "gated_bwd", "q8"])
    if op in ("norm_fwd", "norm_bwd"):
        return {"op": op, "rows": _spread(rng, 1, 16384), "d": _spread(rng, 64, 1280),
                "type": rng.choice(["bf16", "f16", "f32"]), "residual": rng.random() < 0.7, "q8": rng.random() < 0.4}
    if op == "q8":
        return {"op": op, "rows": _spread(rng, 1, 16384), "d": _spread(rng, 64, 3416),
                "type": rng.choice(["bf16", "f16", "f32"])}
    d = 8 * _spread(rng, 32, 160)
    return {"op": op, "rows": _spread(rng, 1, 16384), "d": d, "f": 8 * _spread(rng, max(32, d // 8), d // 3),
            "type": rng.choice(["bf16", "f16"]), "act": rng.choice(["silu", "gelu"]),
            "save": rng.choice(["none", "16", "8"] if op == "gated_fwd" else ["16", "8"])}


# --------------------------------------------------------------------------------------------------------- 8 bits
def _two32(k):
    """2^k in 32 bits for whole k in [-126, 127], from its bits (a library's power need not be exact)."""
    return ((k.int() + 127) << 23).view(torch.float32)


def _two64(k):
    return ((k.long() + 1023) << 52).view(torch.float64)


def _q8(x):
    """8-bit values (in 32 bits, to be multiplied by their scales) and the scales' exponents, of [rows, columns] fp32."""
    rows, cols = x.shape
    pad = -cols % GROUP
    g = torch.nn.functional.pad(x, (0, pad)).view(rows, -1, GROUP)
    amax = torch.where(torch.isfinite(g), g.abs(), torch.zeros_like(g)).amax(-1)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1): the least k with amax <= 448 2^k = 0.875 2^(k + 9)
    k = torch.clamp(e - 9 + (m > 0.875).int(), min=-126)
    k = torch.where(amax > 0, k, torch.full_like(k, -126))
    v = (g * _two32(-k.unsqueeze(-1))).to(torch.float8_e4m3fn)
    return v.view(rows, -1)[:, :cols].contiguous(), (k + 127).to(torch.uint8)


def _dq8(v, b):
    rows, cols = v.shape
    s = _two32(b.int() - 127).repeat_interleave(GROUP, 1)[:, :cols]
    return v.float() * s


# --------------------------------------------------------------------------------------------------------- states
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _stream(g, rows, d):
    """Values of a residual stream: a few channels several times as large as the others."""
    return _randn(g, rows, d) * (0.6 + 3.0 * (torch.rand(d, generator=g, device="cuda") ** 8))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, rows, d, t = case["op"], case["rows"], case["d"], _T[case["type"]]
    st = dict(case)
    if op in ("norm_fwd", "norm_bwd"):
        st["w"] = 1.0 + 0.2 * _randn(g, d)
        s = _stream(g, rows, d)
        if op == "norm_fwd":
            st["x"] = s.to(t)
            st["r"] = (0.5 * _randn(g, rows, d)).to(t) if case["residual"] else None
        else:
            st["rstd"] = torch.rsqrt(s.square().mean(-1) + EPS)
            st["s"] = _q8(s) if case["q8"] else s.to(t)
            st["dy"] = (0.05 * _randn(g, rows, d)).to(t)
            st["dres"] = (0.05 * _randn(g, rows, d)).to(t) if case["residual"] else None
    elif op == "q8":
        st["x"] = _stream(g, rows, d).to(t)
    else:
        f = case["f"]
        st["x"] = _randn(g, rows, d).to(t)
        st["w"] = (_randn(g, 2 * f, d) * d ** -0.5).to(t)
        st["bias"] = 0.1 * _randn(g, 2 * f)
        if op == "gated_bwd":
            st["dh"] = (0.05 * _randn(g, rows, f)).to(t)
            gu = _randn(g, rows, 2 * f)
            if case["save"] == "8":
                v, b = _q8(gu.view(2 * rows, f))
                st["gu"] = (v.view(rows, 2, f), b.view(rows, 2, -1))
                st["xs"] = _q8(st["x"].float())
            else:
                st["gu"] = gu.to(t)
                st["xs"] = st["x"]
    return st


# ---------------------------------------------------------------------------------------------------- plain forms
def _act(name, v):
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    return 0.5 * v * (1.0 + torch.erf(v * 0.7071067811865476))


def _act_grad(name, v):
    if name == "silu":
        p = 1.0 / (1.0 + torch.exp(-v))
        return p * (1.0 + v * (1.0 - p))
    return 0.5 * (1.0 + torch.erf(v * 0.7071067811865476)) + v * 0.3989422804014327 * torch.exp(-0.5 * v * v)


def _plain_norm_fwd(st):
    t = _T[st["type"]]
    s = st["x"].float()
    if st["r"] is not None:
        s = s + st["r"].float()
    rstd = torch.rsqrt(s.square().mean(-1) + EPS)
    y = s * rstd.unsqueeze(-1) * st["w"]
    out = {"y": y.to(t), "rstd": rstd}
    if st["r"] is not None:
        out["s"] = s.to(t)
    if st["q8"]:
        out["kept"] = _dq8(*_q8(y)).to(torch.bfloat16)
    return out


def _plain_norm_bwd(st):
    s = _dq8(*st["s"]) if st["q8"] else st["s"].float()
    n = s * st["rstd"].unsqueeze(-1)
    dy = st["dy"].float()
    g = dy * st["w"]
    dx = st["rstd"].unsqueeze(-1) * (g - n * (g * n).mean(-1, keepdim=True))
    if st["dres"] is not None:
        dx = dx + st["dres"].float()
    return {"dx": dx.to(_T[st["type"]]), "dw": (dy * n).sum(0)}


def _plain_gated_fwd(st):
    t = _T[st["type"]]
    rows, f = st["rows"], st["f"]
    gu = st["x"].float() @ st["w"].float().t() + st["bias"]
    out = {"h": (_act(st["act"], gu[:, :f]) * gu[:, f:]).to(t)}
    if st["save"] == "16":
        out["gu"] = gu.to(t)
    elif st["save"] == "8":
        out["kept"] = _dq8(*_q8(gu.view(2 * rows, f))).view(rows, 2 * f).to(torch.bfloat16)
    return out


def _plain_gated_bwd(st):
    t = _T[st["type"]]
    rows, f = st["rows"], st["f"]
    if st["save"] == "8":
        gu = _dq8(st["gu"][0].view(2 * rows, f), st["gu"][1].view(2 * rows, -1)).view(rows, 2 * f)
        x = _dq8(*st["xs"])
    else:
        gu, x = st["gu"].float(), st["xs"].float()
    g, u, dh = gu[:, :f], gu[:, f:], st["dh"].float()
    a = _act(st["act"], g)
    dgu = torch.cat([dh * u * _act_grad(st["act"], g), dh * a], 1)
    return {"dx": (dgu @ st["w"].float()).to(t), "dw": (dgu.t() @ x).to(t), "db": dgu.sum(0), "h": (a * u).to(t)}


# --------------------------------------------------------------------------------------------- the framework's calls
def _own_norm_fwd(st):
    from dilabhelmholtzoct_amd import kernels
    x, w, r = st["x"], st["w"], st["r"]
    y = torch.empty_like(x)
    rstd = torch.empty(st["rows"], device=x.device)
    s = torch.empty_like(x) if r is not None else None
    q8 = kernels.q8_empty(x.shape, x.device) if st["q8"] else None
    kernels.rmsnorm_fwd(x, w, EPS, y, residual=r, sum_out=s, q8=q8, rstd=rstd)
    out = {"y": y, "rstd": rstd}
    if s is not None:
        out["s"] = s
    if q8 is not None:
        out["kept"] = kernels.dequant8(*q8, torch.empty(x.shape, device=x.device, dtype=torch.bfloat16))
    return out


def _own_norm_bwd(st):
    from dilabhelmholtzoct_amd import kernels
    dx, dw = kernels.rmsnorm_bwd(st["dy"], st["s"], st["rstd"], st["w"], torch.empty_like(st["dy"]), dres=st["dres"])
    return {"dx": dx, "dw": dw}


def _own_act(st):
    from dilabhelmholtzoct_amd import _lib
    return _lib.ACT_SILU if st["act"] == "silu" else _lib.ACT_GELU


def _own_gated_fwd(st):
    from dilabhelmholtzoct_amd import kernels
    x, rows, f = st["x"], st["rows"], st["f"]
    h = torch.empty(rows, f, device=x.device, dtype=x.dtype)
    save = None
    if st["save"] == "16":
        save = torch.empty(rows, 2 * f, device=x.device, dtype=x.dtype)
    elif st["save"] == "8":
        save = kernels.q8_empty((rows, 2, f), x.device)
    kernels.gated_fwd(x, st["w"], h, act=_own_act(st), bias=st["bias"], save=save)
    out = {"h": h}
    if st["save"] == "16":
        out["gu"] = save
    elif st["save"] == "8":
        kept = torch.empty(rows, 2, f, device=x.device, dtype=torch.bfloat16)
        out["kept"] = kernels.dequant8(*save, kept).view(rows, 2 * f)
    return out


def _own_gated_bwd(st):
    from dilabhelmholtzoct_amd import kernels
    dh, w, rows, d, f = st["dh"], st["w"], st["rows"], st["d"], st["f"]
    dx = torch.empty(rows, d, device=dh.device, dtype=dh.dtype)
    dw = torch.empty_like(w)
    db = torch.empty(2 * f, device=dh.device)
    h = torch.empty_like(dh)
    kernels.gated_bwd(dh, st["gu"], st["xs"], w, act=_own_act(st), dx=dx, dw=dw, db=db, h=h)
    return {"dx": dx, "dw": dw, "db": db, "h": h}


def _own_q8(st):
    from dilabhelmholtzoct_amd import kernels
    x = st["x"]
    q, b = kernels.quant8(x)
    return kernels.dequant8(q, b, torch.empty(x.shape, device=x.device, dtype=torch.bfloat16))


def run(state):
    op = state["op"]
    if own:
        return {"norm_fwd": _own_norm_fwd, "norm_bwd": _own_norm_bwd, "gated_fwd": _own_gated_fwd,
                "gated_bwd": _own_gated_bwd, "q8": _own_q8}[op](state)
    if op == "q8":
        return _dq8(*_q8(state["x"].float())).to(torch.bfloat16)
    return {"norm_fwd": _plain_norm_fwd, "norm_bwd": _plain_norm_bwd, "gated_fwd": _plain_gated_fwd,
            "gated_bwd": _plain_gated_bwd}[op](state)


# ------------------------------------------------------------------------------------------------------------- work
def work(case):
    op, rows, d = case["op"], case["rows"], case["d"]
    e = 4 if case["type"] == "f32" else 2
    n, k8 = rows * d, 1 + 1 / GROUP
    if op == "norm_fwd":
        streams = 4 if case["residual"] else 2
        return {"bytes": n * (streams * e + (2 * k8 + 2 if case["q8"] else 0)) + 4 * (d + rows), "flops": 6.0 * n}
    if op == "norm_bwd":
        streams = 3 if case["residual"] else 2
        return {"bytes": n * (streams * e + (k8 if case["q8"] else e)) + 4 * (2 * d + rows), "flops": 10.0 * n}
    if op == "q8":
        return {"bytes": n * (e + 2 * k8 + 2), "flops": 3.0 * n}
    f = case["f"]
    if op == "gated_fwd":
        kept = {"none": 0, "16": 2 * 2, "8": 2 * (2 * k8 + 2)}[case["save"]]
        return {"bytes": 2 * (n + 2 * f * d + rows * f) + kept * rows * f + 8 * f, "flops": 4.0 * n * f}
    kept = k8 if case["save"] == "8" else 2
    return {"bytes": 2 * rows * f * kept + n * kept + 2 * (2 * rows * f + n + 4 * f * d) + 8 * f, "flops": 8.0 * n * f}


# ------------------------------------------------------------------------------------------ the definition in 64 bits
def _grid8(v):
    """v (64 bits) at the nearest values of 4 exponent and 3 fraction bits, ties to even: steps of 2^-3 of the leading
    power of two, 2^-9 below 2^-6."""
    _, e = torch.frexp(v)
    step = _two64(torch.clamp(e - 1, min=-6) - 3)
    return torch.round(v / step) * step


def _exact_q8(y):
    cols, parts = y.shape[1], []
    for at in range(0, cols, GROUP):
        part = y[:, at:at + GROUP]
        top = part.abs().amax(1, keepdim=True)
        k = torch.ceil(torch.log2(torch.clamp(top, min=1e-300) / 448.0))
        scale = _two64(torch.clamp(k, min=-126.0))
        parts.append(_grid8(part / scale) * scale)
    return torch.cat(parts, 1)


def _exact_read(pair):
    v, b = pair
    v, b = v.reshape(-1, v.shape[-1]), b.reshape(-1, b.shape[-1])
    col = torch.arange(v.shape[1], device=v.device) // GROUP
    return v.double() * _two64(b.long() - 127)[:, col]


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "q8":
        return _exact_q8(st["x"].double())
    if op == "norm_fwd":
        s = st["x"].double() + (st["r"].double() if st["r"] is not None else 0.0)
        rstd = ((s * s).sum(1) / case["d"] + EPS) ** -0.5
        y = torch.einsum("rc,r,c->rc", s, rstd, st["w"].double())
        return {"y": y, "rstd": rstd, "s": s if st["r"] is not None else None, "kept": _exact_q8(y) if case["q8"] else None}
    if op == "norm_bwd":
        s = _exact_read(st["s"]) if case["q8"] else st["s"].double()
        rstd, dy = st["rstd"].double()[:, None], st["dy"].double()
        dot = (dy * st["w"].double() * s).sum(1, keepdim=True)
        dx = rstd * dy * st["w"].double() - s * rstd ** 3 * dot / case["d"]
        return {"dx": dx + (st["dres"].double() if st["dres"] is not None else 0.0), "dw": ((s * rstd) * dy).sum(0)}
    f, silu = case["f"], case["act"] == "silu"
    if op == "gated_fwd":
        x, w, b = st["x"].double(), st["w"].double(), st["bias"].double()
        g, u = x @ w[:f].t() + b[:f], x @ w[f:].t() + b[f:]
        cdf = torch.sigmoid(g) if silu else torch.special.ndtr(g)
        kept = torch.cat([_exact_q8(g), _exact_q8(u)], 1) if case["save"] == "8" else None
        return {"h": g * cdf * u, "gu": torch.cat([g, u], 1) if case["save"] == "16" else None, "kept": kept}
    if case["save"] == "8":
        gu, x = _exact_read(st["gu"]).view(case["rows"], 2, f), _exact_read(st["xs"])
    else:
        gu, x = st["gu"].double().view(case["rows"], 2, f), st["xs"].double()
    g, u, dh, w = gu[:, 0], gu[:, 1], st["dh"].double(), st["w"].double()
    cdf = torch.sigmoid(g) if silu else torch.special.ndtr(g)
    slope = g * cdf * (1 - cdf) if silu else g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    dg, du = dh * u * (cdf + slope), dh * g * cdf
    return {"dx": dg @ w[:f] + du @ w[f:], "dw": torch.cat([dg.t() @ x, du.t() @ x]),
            "db": torch.cat([dg.sum(0), du.sum(0)]), "h": g * cdf * u}
