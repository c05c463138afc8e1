"""The gated unit's activations relative to their own value, far into their tails, and the norm's rstd, where the sum of
squares is exact. Tolerances in half steps of fp32 (U32) come from the kernels' arithmetic:

GELU's g P(-|g|): t = 1 / (1 + p |g|) is off by 4 (constant, fma, one step of the reciprocal), which the polynomial's slope
multiplies by at most 2.7; the polynomial's eight terms by 15 at most (weighted by their size); its fit by 2; the exponential
by 2 and by what its argument is off: three roundings of g^2 / 2, 1.5 g^2 half steps; the products and 1 - q by 3: 36 + 1.5 g^2.
SiLU: two roundings of the exponent, 2 |g|; the exponential 2, the sum 1, the reciprocal 2, the products 2: 8 + 2 |g|.
The others are exact. The factors u and dh are powers of two."""
import math

import pytest
import torch

import gated_ref as ref
from gated_ref import U32, half_step, tiny

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAMES = ["gelu", "silu", "relu", "none"]


@pytest.fixture(scope="module")
def k(cuda):
    from dilabhelmholtzoct_amd import kernels
    return kernels


def code(name):
    from dilabhelmholtzoct_amd import _lib
    return {"none": _lib.ACT_NONE, "relu": _lib.ACT_RELU, "gelu": _lib.ACT_GELU, "silu": _lib.ACT_SILU}[name]


def cdf_of(g):
    """The normal distribution function without the cancellation of 1 + erf."""
    return 0.5 * torch.special.erfc(g * -math.sqrt(0.5))


def act(name, g):
    """As ref.act, without cancellation in the left tail."""
    return g * cdf_of(g) if name == "gelu" else ref.act(name, g)


def steps(name, g):
    """Relative error of act(g) in half steps of fp32."""
    return {"gelu": 36 + 1.5 * g * g, "silu": 8 + 2 * g.abs()}.get(name, torch.zeros_like(g))


def within(got, want, tol):
    tol = tol * (1 + 2.0 ** -10)  # (errors of errors)
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - want).abs() / tol)[bad].max()))


def powers(n, dtype):
    """+-2^k, large in fp16, whose range ends before the tails do."""
    i = torch.arange(n, device="cuda")
    return (2.0 ** ((i % 5) + (6 if dtype == F16 else -2)) * torch.where(i % 3 == 0, -1.0, 1.0)).to(dtype)


# few rows (8, 16 and, with the 8-bit save, 32 features a workgroup), 64 x 64 and 128 x 128 tiles, two workgroups to a CU
@pytest.mark.parametrize("M,F,eight", [(16, 64, False), (16, 4104, False), (32, 96, True), (500, 64, False), (4096, 688, False),
                                       (25600, 136, False)])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("name", NAMES)
def test_forward(k, M, F, eight, dtype, name):
    g = torch.linspace(-12, 12, M, device="cuda").to(dtype)
    x = torch.zeros(M, 8, device="cuda", dtype=dtype)
    x[:, 0], x[:, 1] = g, 1.0
    w = torch.zeros(2 * F, 8, device="cuda", dtype=dtype)
    u = powers(F, dtype)
    w[:F, 0], w[F:, 1] = 1.0, u
    h = torch.empty(M, F, device="cuda", dtype=dtype)
    k.gated_fwd(x, w, h, act=code(name), save=k.q8_empty((M, 2, F), "cuda") if eight else None)
    g = g.double()[:, None]
    want = act(name, g) * u.double()
    within(h, want, want.abs() * (half_step(dtype) + steps(name, g) * U32) + tiny(dtype))


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("name", NAMES)
def test_backward(k, dtype, name):
    """h, and dg and du in fp32: db of a single row."""
    F = 4096
    g, u, dh = torch.linspace(-12, 12, F, device="cuda").to(dtype), powers(F, dtype), powers(F, dtype).flip(0).contiguous()
    gu, h, db = torch.cat([g, u])[None], torch.empty(1, F, device="cuda", dtype=dtype), torch.empty(2 * F, device="cuda")
    k.gated_bwd(dh[None], gu, None, torch.zeros(2 * F, 8, device="cuda", dtype=dtype), act=code(name), h=h, db=db)
    g, u, dh = g.double(), u.double(), dh.double()
    a = act(name, g)
    within(h[0], a * u, (a * u).abs() * (half_step(dtype) + steps(name, g) * U32) + tiny(dtype))
    within(db[F:], dh * a, (dh * a).abs() * steps(name, g) * U32)
    if name == "gelu":  # the distribution function, as above, + g times the density (constant, product, exponential), + 2
        cdf, rest = cdf_of(g), g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        off = cdf * steps(name, g) + rest.abs() * (4 + 1.5 * g * g)
    elif name == "silu":  # p (1 + g (1 - p)): 1 - p is off by p's error and half a step of 1 - p
        p = torch.sigmoid(g)
        cdf, rest, e = p, p * g * (1 - p), 5 + 2 * g.abs()
        off = e * (cdf + rest.abs()) + p * g.abs() * (p * e + 1 - p)
    else:
        cdf, rest, off = ref.act_grad(name, g), torch.zeros_like(g), torch.zeros_like(g)
    slope = cdf + rest
    within(db[:F], dh * u * slope, (dh * u).abs() * (off + 2 * (cdf + rest.abs())) * U32)


# lanes with 8 columns and with single ones, rows in one wave, in part of one and in four; beyond 8192 columns
@pytest.mark.parametrize("d", [8, 250, 256, 1000, 1021, 4096, 8000, 9000])
def test_rstd(k, d):
    """Whole values whose squares add up exactly. The mean + eps is off by two roundings (1 / d, one fma), which the root
    halves; rstd's own is half a step, the Newton step's square nothing: 2 half steps. y: one more for each product."""
    rows, eps = 512, 1e-6
    g = torch.Generator(device="cuda")
    g.manual_seed(d)
    x = torch.randint(-9, 10, (rows, d), generator=g, device="cuda").float() * torch.randint(1, 5, (rows, 1), generator=g, device="cuda")
    w = 1 + 0.2 * torch.randn(d, generator=g, device="cuda")
    y, rstd = torch.empty_like(x), torch.empty(rows, device="cuda")
    k.rmsnorm_fwd(x, w, eps, y, rstd=rstd)
    _, wr, wy = ref.norm_fwd(x, w, float(torch.tensor(eps, dtype=F32)))
    within(rstd, wr, wr * 2 * U32)
    within(y, wy, wy.abs() * 4 * U32)
