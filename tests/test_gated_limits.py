"""Sizes at the ends of what the block operators' entries can count: widths that 32 bits do not hold are refused instead of
being cut to what is left of them, and so are widths whose loops or launches would pass 32 bits. No memory is touched: meta
tensors and pointers that are never dereferenced."""
import pytest
import torch

from dilabhelmholtzoct_amd import _lib, kernels

BF, F32 = torch.bfloat16, torch.float32
WIDE = 2 ** 32 + 64  # 64 in its lower 32 bits


def meta(*shape, dtype=BF):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(kernels, "_device_of", lambda *ts: 0)

    def never(*a):
        raise AssertionError("launched")
    monkeypatch.setattr(_lib, "call_on", never)


def test_widths_past_32_bits(no_launch):
    x, q = meta(1, WIDE), kernels.q8_empty((1, WIDE), "meta")
    w, rstd = meta(WIDE, dtype=F32), meta(1, dtype=F32)
    gw, gx, h, gu = meta(16, WIDE), meta(1, WIDE), meta(1, 8), meta(1, 16)
    tall, th, tx = meta(2 * WIDE, 8), meta(1, WIDE), meta(1, 8)
    for i, f in enumerate((lambda: kernels.quant8(x), lambda: kernels.quant8(x, q),
                           lambda: kernels.dequant8(*q, x),
                           lambda: kernels.rmsnorm_fwd(x, w, 1e-6, x),
                           lambda: kernels.rmsnorm_bwd(x, x, rstd, w, x, dw=w),
                           lambda: kernels.gated_fwd(gx, gw, h),
                           lambda: kernels.gated_fwd(tx, tall, th),
                           lambda: kernels.gated_bwd(h, gu, gx, gw, dx=gx),
                           lambda: kernels.gated_bwd(th, meta(1, 2 * WIDE), tx, tall, dx=tx))):
        with pytest.raises(ValueError, match="32 bits"):
            f()
            pytest.fail(f"case {i} was taken")


P = 1 << 20  # a 16-B aligned address


@pytest.mark.parametrize("rows,D", [(4, 2 ** 31 - 63), (4, 2 ** 31 - 1)])
def test_norm_forward_width(rows, D):
    lib = _lib.load()
    assert lib.octsam_rmsnorm_fwd(P, 0, 1 << 32, None, 0, 0, P, rows, D, 1e-6, None, 0, P, 0, 1 << 32, None, 0, None, 0, None, None) != 0
    assert b"D at most" in lib.octsam_last_error(), lib.octsam_last_error()


@pytest.mark.parametrize("rows,D", [(0, 2 ** 28), (17, 2 ** 28 - 15), (1 << 20, 2 ** 31 - 1), (16, 2 ** 30 - 63), (1, 2 ** 31 - 1)])
def test_norm_backward_width(rows, D):
    lib = _lib.load()
    assert lib.octsam_rmsnorm_bwd(P, 0, 1 << 32, P, 0, 1 << 32, None, 0, P, P, rows, D, None, 0, P, 0, 1 << 32, P, P, 1 << 62, None) != 0
    assert b"D at most" in lib.octsam_last_error(), lib.octsam_last_error()
