"""Refusals of the RMS norm, gated unit and 8-bit checkpoint entries: checked on the host, before any launch, so they need
no GPU. Pointers here are never dereferenced."""
import pytest
import torch

from dilabhelmholtzoct_amd import _lib, kernels

P = 1 << 20  # a 16-B aligned address
BF, F32, F16, Q8 = 0, 1, 2, 3


def refused(name, args, word):
    lib = _lib.load()
    assert getattr(lib, name)(*args) != 0
    assert word in lib.octsam_last_error(), lib.octsam_last_error()


def changed(base, **kw):
    d = dict(base)
    for key in kw:
        assert key in d, key
    d.update(kw)
    return list(d.values())


QUANT = dict(x=P, t=BF, ldx=64, rows=4, cols=64, q=P, ldq=64, s=P, lds=2, stream=None)
DEQUANT = dict(q=P, ldq=64, s=P, lds=2, rows=4, cols=64, y=P, t=F32, ldy=64, stream=None)
NORM = dict(x=P, xt=BF, ldx=64, r=P, rt=BF, ldr=64, w=P, rows=4, D=64, eps=1e-6, s=P, lds=64, y=P, yt=BF, ldy=64, q=P, ldq=64,
            sc=P, ldsc=2, rstd=P, stream=None)
NORM_B = dict(dy=P, dt=BF, lddy=64, s=P, st=BF, lds=64, sc=None, ldsc=0, rstd=P, w=P, rows=64, D=64, dres=P, lddres=64, dx=P, xt=BF,
              lddx=64, dw=P, ws=P, nb=1 << 20, stream=None)
GATED = dict(x=P, ldx=64, w=P, ldw=64, b=P, M=4, D=64, F=32, act=3, t=BF, h=P, ldh=32, save=P, st=BF, ldsave=64, sc=None, ldsc=0,
             stream=None)
GATED_B = dict(dh=P, lddh=32, gu=P, gt=BF, ldgu=64, gs=None, ldgs=0, x=P, xt=BF, ldx=64, xs=None, ldxs=0, w=P, ldw=64, M=4, D=64, F=32,
               act=3, t=BF, h=P, ldh=32, dx=P, lddx=64, dw=P, dwt=BF, lddw=64, db=P, ws=P, nb=1 << 30, stream=None)


@pytest.mark.parametrize("kw,word", [(dict(t=3), b"type"), (dict(x=None), b"null"), (dict(s=None), b"null"), (dict(ldx=63), b"stride"),
                                     (dict(lds=1), b"stride"), (dict(rows=-1), b"rows"), (dict(x=P + 1), b"aligned")])
def test_quant8(kw, word):
    refused("octsam_quant8", changed(QUANT, **kw), word)


@pytest.mark.parametrize("kw,word", [(dict(t=7), b"type"), (dict(y=None), b"null"), (dict(ldy=3), b"stride"), (dict(cols=-4), b"cols"),
                                     (dict(y=P + 2), b"aligned")])
def test_dequant8(kw, word):
    refused("octsam_dequant8", changed(DEQUANT, **kw), word)


@pytest.mark.parametrize("kw,word", [
    (dict(xt=4), b"type"), (dict(rt=F16), b"residual"), (dict(r=None), b"sum_out"), (dict(q=None), b"together"), (dict(D=0), b"D 0"),
    (dict(w=None), b"null"), (dict(lds=8), b"stride"), (dict(ldsc=1), b"stride"), (dict(y=P + 1), b"aligned"),
    (dict(r=None, s=None, y=None, q=None, sc=None, rstd=None), b"no output")])
def test_rmsnorm_fwd(kw, word):
    refused("octsam_rmsnorm_fwd", changed(NORM, **kw), word)


@pytest.mark.parametrize("kw,word", [
    (dict(dt=3), b"type"), (dict(st=Q8), b"8-bit"), (dict(sc=P), b"8-bit"), (dict(dw=None), b"null"), (dict(rstd=None), b"null"),
    (dict(lddres=1), b"stride"), (dict(ws=None), b"workspace"), (dict(nb=16), b"workspace"), (dict(dx=P + 1), b"aligned")])
def test_rmsnorm_bwd(kw, word):
    refused("octsam_rmsnorm_bwd", changed(NORM_B, **kw), word)


@pytest.mark.parametrize("kw,word", [
    (dict(t=F32), b"bf16 or fp16"), (dict(act=4), b"activation"), (dict(D=60, ldx=64, ldw=64), b"multiples of 8"),
    (dict(F=28), b"multiples of 8"), (dict(h=None), b"null"), (dict(st=F16), b"save"), (dict(st=Q8), b"scales"),
    (dict(save=None, sc=P), b"scales"), (dict(ldsave=32), b"stride"), (dict(ldx=68), b"16 bytes"), (dict(w=P + 8), b"16 bytes"),
    (dict(M=-1), b"M -1"), (dict(M=1 << 31), b"M 2147483648")])
def test_gated_fwd(kw, word):
    refused("octsam_gated_fwd", changed(GATED, **kw), word)


@pytest.mark.parametrize("kw,word", [
    (dict(t=F32), b"bf16 or fp16"), (dict(act=-1), b"activation"), (dict(D=4), b"multiples of 8"), (dict(dh=None), b"null"),
    (dict(gt=F16), b"projections"), (dict(gt=Q8), b"scales"), (dict(w=None), b"dx needs w"), (dict(dwt=F16), b"dw is"),
    (dict(x=None), b"dw needs x"), (dict(xt=Q8), b"dw needs x"), (dict(xt=F16), b"dw needs x"), (dict(lddw=8), b"stride"),
    (dict(lddx=68), b"16 bytes"), (dict(nb=64), b"workspace"), (dict(ws=None), b"workspace"),
    (dict(h=None, dx=None, dw=None, db=None), b"no output")])
def test_gated_bwd(kw, word):
    refused("octsam_gated_bwd", changed(GATED_B, **kw), word)


def test_workspace_queries():
    lib = _lib.load()
    assert lib.octsam_rmsnorm_bwd_workspace(-1, 8) == 0 and lib.octsam_rmsnorm_bwd_workspace(4, 0) == 0
    assert lib.octsam_gated_bwd_workspace(4, 64, 32, 1) > lib.octsam_gated_bwd_workspace(4, 64, 32, 0) > 0
    assert lib.octsam_gated_bwd_workspace(-1, 64, 32, 0) == 0
    assert lib.octsam_gated_bwd_workspace(0, 64, 32, 1) >= 0  # (no rows: no division by a tile count of zero)


def test_empty_calls_do_nothing():
    lib = _lib.load()
    assert lib.octsam_quant8(*changed(QUANT, rows=0, x=None)) == 0
    assert lib.octsam_dequant8(*changed(DEQUANT, rows=0, q=None)) == 0
    assert lib.octsam_rmsnorm_fwd(*changed(NORM, rows=0, x=None)) == 0
    assert lib.octsam_gated_fwd(*changed(GATED, M=0, x=None)) == 0


def test_wrappers_refuse():
    """What the Python wrappers refuse before the C entry sees it. Host tensors are refused first; the shape and type
    checks are reached with the device check out of the way."""
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="device tensors"):
        kernels.quant8(x)
    with pytest.raises(ValueError, match="device tensors"):
        kernels.rmsnorm_fwd(x, torch.ones(64), 1e-6, x.clone())
    with pytest.raises(ValueError, match="device tensors"):
        kernels.gated_fwd(x.bfloat16(), torch.zeros(16, 64).bfloat16(), torch.zeros(4, 8).bfloat16())


def test_wrapper_checks(monkeypatch):
    monkeypatch.setattr(kernels, "_device_of", lambda *ts: torch.device("cpu"))

    def never(*a):
        raise AssertionError("launched")
    monkeypatch.setattr(_lib, "call_on", never)
    bf = torch.bfloat16
    x, w, h = torch.zeros(4, 64, dtype=bf), torch.zeros(32, 64, dtype=bf), torch.zeros(4, 16, dtype=bf)
    wn, q = torch.ones(64), kernels.q8_empty((4, 64), "cpu")
    cases = [
        (lambda: kernels.quant8(x.int()), "bf16, fp32 or fp16"),
        (lambda: kernels.quant8(x.t()), "contiguous"),
        (lambda: kernels.quant8(x[:1].expand(4, 64)), "overlap"),
        (lambda: kernels.quant8(torch.zeros(2, 4, 64)[:, ::2]), "contiguous"),
        (lambda: kernels.quant8(x, kernels.q8_empty((4, 32), "cpu")), "expected"),
        (lambda: kernels.quant8(x, (q[1], q[1])), "8-bit pair"),
        (lambda: kernels.dequant8(q[0], q[1][:, :1], x), "scales"),
        (lambda: kernels.rmsnorm_fwd(x, wn.bfloat16(), 1e-6, x), "fp32"),
        (lambda: kernels.rmsnorm_fwd(x, wn, 1e-6, x, sum_out=x), "residual"),
        (lambda: kernels.rmsnorm_fwd(x, wn, 1e-6, x, residual=x, sum_out=x.float()), "residual"),
        (lambda: kernels.rmsnorm_fwd(x, wn, 1e-6, x, residual=x[:3]), "expected"),
        (lambda: kernels.rmsnorm_fwd(x, wn, 1e-6, x, rstd=torch.zeros(3)), "rstd"),
        (lambda: kernels.rmsnorm_bwd(x, x, torch.zeros(4), wn, x, dres=x.float()), "dres"),
        (lambda: kernels.rmsnorm_bwd(x, x, torch.zeros(4), wn, x, dw=torch.zeros(63)), "dw"),
        (lambda: kernels.rmsnorm_bwd(x, (q[0][:3], q[1]), torch.zeros(4), wn, x), "expected"),
        (lambda: kernels.gated_fwd(x, w.half(), h), "one type"),
        (lambda: kernels.gated_fwd(x, w[:31], h), "2F"),
        (lambda: kernels.gated_fwd(x, w, h[:, :8]), "expected"),
        (lambda: kernels.gated_fwd(x, w, h, bias=torch.zeros(31)), "bias"),
        (lambda: kernels.gated_fwd(x, w, h, save=torch.zeros(4, 16, dtype=bf)), "expected"),
        (lambda: kernels.gated_fwd(x, w, h, save=torch.zeros(4, 32)), "8-bit pair"),
        (lambda: kernels.gated_fwd(x, w, h, save=kernels.q8_empty((4, 32), "cpu")), "8-bit pair"),
        (lambda: kernels.gated_bwd(h, torch.zeros(4, 32, dtype=bf), None, w, dw=w), "needs x"),
        (lambda: kernels.gated_bwd(h, torch.zeros(4, 32, dtype=bf), x, w.half(), dx=x), "expected"),
        (lambda: kernels.gated_bwd(h, torch.zeros(4, 32, dtype=bf), x, w, dx=x.float()), "dx and h"),
        (lambda: kernels.gated_bwd(h, torch.zeros(4, 32, dtype=bf), x.float(), w, dw=w), "8-bit pair"),
        (lambda: kernels.gated_bwd(h.float(), torch.zeros(4, 32, dtype=bf), x, w, dw=w), "bf16 or fp16"),
    ]
    for i, (f, word) in enumerate(cases):
        with pytest.raises(ValueError, match=word):
            f()
            pytest.fail(f"case {i} was taken")
