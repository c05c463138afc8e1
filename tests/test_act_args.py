"""The activation codes of the C entries: SiLU belongs to the gated unit, and the products and the layer norm, which do not
have it, refuse it (and unknown codes) on the host instead of leaving the activation out. Pointers are never dereferenced."""
import ctypes

import pytest

from dilabhelmholtzoct_amd import _lib

P = 1 << 20  # a 16-B aligned address


def refused(name, *args):
    lib = _lib.load()
    assert getattr(lib, name)(*args) != 0
    assert b"activation" in lib.octsam_last_error(), lib.octsam_last_error()


@pytest.mark.parametrize("act", [_lib.ACT_SILU, 4, -1])
def test_unknown_activation_is_refused(act):
    for name in ("octsam_gemm", "octsam_gemm_f16"):
        args = _lib.GemmArgs(A=P, B=P, C=P, M=64, N=64, K=64, batch=1, lda=64, ldb=64, ldc=64, ldr=64, alpha=1.0, act=act,
                             a_rep=1, b_rep=1, r_rep=1)
        refused(name, ctypes.byref(args), None)
    refused("octsam_layernorm_fwd", P, 0, None, 4, 256, P, P, 1e-6, P, 0, None, act, None, None, None)
    refused("octsam_layernorm_bwd", P, 0, P, 0, P, P, P, P, act, 4, 256, P, 0, 0.0, None, P, P, 8, None)
