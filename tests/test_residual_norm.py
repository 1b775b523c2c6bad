"""The residual-norm entry points refuse bad arguments before they touch a device."""
import ctypes

import pytest

from fbcunn_b200 import build as fb_build
from fbcunn_b200 import capi


@pytest.fixture(scope="module")
def lib():
    fb_build.build()
    return capi.lib()


def _desc(**kw):
    base = dict(rows=4, gate_rows=4, channels=64, type=capi.BFLOAT16, residual_type=capi.FLOAT32, post=capi.NORM_RMS,
                pre=capi.NORM_LAYER, gate=capi.GATE_SIGMOID, eps=1e-6, residual_scale=1.0, branch_scale=1.0, device=0)
    return capi.NormDesc(**{**base, **kw})


BAD = [dict(rows=-1), dict(channels=0), dict(channels=16385), dict(type=3), dict(residual_type=capi.FLOAT16),
       dict(type=capi.FLOAT32, residual_type=capi.BFLOAT16), dict(post=3), dict(pre=-1), dict(post=0, pre=0), dict(gate=3),
       dict(gate_rows=3), dict(gate_rows=0), dict(gate_rows=-2), dict(eps=-1.0), dict(eps=float("nan")),
       dict(residual_scale=float("inf"))]


@pytest.mark.parametrize("bad", range(len(BAD)))
def test_bad_descriptors(lib, bad):
    desc = _desc(**BAD[bad])
    refused = (capi.ERR_INVALID_ARGUMENT, capi.ERR_UNSUPPORTED_SIZE)
    assert lib.fbfftconv_residual_norm(ctypes.byref(desc), *[4096] * 10, None) in refused
    assert lib.fbfftconv_residual_norm_backward(ctypes.byref(desc), *[4096] * 16, 1.0, 0, 4096, 1 << 20, None) in refused
    assert lib.fbfftconv_residual_norm_workspace_bytes(ctypes.byref(desc)) == 0


def test_null_and_misaligned_pointers(lib):
    d = ctypes.byref(_desc())
    assert lib.fbfftconv_residual_norm(None, *[4096] * 10, None) == capi.ERR_INVALID_ARGUMENT
    for i in (1, 2, 3, 5, 7, 8):  # r, gate, weights, outputs
        args = [4096] * 10
        args[i] = None
        assert lib.fbfftconv_residual_norm(d, *args, None) == capi.ERR_INVALID_ARGUMENT
        args[i] = 4097
        assert lib.fbfftconv_residual_norm(d, *args, None) == capi.ERR_INVALID_ARGUMENT
        assert "aligned" in capi.last_error()
    assert lib.fbfftconv_residual_norm(d, None, *[4096] * 9, None) == capi.ERR_INVALID_ARGUMENT  # a gate, but no block
    assert lib.fbfftconv_residual_norm(d, *[4096] * 9, 4100, None) == capi.ERR_INVALID_ARGUMENT  # stats
    assert lib.fbfftconv_residual_norm_backward(d, *[4096] * 16, float("nan"), 0, 4096, 1 << 20, None) == capi.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("field", ["u_stride", "r_stride", "gate_stride"])
@pytest.mark.parametrize("stride", [-1, -64, -(1 << 32) + 64, -(1 << 63)])
def test_negative_strides(lib, field, stride):
    """Also those that would be a sound one in 32 bits."""
    d = ctypes.byref(_desc(**{field: stride}))
    assert lib.fbfftconv_residual_norm(d, *[4096] * 10, None) == capi.ERR_INVALID_ARGUMENT
    assert "negative stride" in capi.last_error()
    assert lib.fbfftconv_residual_norm_backward(d, *[4096] * 16, 1.0, 0, 4096, 1 << 20, None) == capi.ERR_INVALID_ARGUMENT
    assert "negative stride" in capi.last_error()
