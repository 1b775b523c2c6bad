"""The AdamW entry points refuse bad arguments before they touch a device."""
import ctypes

import pytest

from fbcunn_b200 import build as fb_build
from fbcunn_b200 import capi


@pytest.fixture(scope="module")
def lib():
    fb_build.build()
    return capi.lib()


def _tensor(**kw):
    base = dict(param=4096, grad=8192, moment1=12288, moment2=16384, count=16)
    return capi.AdamwTensor(**{**base, **kw})


def _options(**kw):
    base = dict(beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1, steps=1 << 20, device=0)
    return capi.AdamwOptions(**{**base, **kw})


def _create(lib, tensors, options):
    out = ctypes.c_void_p()
    array = (capi.AdamwTensor * max(1, len(tensors)))(*tensors)
    rc = lib.fbfftconv_adamw_create(array, len(tensors), ctypes.byref(options), ctypes.byref(out))
    assert not out.value
    return rc


@pytest.mark.parametrize("bad,message", [
    (dict(count=-1), "negative"), (dict(param_type=3), "type"), (dict(grad_type=-1), "type"), (dict(param=None), "null"),
    (dict(moment2=None), "null"), (dict(scale1=20480), "8 bits"), (dict(master=24576), "master"), (dict(grad=8193), "aligned"),
    (dict(param=4098), "aligned"), (dict(moment1=12289), "aligned"), (dict(moment1=4096), "share memory"),
    (dict(moment2=4096 + 60), "share memory"), (dict(count=(1 << 38) + 1), "2^38")])
def test_bad_tensors(lib, bad, message):
    assert _create(lib, [_tensor(**bad)], _options()) in (capi.ERR_INVALID_ARGUMENT, capi.ERR_UNSUPPORTED_SIZE)
    assert message in capi.last_error()


@pytest.mark.parametrize("bad", [dict(beta1=1.0), dict(beta1=-0.1), dict(beta2=float("nan")), dict(eps=-1e-8),
                                 dict(eps=float("inf")), dict(weight_decay=-1.0), dict(steps=None), dict(steps=(1 << 20) + 4)])
def test_bad_options(lib, bad):
    assert _create(lib, [_tensor()], _options(**bad)) == capi.ERR_INVALID_ARGUMENT


def test_null_arguments(lib):
    out = ctypes.c_void_p()
    assert lib.fbfftconv_adamw_create(None, 1, ctypes.byref(_options()), ctypes.byref(out)) == capi.ERR_INVALID_ARGUMENT
    assert lib.fbfftconv_adamw_create(None, 0, None, ctypes.byref(out)) == capi.ERR_INVALID_ARGUMENT
    assert lib.fbfftconv_adamw_create(None, 0, ctypes.byref(_options()), None) == capi.ERR_INVALID_ARGUMENT
    assert lib.fbfftconv_adamw_step(None, 1e-3, 1.0, None, None) == capi.ERR_INVALID_ARGUMENT
    assert lib.fbfftconv_adamw_set_gradients(None, None, 0) == capi.ERR_INVALID_ARGUMENT
    assert lib.fbfftconv_adamw_destroy(None) == capi.OK


def test_tensors_that_touch_do_not_overlap(lib):
    """Neighbours in one flat array are no overlap: the call gets past the checks, to the device's."""
    tensors = [_tensor(), _tensor(param=4096 + 64, grad=8192 + 64, moment1=12288 + 64, moment2=16384 + 64)]
    rc = _create(lib, tensors, _options())
    assert "share memory" not in capi.last_error() and rc in (capi.ERR_CUDA, capi.ERR_INVALID_ARGUMENT)


@pytest.mark.parametrize("grad,message", [
    (4096, "gradient"), (4096 + 60, "gradient"), (4096 - 60, "gradient"), (12288 + 32, "gradient"), (16384 + 60, "gradient"),
    ((1 << 20) - 60, "gradient"), ((1 << 20) + 12, "gradient"), (4096 + 64, None), (4096 - 64, None), ((1 << 20) + 16, None)])
def test_gradients_apart_from_what_is_written(lib, grad, message):
    """A gradient that lies in a parameter, a moment or the count is refused, one beside them is not."""
    rc = _create(lib, [_tensor(grad=grad)], _options())
    if message:
        assert rc == capi.ERR_INVALID_ARGUMENT and "share memory" in capi.last_error() and message in capi.last_error()
    else:
        assert "share memory" not in capi.last_error()


def test_counts_apart_from_what_is_written(lib):
    assert _create(lib, [_tensor()], _options(steps=4096 + 56)) == capi.ERR_INVALID_ARGUMENT
    assert "share memory" in capi.last_error()


def test_tensors_may_share_a_gradient(lib):
    tensors = [_tensor(), _tensor(param=4096 + 64, moment1=12288 + 64, moment2=16384 + 64)]
    _create(lib, tensors, _options())
    assert "share memory" not in capi.last_error()
