"""What the decoder-layer operators' handles do after free(), and host operands of the wrong kind, on a host without a GPU:
the library refuses arguments ahead of its context (here there is none, which it reports once they pass)."""

import ctypes

import pytest

from transmuter_amd import _lib, serving
from transmuter_amd._lib import TmhArgumentError
from transmuter_amd.device import DeviceTensor


class _NoContext:
    """A context whose tensors have an address that no call gets to use."""

    handle = None

    def empty(self, shape, dtype):
        return DeviceTensor(self, ctypes.c_void_p(4096), shape, dtype, 0)

    def free(self, ptr):
        pass

    def check(self, status):
        _lib.check(status)


CTX = _NoContext()


def _t(dtype, *shape):
    return CTX.empty(shape, dtype)


@pytest.mark.parametrize("call", [lambda c: c.append(_t("f16", 2, 256), 2, _t("s64", 2)),
                                  lambda c: c.attend(_t("f16", 2, 128), _t("s32", 2, 4), _t("s32", 2))])
def test_a_freed_cache_is_refused(call):
    cache = serving.PagedCache(CTX, 4, 16, 1, 64)
    with pytest.raises(TmhArgumentError, match="context is NULL"):
        call(cache)
    cache.free()
    for _ in range(2):
        with pytest.raises(TmhArgumentError, match="k and v must not be NULL"):
            call(cache)
        cache.free()  # (once more is nothing)


def test_a_freed_weight_is_refused():
    weight = serving.Fp8Weight(CTX, None, 128, 64)
    weight.free()
    with pytest.raises(TmhArgumentError, match="weight is NULL"):
        serving.matmul_fp8(serving.Rows8(_t("f8_e4m3fn", 2, 128), _t("f32", 1, 2)), weight)
    with pytest.raises(TmhArgumentError, match="weight is NULL"):
        weight.device_bytes()


def _freed(dtype, *shape):
    t = _t(dtype, *shape)
    t.free()
    return t


@pytest.mark.parametrize("call", [
    lambda: serving.rms_norm(_t("f16", 2, 128), _t("f16", 128), _freed("f16", 2, 128)),
    lambda: serving.rms_norm(_t("f16", 2, 128), _t("f16", 128), _t("f16", 2, 128), out=serving.Norm(None, None, _freed("f16", 2, 128))),
    lambda: serving.rms_norm(_t("f16", 2, 128), _t("f16", 128), y=True, out=serving.Norm(_freed("f16", 2, 128), None, None)),
    lambda: serving.matmul_fp8(serving.Rows8(_t("f8_e4m3fn", 2, 128), _t("f32", 1, 2)), serving.Fp8Weight(CTX, None, 128, 64),
                               _freed("f16", 64)),
])
def test_a_freed_operand_is_not_left_out(call):
    """A residual, bias or answer that was freed is refused, not taken for one that was not given."""
    with pytest.raises(TmhArgumentError, match="has been freed"):
        call()
