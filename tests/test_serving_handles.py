"""What the decoder-layer operators' handles do after free(), and host operands of the wrong kind, on a host without a GPU:
the library refuses arguments ahead of its context (here there is none, which it reports once they pass)."""

import ctypes

import numpy as np
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


class _Host(_NoContext):
    """A context that keeps what is put."""

    def put(self, array, dtype=None):
        t = self.empty(np.shape(array), dtype or "f32")
        self.host = array if dtype == "f8_e4m3fn" else self.host
        return t


@pytest.mark.parametrize("b", [np.full((4, 128), 1.5, np.float32), np.ones((4, 128), np.float16), np.ones((4, 128), bool),
                               np.full((4, 128), 256), np.full((4, 128), -1)])
def test_a_weight_of_values_is_not_taken_for_bytes(b):
    with pytest.raises(TmhArgumentError, match="array of f8_e4m3fn bytes"):
        serving.Fp8Weight.prepare(_Host(), b, np.ones((1, 1), np.float32))


@pytest.mark.parametrize("dtype", [np.uint8, np.int8, np.int64])
def test_a_weight_of_bytes(dtype):
    """Bytes in any integer type that holds them reach the library as they are."""
    host = np.arange(4 * 128).reshape(4, 128) % 256
    ctx = _Host()
    with pytest.raises(TmhArgumentError, match="context is NULL"):
        serving.Fp8Weight.prepare(ctx, host.astype(dtype), np.ones((1, 1), np.float32))
    assert ctx.host.dtype == np.uint8 and np.array_equal(ctx.host, host)


@pytest.mark.parametrize("tables", [(None, True), (True, None)])
def test_half_the_rotary_tables(tables):
    """One table without the other is refused, not a step without rotary positions."""
    cache = serving.PagedCache(CTX, 4, 16, 1, 64)
    cos, sin = (_t("f32", 100, 32) if given else None for given in tables)
    with pytest.raises(TmhArgumentError, match="tables cos and sin"):
        cache.append(_t("f16", 2, 256), 2, _t("s64", 2), _t("s64", 2), cos, sin)
