"""Answers' memory that the caller gives (out=) and operands of another shape or type than the operator's, on a
host without a GPU: both are refused before the library is called."""

import ctypes

import pytest

from transmuter_amd import serving
from transmuter_amd._lib import TmhArgumentError
from transmuter_amd.device import DeviceTensor


class _NoDevice:
    """A context whose tensors have no memory; reaching the library with it fails the test."""

    handle = None

    def empty(self, shape, dtype):
        return DeviceTensor(self, ctypes.c_void_p(None), shape, dtype, 0)

    def check(self, status):
        raise AssertionError(f"the call reached the library ({status})")


CTX = _NoDevice()


def _t(dtype, *shape):
    return CTX.empty(shape, dtype)


def _rows8(rows, n, q="f8_e4m3fn", s="f32", blocks=None):
    return serving.Rows8(_t(q, rows, n), _t(s, -(-n // 128) if blocks is None else blocks, rows))


@pytest.mark.parametrize("out,asked", [
    (serving.Norm(_t("f16", 3, 200), None, None), dict(y=True, rows=False)),
    (serving.Norm(_t("f32", 2, 200), None, None), dict(y=True, rows=False)),
    (serving.Norm(None, _rows8(2, 201), None), {}),
    (serving.Norm(None, _rows8(2, 200, q="u8"), None), {}),
    (serving.Norm(None, _rows8(2, 200, blocks=1), None), {}),
    (serving.Norm(None, _rows8(2, 200, s="f16"), None), {}),
    (serving.Norm(None, None, _t("bf16", 2, 200)), dict(residual=_t("f16", 2, 200))),
    (serving.Norm(None, None, _t("f16", 400)), dict(residual=_t("f16", 2, 200))),
])
def test_norm_out(out, asked):
    with pytest.raises(TmhArgumentError, match="out must be"):
        serving.rms_norm(_t("f16", 2, 200), _t("f16", 200), out=out, **asked)


def test_norm_operands():
    with pytest.raises(TmhArgumentError, match="gamma must be"):
        serving.rms_norm(_t("f16", 2, 200), _t("f16", 2, 200))
    with pytest.raises(TmhArgumentError, match="residual must be"):
        serving.rms_norm(_t("f16", 2, 200), _t("f16", 200), _t("f16", 200, 2))
    with pytest.raises(TmhArgumentError, match="got s32"):
        serving.rms_norm(_t("s32", 2, 200), _t("f16", 200))
    with pytest.raises(TmhArgumentError, match="scalar"):
        serving.quantize_rows(_t("f16"))


@pytest.mark.parametrize("out", [_rows8(2, 201), _rows8(3, 200), _rows8(2, 200, q="s8"), _rows8(2, 200, blocks=3)])
def test_quantize_out(out):
    with pytest.raises(TmhArgumentError, match="out must be"):
        serving.quantize_rows(_t("bf16", 2, 200), out=out)
    with pytest.raises(TmhArgumentError, match="out must be"):
        serving.quantize_swiglu(_t("bf16", 2, 400), out=out)


def test_swiglu_halves():
    with pytest.raises(TmhArgumentError, match="two equal halves"):
        serving.quantize_swiglu(_t("f32", 2, 401))


@pytest.mark.parametrize("a,kw,needle", [
    (_rows8(2, 200), dict(out=_t("f32", 2, 70)), "out must be"),
    (_rows8(2, 200), dict(out=_t("f16", 2, 72)), "out must be"),
    (_rows8(2, 201), {}, "K is 200"),
    (_rows8(2, 200, blocks=1), {}, "scales"),
    (_rows8(2, 200, q="u8"), {}, "must be f8_e4m3fn"),
    (_rows8(2, 200), dict(bias=_t("f16", 2, 70)), "bias must be"),
    (_rows8(2, 200), dict(y_type="s32"), "y must be"),
])
def test_product_out_and_operands(a, kw, needle):
    with pytest.raises(TmhArgumentError, match=needle):
        serving.matmul_fp8(a, serving.Fp8Weight(CTX, None, 200, 70), **kw)


@pytest.mark.parametrize("out", [_t("f32", 2, 128), _t("f16", 2, 64), _t("f16", 3, 128)])
def test_cache_out(out):
    cache = serving.PagedCache(CTX, 4, 16, 1, 64)
    with pytest.raises(TmhArgumentError, match="out must be"):
        cache.append(_t("f16", 2, 256), 2, _t("s64", 2), out=out)
    with pytest.raises(TmhArgumentError, match="out must be"):
        cache.attend(_t("f16", 2, 128), _t("s32", 2, 4), _t("s32", 2), out=out)


def test_cache_operands():
    cache = serving.PagedCache(CTX, 4, 16, 1, 64)
    tables = _t("f32", 100, 32)
    for call in (lambda: cache.append(_t("f16", 2, 255), 2, _t("s64", 2)),
                 lambda: cache.append(_t("bf16", 2, 256), 2, _t("s64", 2)),
                 lambda: cache.append(_t("f16", 2, 256), 2, _t("s32", 2)),
                 lambda: cache.append(_t("f16", 2, 256), 2, _t("s64", 3)),
                 lambda: cache.append(_t("f16", 2, 256), 2, _t("s64", 2), None, tables, tables),
                 lambda: cache.append(_t("f16", 2, 256), 2, _t("s64", 2), _t("s64", 2), tables, _t("f32", 99, 32)),
                 lambda: cache.append(_t("f16", 2, 256), 2, _t("s64", 2), _t("s32", 2), tables, tables),
                 lambda: cache.attend(_t("f16", 2, 100), _t("s32", 2, 4), _t("s32", 2)),
                 lambda: cache.attend(_t("f16", 2, 128), _t("s64", 2, 4), _t("s32", 2)),
                 lambda: cache.attend(_t("f16", 2, 128), _t("s32", 3, 4), _t("s32", 2)),
                 lambda: cache.attend(_t("f16", 2, 128), _t("s32", 2, 4), _t("s32", 2, 1))):
        with pytest.raises(TmhArgumentError):
            call()


@pytest.mark.parametrize("kw", [dict(order="rows"), dict(dtype="s8"), dict(pages=0), dict(head_dim=0)])
def test_cache_refuses(kw):
    with pytest.raises(TmhArgumentError):
        serving.PagedCache(CTX, **{**dict(pages=4, page_size=16, kv_heads=1, head_dim=64), **kw})
