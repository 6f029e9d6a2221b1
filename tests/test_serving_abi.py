"""Refusals of the decoder-layer operators on a host without a GPU: arguments are checked before the context is
(here there is none, which is what the calls report once their arguments pass)."""

import ctypes
import math

import numpy as np
import pytest

import serving_plain as plain
from transmuter_amd import _lib
from transmuter_amd._lib import PagedCacheDesc, lib

P = 4096  # a device address that no call here gets to use


def _norm(**kw):
    a = dict(x=P, ldx=64, r=None, ldr=64, dtype=_lib.F16, t=2, n=64, gamma=P, gdt=_lib.F16, eps=1e-6, sum=None, lds=64,
             y=P, ldy=64, q=None, ldq=64, scales=None)
    a.update(kw)
    return lib().tmh_rms_norm(None, a["x"], a["ldx"], a["r"], a["ldr"], a["dtype"], a["t"], a["n"], a["gamma"], a["gdt"],
                              a["eps"], a["sum"], a["lds"], a["y"], a["ldy"], a["q"], a["ldq"], a["scales"], None)


@pytest.mark.parametrize("kw,needle", [
    (dict(), b"context is NULL"),
    (dict(dtype=_lib.S8), b"f32, f16 or bf16 rows"),
    (dict(dtype=_lib.F8E4M3), b"got f8_e4m3fn"),
    (dict(gdt=_lib.S32), b"gamma must be"),
    (dict(t=-1), b"-1 rows"),
    (dict(n=0), b"0 columns"),
    (dict(eps=-1.0), b"eps"),
    (dict(eps=math.nan), b"eps"),
    (dict(y=None), b"no output"),
    (dict(q=P), b"go together"),
    (dict(scales=P), b"go together"),
    (dict(ldx=63), b"leading dimensions"),
    (dict(r=P, ldr=63), b"leading dimensions"),
    (dict(sum=P, lds=63), b"leading dimensions"),
    (dict(ldy=63), b"leading dimensions"),
    (dict(q=P, scales=P, ldq=63), b"leading dimensions"),
])
def test_norm_refusals(kw, needle):
    assert _norm(**kw) == _lib.ERR_INVALID
    assert needle in lib().tmh_last_error(None)


@pytest.mark.parametrize("kw,needle", [
    (dict(), b"context is NULL"),
    (dict(dtype=_lib.U8), b"f32, f16 or bf16"),
    (dict(t=-1), b"-1 rows"),
    (dict(n=0), b"0 columns"),
    (dict(ldx=63), b"leading dimensions"),
    (dict(gate=P, ldg=63), b"leading dimensions"),
    (dict(ldq=63), b"leading dimensions"),
])
def test_quantize_refusals(kw, needle):
    a = dict(ldx=64, gate=None, ldg=64, dtype=_lib.BF16, t=2, n=64, ldq=64)
    a.update(kw)
    st = lib().tmh_quantize_rows(None, P, a["ldx"], a["gate"], a["ldg"], a["dtype"], a["t"], a["n"], P, a["ldq"], P, None)
    assert st == _lib.ERR_INVALID
    assert needle in lib().tmh_last_error(None)


def test_weight_and_product_refusals():
    out = ctypes.c_void_p(1)
    prepare = lib().tmh_fp8_weight_prepare
    assert prepare(None, P, P, 128, 128, None, None) == _lib.ERR_INVALID
    for k, n, status in ((0, 1, _lib.ERR_INVALID), (1, 0, _lib.ERR_INVALID), (2 ** 22 + 1, 1, _lib.ERR_UNSUPPORTED),
                         (1, 2 ** 22 + 1, _lib.ERR_UNSUPPORTED), (128, 128, _lib.ERR_INVALID)):
        assert prepare(None, P, P, k, n, None, ctypes.byref(out)) == status
        assert out.value is None
    assert b"context is NULL" in lib().tmh_last_error(None)
    assert lib().tmh_matmul_fp8(None, None, P, 1, 128, P, None, 0, P, _lib.F16, 128, None) == _lib.ERR_INVALID
    assert b"weight is NULL" in lib().tmh_last_error(None)
    assert lib().tmh_fp8_weight_info(None, None, None, None) == _lib.ERR_INVALID
    lib().tmh_fp8_weight_free(None)


def _cache(**kw):
    a = dict(k=P, v=P, dtype=_lib.F16, kv_heads=2, head_dim=64, page_size=16, pages=8, page_stride=2048, token_stride=128,
             head_stride=64)
    a.update(kw)
    return PagedCacheDesc(**a)


BAD_CACHES = [
    (dict(dtype=_lib.S8), _lib.ERR_INVALID, b"holds f32, f16 or bf16"),
    (dict(kv_heads=0), _lib.ERR_INVALID, b"at least 1"),
    (dict(page_size=0), _lib.ERR_INVALID, b"at least 1"),
    (dict(pages=0), _lib.ERR_INVALID, b"at least 1"),
    (dict(head_dim=0), _lib.ERR_UNSUPPORTED, b"head_dim"),
    (dict(head_dim=60), _lib.ERR_UNSUPPORTED, b"head_dim"),
    (dict(head_dim=264), _lib.ERR_UNSUPPORTED, b"head_dim"),
    (dict(pages=2 ** 27), _lib.ERR_UNSUPPORTED, b"2^31"),
    (dict(pages=2 ** 40), _lib.ERR_UNSUPPORTED, b"2^31"),
    (dict(page_size=3, pages=715827883), _lib.ERR_UNSUPPORTED, b"2^31"),
    (dict(k=None), _lib.ERR_INVALID, b"must not be NULL"),
    (dict(v=None), _lib.ERR_INVALID, b"must not be NULL"),
    (dict(k=P + 8), _lib.ERR_UNSUPPORTED, b"16 bytes"),
    (dict(token_stride=132), _lib.ERR_UNSUPPORTED, b"16 bytes"),
    (dict(head_stride=-64), _lib.ERR_INVALID, b"negative"),
]


def _append(cache, **kw):
    a = dict(q=P, ldq=512, k=P, ldk=512, v=P, ldv=512, t=2, heads=4, table=_lib.F32, most=16, rotary=64, slots=P, qo=P + 4096,
             ldqo=256)
    a.update(kw)
    return lib().tmh_paged_append(None, a["q"], a["ldq"], a["k"], a["ldk"], a["v"], a["ldv"], a["t"], a["heads"], P, P, P,
                                  a["table"], a["most"], a["rotary"], 0, a["slots"],
                                  ctypes.byref(cache) if cache is not None else None, a["qo"], a["ldqo"], None)


def _attend(cache, **kw):
    a = dict(q=P, ldq=256, b=2, heads=4, table=P, most=4, lengths=P, scale=0.125, window=0, y=P, ldy=256)
    a.update(kw)
    return lib().tmh_paged_attention(None, a["q"], a["ldq"], a["b"], a["heads"],
                                     ctypes.byref(cache) if cache is not None else None, a["table"], a["most"], a["lengths"],
                                     a["scale"], a["window"], a["y"], a["ldy"], None)


@pytest.mark.parametrize("call", [_append, _attend])
@pytest.mark.parametrize("kw,status,needle", BAD_CACHES)
def test_cache_refusals(call, kw, status, needle):
    assert call(_cache(**kw)) == status
    assert needle in lib().tmh_last_error(None)


@pytest.mark.parametrize("call", [_append, _attend])
def test_no_cache_and_no_context(call):
    assert call(None) == _lib.ERR_INVALID and b"cache is NULL" in lib().tmh_last_error(None)
    assert call(_cache()) == _lib.ERR_INVALID and b"context is NULL" in lib().tmh_last_error(None)
    # The largest cache: pages * page_size one below 2^31 for a page size that divides it, or just below.
    assert call(_cache(pages=2 ** 27 - 1)) == _lib.ERR_INVALID and b"context is NULL" in lib().tmh_last_error(None)
    assert call(_cache(page_size=3, pages=715827882)) == _lib.ERR_INVALID
    assert b"context is NULL" in lib().tmh_last_error(None)


@pytest.mark.parametrize("kw,needle", [
    (dict(t=-1), b"-1 tokens"),
    (dict(heads=-1), b"query heads"),
    (dict(rotary=66), b"rotary_dim"),
    (dict(rotary=7), b"rotary_dim"),
    (dict(rotary=-2), b"rotary_dim"),
    (dict(table=_lib.S64), b"rotary tables"),
    (dict(most=0), b"no positions"),
    (dict(ldk=127), b"leading dimensions"),
    (dict(ldv=127), b"leading dimensions"),
    (dict(ldq=255), b"leading dimensions"),
    (dict(ldqo=255), b"leading dimensions"),
])
def test_append_refusals(kw, needle):
    assert _append(_cache(), **kw) == _lib.ERR_INVALID
    assert needle in lib().tmh_last_error(None)


@pytest.mark.parametrize("kw,status,needle", [
    (dict(heads=3), _lib.ERR_INVALID, b"no multiple"),
    (dict(heads=0), _lib.ERR_INVALID, b"no multiple"),
    (dict(b=-1), _lib.ERR_INVALID, b"sequences"),
    (dict(b=65536), _lib.ERR_INVALID, b"sequences"),
    (dict(most=-1), _lib.ERR_INVALID, b"negative"),
    (dict(window=-1), _lib.ERR_INVALID, b"negative"),
    (dict(scale=math.nan), _lib.ERR_INVALID, b"NaN"),
    (dict(ldq=255), _lib.ERR_INVALID, b"leading dimensions"),
    (dict(ldy=255), _lib.ERR_INVALID, b"leading dimensions"),
    (dict(most=2 ** 27), _lib.ERR_UNSUPPORTED, b"2^31"),
])
def test_attention_refusals(kw, status, needle):
    assert _attend(_cache(), **kw) == status
    assert needle in lib().tmh_last_error(None)


def test_plain_e4m3():
    """The tests' own e4m3: every number comes back, and halfway values round to even."""
    bits = np.array([b for b in range(256) if b & 127 != 127], dtype=np.uint8)
    assert np.array_equal(plain.f8_bits(plain.F8[bits]), bits)
    pos = plain.F8[:127]
    halfway = (pos[:-1] + pos[1:]) / 2
    assert np.array_equal(plain.f8_bits(halfway), [i if i % 2 == 0 else i + 1 for i in range(126)])
    assert plain.F8[126] == 448 and plain.F8[1] == 2.0 ** -9
