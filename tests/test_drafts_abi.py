"""Refusals of the operators of a drafted step on a host without a GPU: arguments are checked before the context is (here
there is none, which is what the calls report once their arguments pass)."""

import ctypes
import math

import pytest

from test_serving_abi import BAD_CACHES, P, _cache
from transmuter_amd import _lib
from transmuter_amd._lib import lib


def _append_norm(cache, **kw):
    a = dict(q=P, ldq=512, k=P, ldk=512, v=P, ldv=512, t=2, heads=4, qg=P, kg=P, gdt=_lib.F16, eps=1e-6, table=_lib.F32, most=16,
             rotary=64, slots=P, qo=P + 4096, ldqo=256)
    a.update(kw)
    return lib().tmh_paged_append_norm(None, a["q"], a["ldq"], a["k"], a["ldk"], a["v"], a["ldv"], a["t"], a["heads"], a["qg"], a["kg"],
                                       a["gdt"], a["eps"], P, P, P, a["table"], a["most"], a["rotary"], 0, a["slots"],
                                       ctypes.byref(cache) if cache is not None else None, a["qo"], a["ldqo"], None)


def _tree(cache, **kw):
    a = dict(q=P, ldq=256, t=6, heads=4, table=P, b=2, most=4, lengths=P, starts=P, mask=P, words=1, scale=0.125, window=0, y=P, ldy=256)
    a.update(kw)
    return lib().tmh_paged_tree_attention(None, a["q"], a["ldq"], a["t"], a["heads"], ctypes.byref(cache) if cache is not None else None,
                                          a["table"], a["b"], a["most"], a["lengths"], a["starts"], a["mask"], a["words"], a["scale"],
                                          a["window"], a["y"], a["ldy"], None)


def _sample(**kw):
    a = dict(x=P, ld=100, dtype=_lib.F32, t=2, v=100, temperature=P, k=P, p=P, m=P, u=P, tokens=P)
    a.update(kw)
    return lib().tmh_sample(None, a["x"], a["ld"], a["dtype"], a["t"], a["v"], a["temperature"], a["k"], a["p"], a["m"], a["u"],
                            a["tokens"], None)


@pytest.mark.parametrize("kw,status,needle", BAD_CACHES)
def test_bad_caches(kw, status, needle):
    for call in (_append_norm, _tree):
        assert call(_cache(**kw)) == status
        assert needle in lib().tmh_last_error(None)


@pytest.mark.parametrize("kw,status,needle", [
    (dict(), _lib.ERR_INVALID, b"context is NULL"),
    (dict(kg=None), _lib.ERR_INVALID, b"context is NULL"),
    (dict(qg=None), _lib.ERR_INVALID, b"context is NULL"),
    (dict(qg=None, kg=None), _lib.ERR_INVALID, b"no gamma"),
    (dict(gdt=_lib.S32), _lib.ERR_INVALID, b"gammas must be"),
    (dict(eps=-1.0), _lib.ERR_INVALID, b"eps"),
    (dict(eps=math.nan), _lib.ERR_INVALID, b"eps"),
    (dict(t=-1), _lib.ERR_INVALID, b"-1 tokens"),
    (dict(heads=-1), _lib.ERR_INVALID, b"query heads"),
    (dict(rotary=63), _lib.ERR_INVALID, b"rotary_dim"),
    (dict(rotary=66), _lib.ERR_INVALID, b"rotary_dim"),
    (dict(table=_lib.S8), _lib.ERR_INVALID, b"rotary tables"),
    (dict(most=0), _lib.ERR_INVALID, b"no positions"),
    (dict(ldk=127), _lib.ERR_INVALID, b"leading dimensions"),
    (dict(ldqo=255), _lib.ERR_INVALID, b"leading dimensions"),
])
def test_append_norm_refusals(kw, status, needle):
    assert _append_norm(_cache(), **kw) == status
    assert needle in lib().tmh_last_error(None)


@pytest.mark.parametrize("kw,status,needle", [
    (dict(), _lib.ERR_INVALID, b"context is NULL"),
    (dict(mask=None, words=0), _lib.ERR_INVALID, b"context is NULL"),
    (dict(heads=3), _lib.ERR_INVALID, b"no multiple"),
    (dict(heads=0), _lib.ERR_INVALID, b"no multiple"),
    (dict(heads=2 ** 21, ldq=2 ** 27, ldy=2 ** 27), _lib.ERR_UNSUPPORTED, b"2^20"),
    (dict(b=-1), _lib.ERR_INVALID, b"65535"),
    (dict(b=65536), _lib.ERR_INVALID, b"65535"),
    (dict(t=-1), _lib.ERR_INVALID, b"-1 rows"),
    (dict(t=2 ** 31), _lib.ERR_INVALID, b"rows"),
    (dict(most=-1), _lib.ERR_INVALID, b"negative"),
    (dict(window=-1), _lib.ERR_INVALID, b"negative"),
    (dict(words=0), _lib.ERR_INVALID, b"words"),
    (dict(words=-1), _lib.ERR_INVALID, b"words"),
    (dict(words=2 ** 21), _lib.ERR_INVALID, b"words"),
    (dict(scale=math.nan), _lib.ERR_INVALID, b"NaN"),
    (dict(ldq=255), _lib.ERR_INVALID, b"leading dimensions"),
    (dict(ldy=255), _lib.ERR_INVALID, b"leading dimensions"),
    (dict(most=2 ** 27), _lib.ERR_UNSUPPORTED, b"2^31"),
])
def test_tree_refusals(kw, status, needle):
    assert _tree(_cache(), **kw) == status
    assert needle in lib().tmh_last_error(None)


@pytest.mark.parametrize("kw,status,needle", [
    (dict(), _lib.ERR_INVALID, b"context is NULL"),
    (dict(temperature=None, k=None, p=None, m=None), _lib.ERR_INVALID, b"context is NULL"),
    (dict(dtype=_lib.S32), _lib.ERR_INVALID, b"logits"),
    (dict(t=-1), _lib.ERR_INVALID, b"-1 rows"),
    (dict(t=2 ** 31), _lib.ERR_INVALID, b"rows"),
    (dict(v=0), _lib.ERR_INVALID, b"vocabulary"),
    (dict(v=2 ** 20, ld=2 ** 20), _lib.ERR_UNSUPPORTED, b"2^20"),
    (dict(ld=99), _lib.ERR_INVALID, b"leading dimension"),
])
def test_sample_refusals(kw, status, needle):
    assert _sample(**kw) == status
    assert needle in lib().tmh_last_error(None)
