"""Where attention of drafted steps stops taking wide tables, on a host without a GPU (test_drafts_abi.py has the other refusals): its workgroups
count tokens in 32 bits, and up to two units past their last."""

import pytest

from test_drafts_abi import _tree
from test_serving_abi import _cache
from transmuter_amd import _lib
from transmuter_amd._lib import lib

MOST = 2 ** 31 - 1024


@pytest.mark.parametrize("page", [1, 16, 20, 1024, 2 ** 20])
def test_widest_table(page):
    cache = dict(page_size=page, pages=16)
    assert _tree(_cache(**cache), most=MOST // page) == _lib.ERR_INVALID  # (all that is wrong is that there is no context)
    assert b"context is NULL" in lib().tmh_last_error(None)
    for more in (MOST // page + 1, (2 ** 31 - 1) // page, 2 ** 31 // page, 2 ** 62):
        if more > MOST // page:
            assert _tree(_cache(**cache), most=more) == _lib.ERR_UNSUPPORTED
            assert b"2^31 - 1024" in lib().tmh_last_error(None)
