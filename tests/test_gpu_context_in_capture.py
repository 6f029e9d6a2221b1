"""A context made while another one's stream is being captured, and its first attention call."""

import ctypes

import numpy as np
import pytest

from transmuter_amd import Context
from transmuter_amd._lib import lib
from transmuter_amd.serving import PagedCache

pytestmark = pytest.mark.gpu


def test_a_context_made_in_a_capture():
    print("a context made in a capture", flush=True)
    a, b = Context(0), None
    try:
        x = a.put(np.arange(8, dtype=np.float32))
        graph = ctypes.c_void_p()
        a.check(lib().tmh_graph_begin(a.handle, None))
        try:
            b = Context(0)
        finally:
            a.check(lib().tmh_graph_end(a.handle, None, ctypes.byref(graph)))
            a.check(lib().tmh_graph_destroy(a.handle, graph))
        assert np.array_equal(x.numpy(), np.arange(8))
        # Two sequences in parts that meet in the kernel, twice: the new context has its counters.
        cache = PagedCache(b, 64, 128, 1, 64, "f32")
        ones = np.ones(cache.k.shape, np.float32)
        cache.k, cache.v = b.put(ones), b.put(ones * 3)
        cache.desc.k, cache.desc.v = cache.k.ptr, cache.v.ptr
        table, lengths = b.put(np.arange(64, dtype=np.int32).reshape(2, 32)), b.put(np.array([4000, 3], np.int32))
        for _ in range(3):  # (exact sums; the reciprocal of the weights' sum and the product with it are rounded)
            y = cache.attend(b.put(np.ones((2, 64), np.float32)), table, lengths).numpy()
            assert (np.abs(y - 3) <= 2 * 2.0 ** -24 * 3).all()
        cache.free()
    finally:
        if b is not None:
            b.close()
        a.close()
