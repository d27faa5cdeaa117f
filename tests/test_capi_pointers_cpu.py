"""What the ctypes view takes in the place of a pointer, and what it refuses before anything is launched."""
import ctypes

import numpy as np
import pytest


@pytest.fixture(scope="module")
def call():
    """An entry point with one pointer that gives it back, in the wrapper of the real ones."""
    from gradcraft_b200 import capi

    proto = ctypes.CFUNCTYPE(ctypes.c_void_p, ctypes.c_void_p)
    entry = proto(lambda p: p)
    entry.argtypes = [ctypes.c_void_p]
    return capi.Lib._wrap(None, entry, False, [0])


def test_arrays_tensors_integers_and_ctypes_values(call):
    import torch

    x, t = np.arange(6, dtype=np.float32).reshape(2, 3), torch.zeros(4)
    value = ctypes.c_int64(3)
    assert call(x) == x.ctypes.data and call(x[1:]) == x.ctypes.data + 12 and call(np.array(5)) is not None
    assert call(t) == t.data_ptr() and call(t[1:]) == t.data_ptr() + 4
    assert call(None) is None and call(4096) == 4096 and call(ctypes.addressof(value)) == ctypes.addressof(value)
    assert call(ctypes.byref(value)) == ctypes.addressof(value) and call(ctypes.c_void_p(4096)) == 4096


class Lookalike:
    __array_interface__ = dict(np.zeros(3).__array_interface__)


@pytest.mark.parametrize("x", [np.int64(4096), np.uint64(4096), np.float32(1.0), np.bool_(True), Lookalike(), 1.5, [1, 2]], ids=lambda x: type(x).__name__)
def test_what_is_neither_is_refused(call, x):
    """A numpy scalar offers an array interface too, to a copy of its own that is gone with the call."""
    with pytest.raises((TypeError, ctypes.ArgumentError)):
        call(x)
