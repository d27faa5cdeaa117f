"""Layouts of outputs and gradients that attention under a visibility rule refuses before it looks at a device: rows on top of one another."""
import ctypes

import numpy as np
import pytest


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as entry

    entry.build()
    from gradcraft_b200 import capi

    return capi.lib()


@pytest.fixture
def ctx():
    return ctypes.create_string_buffer(1 << 14)  # zeros: a context that nothing below may touch


def refused(capi_call):
    from gradcraft_b200 import capi

    with pytest.raises(capi.GcbError) as e:
        capi_call()
    assert e.value.status == capi.INVALID_ARG and "overlap" in str(e.value)


# strides of a row, a sequence and a head of 2 x 3 sequences of 4 rows of 8 columns, which are (24, 96, 8) or (8, 96, 32) where they are dense
@pytest.mark.parametrize("at", [(24, 96, 4), (24, 4, 8), (7, 96, 32), (8, 96, 8), (24, 24, 8), (24, 96, 24), (8, 96, 16), (24, 8, 8), (24, 92, 8), (8, 96, 28), (24, 96, 0), (24, -96, 8), (24, 48, 8)], ids=str)
def test_rows_on_top_of_one_another(lib, ctx, at):
    x, good, rule = np.zeros(256, np.float32), (24, 96, 8), (1.0, 4, 1, None, 0, None)
    refused(lambda: lib.window_attention_fwd_f32(ctypes.addressof(ctx), 2, 3, 4, 8, x, *at, x, x, *good, x, *good, x, *good, *rule))
    refused(lambda: lib.window_attention_bwd_f32(ctypes.addressof(ctx), 2, 3, 4, 8, x, x, x, *at, None, 0, x, *good, x, *good, x, x, *good, x, *good, x, *good, *rule))


# strides of a sequence and a head of 4 x 3 rows, which are (24, 8) or (8, 32) where they are dense
@pytest.mark.parametrize("at", [(24, 4), (4, 24), (8, 8), (16, 8), (8, 24), (20, 8), (24, 0), (-24, 8), (24, -8)], ids=str)
def test_single_positions_on_top_of_one_another(lib, ctx, at):
    x, good, rule = np.zeros(256, np.float32), (24, 96, 8), (1.0, 4, 1, None, 0, None)
    refused(lambda: lib.window_attention_step_f32(ctypes.addressof(ctx), 4, 3, 8, x, *at, x, 24, 8, x, *good, x, *good, 4, np.zeros(4, np.int64), *rule))
