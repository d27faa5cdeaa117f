"""Attention under a visibility rule without a GPU: the oracle of its GPU tests against differences, bucket borders in whole numbers, and what
the entry points refuse before they look at a device."""
import ctypes

import numpy as np
import pytest

from tests import attention_rule as R


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as entry

    entry.build()
    from gradcraft_b200 import capi

    return capi.lib()


@pytest.mark.parametrize("buckets,reach", [(1, 1), (1, 5), (2, 2), (3, 1000), (8, 64), (16, 128), (32, 128), (32, 256), (32, 16), (33, 1000), (64, 64), (64, 1 << 20), (5, (1 << 30) - 1)])
def test_bucket_starts_are_exact(lib, buckets, reach):
    got = np.empty(buckets, np.int64)
    lib.relative_bucket_starts(buckets, reach, got)
    assert got.tolist() == R.bucket_starts(buckets, reach).tolist()
    assert got[0] == 0 and (np.diff(got) >= 0).all()


def test_a_border_that_a_logarithm_rounds_to_either_side(lib):
    # 16 (256 / 16)^(k / 16) = 2^(4 + k / 4) is whole for every fourth k
    got = np.empty(32, np.int64)
    lib.relative_bucket_starts(32, 256, got)
    assert [got[16 + k] for k in (0, 4, 8, 12)] == [16, 32, 64, 128]


@pytest.mark.parametrize("buckets,reach", [(0, 8), (65, 8), (-1, 8), (8, 0), (8, -3), (8, 1 << 30)])
def test_bucket_starts_refuse(lib, buckets, reach):
    from gradcraft_b200 import capi

    with pytest.raises(capi.GcbError) as e:
        lib.relative_bucket_starts(buckets, reach, np.empty(64, np.int64))
    assert e.value.status == capi.INVALID_ARG


@pytest.mark.parametrize("window,sinks,biased", [(0, 0, False), (2, 0, True), (2, 2, True), (1, 0, False)])
def test_the_oracle_s_gradients_against_differences(window, sinks, biased):
    rng = np.random.default_rng(3)
    q, k, v, g = (rng.standard_normal((1, 2, 6, 3)) for _ in range(4))
    starts = np.array([0, 1, 3])
    bias = rng.standard_normal((2, 3)) if biased else None
    args = (0.7, window, sinks, bias, starts)
    grads = R.attention(q, k, v, *args, dout=g)[1:]
    for x, dx in zip((q, k, v) + ((bias,) if biased else ()), grads):
        for at in np.ndindex(x.shape):
            keep, f = x[at], []
            for eps in (1e-5, -1e-5):
                x[at] = keep + eps
                f.append((R.attention(q, k, v, *args) * g).sum())
            x[at] = keep
            assert abs((f[0] - f[1]) / 2e-5 - dx[at]) < 1e-8


BAD = [dict(window=-1), dict(sinks=-1), dict(sinks=65), dict(buckets=0), dict(buckets=65), dict(starts=[1, 2, 3]), dict(starts=[0, 3, 2]), dict(B=-1), dict(T=-1), dict(D=-2)]


@pytest.mark.parametrize("bad", BAD, ids=lambda b: "-".join("%s=%s" % kv for kv in b.items()))
@pytest.mark.parametrize("entry", ["window_attention_fwd_f32", "window_attention_bwd_f32", "window_attention_step_f32"])
def test_refusals_before_a_device_is_looked_at(lib, entry, bad):
    from gradcraft_b200 import capi

    ctx = ctypes.create_string_buffer(1 << 14)  # zeros: a context that nothing below may touch
    a = dict(dict(window=4, sinks=1, buckets=3, starts=[0, 1, 2], B=1, H=1, T=4, D=4), **bad)
    some, at, starts = np.zeros(64, np.float32), (4, 16, 16), np.array(a["starts"], np.int64)
    rule = (1.0, a["window"], a["sinks"], some, a["buckets"], starts)
    size = (a["B"], a["H"], a["T"], a["D"])
    if entry.endswith("fwd_f32"):
        args = size + (some, *at, some, some, *at, some, *at, some, *at) + rule
    elif entry.endswith("bwd_f32"):
        args = size + (some, some, some, *at, some, 0, some, *at, some, *at, some, some, *at, some, *at, some, *at) + rule
    else:
        args = (a["B"], a["H"], a["D"], some, 4, 4, some, 4, 4, some, *at, some, *at, a["T"], np.zeros(1, np.int64)) + rule
    with pytest.raises(capi.GcbError) as e:
        getattr(lib, entry)(ctypes.addressof(ctx), *args)
    assert e.value.status == capi.INVALID_ARG


@pytest.mark.parametrize("p", [-0.1, 1.5, float("nan")])
def test_dropout_refuses_what_is_no_probability(lib, p):
    from gradcraft_b200 import capi

    ctx, x = ctypes.create_string_buffer(1 << 14), np.zeros(4, np.float32)
    for call in (lambda: lib.dropout_fwd_f32(ctypes.addressof(ctx), x, x, None, 4, p, 0, 0), lambda: lib.dropout_bwd_f32(ctypes.addressof(ctx), x, x, 4, p, 0, 0, 0)):
        with pytest.raises(capi.GcbError) as e:
            call()
        assert e.value.status == capi.INVALID_ARG


def test_philox_matches_the_published_vectors():
    # Random123's known answers for philox4x32-10: counter and key all zeros, and all ones (only the first two counter words are free here)
    assert [hex(w) for w in R.philox_words(4, 0, 0)] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
