"""Attention of single positions on values that are not finite: a query or a key that it sees passes them on, what a bias of -inf hides does not.

Tolerance as in test_window_attention_gpu.py: two products of up to 128 terms and an exponential, well below 2e-5 of the largest value."""
import numpy as np
import pytest

from tests import attention_rule as R
from tests.helpers import max_abs_rel

pytestmark = pytest.mark.gpu
TOL = 2e-5
SIZES = [
    # B, H, D, cap, window, sinks, whether the streaming kernel takes it
    (3, 2, 16, 5, 2, 1, False),
    (3, 2, 7, 90, 0, 0, False),
    (3, 3, 64, 700, 500, 4, False),
    (3, 2, 128, 300, 0, 0, False),
    (6, 12, 64, 1000, 900, 3, False),
    (7, 12, 64, 1000, 900, 3, True),
    (6, 12, 40, 2000, 0, 0, True),
    (4, 16, 96, 800, 0, 0, True),
]
ids = pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s[:6])))


@pytest.fixture(scope="module")
def env():
    import torch

    from gradcraft_b200 import capi

    ctx = capi.Context(0)
    yield ctx, torch
    ctx.sync()
    ctx.close()


def data(size, seed=0):
    B, H, D, cap = size[:4]
    rng = np.random.default_rng(seed)
    lengths = rng.integers(1, cap + 1, B)
    lengths[0], lengths[-1] = cap, 0
    return [rng.standard_normal(s, dtype=np.float32) for s in ((B, H, D), (B, H, cap, D), (B, H, cap, D))] + [lengths]


def run(env, size, q, k, v, lengths, bias=None, starts=None):
    ctx, torch = env
    B, H, D, cap, window, sinks, streamed = size
    out = torch.full((B, H, D), 7.0, device="cuda")
    kd, vd = (torch.from_numpy(x).cuda().transpose(1, 2).contiguous() for x in (k, v))
    at, before = (H * D, cap * H * D, D), ctx.ctx_launch_count_named(b"window_attention_stream")
    ctx.window_attention_step_f32(B, H, D, out, H * D, D, torch.from_numpy(q).cuda(), H * D, D, kd, *at, vd, *at, cap, torch.from_numpy(lengths).cuda(), D**-0.5, window, sinks,
                                  None if bias is None else torch.from_numpy(bias).cuda(), 0 if bias is None else len(starts), starts)
    ctx.sync()
    assert ctx.ctx_launch_count_named(b"window_attention_stream") == before + streamed
    return out.cpu().numpy()


@ids
@pytest.mark.parametrize("biased", [False, True])
def test_a_query_that_is_not_a_number(env, size, biased):
    """The heads with such a query give no numbers, unless their sequence is empty; all others are what they were."""
    B, H, D, cap, window, sinks, _ = size
    q, k, v, lengths = data(size)
    starts = R.bucket_starts(8, 64) if biased else None
    bias = np.random.default_rng(5).standard_normal((H, 8), dtype=np.float32) if biased else None
    want = R.step(q, k, v, lengths, D**-0.5, window, sinks, bias, starts)
    q[0, 1, D // 2] = q[1, 0, 0] = q[-1, 0, D - 1] = np.nan
    got = run(env, size, q, k, v, lengths, bias, starts)
    lost = np.zeros((B, H), bool)
    lost[0, 1] = lost[1, 0] = True
    assert np.isnan(got[lost]).all()
    assert max_abs_rel(got[~lost], want[~lost]) < TOL and not got[-1].any()


@ids
def test_keys_that_are_not_numbers(env, size):
    """All keys that a head sees, or one of them; a row of values that holds infinities."""
    B, H, D, cap, window, sinks, _ = size
    q, k, v, lengths = data(size, 1)
    want = R.step(q, k, v, lengths, D**-0.5, window, sinks)
    k[0, 0] = np.nan
    k[1, 1, lengths[1] - 1, 0] = np.nan
    v[0, 1, lengths[0] - 1] = np.inf
    got = run(env, size, q, k, v, lengths)
    lost = np.zeros((B, H), bool)
    lost[0, 0] = lost[1, 1] = True
    assert np.isnan(got[lost]).all() and np.isposinf(got[0, 1]).all()
    lost[0, 1] = True
    assert max_abs_rel(got[~lost], want[~lost]) < TOL


@ids
@pytest.mark.parametrize("hidden", [[0], [2], [7], [1, 3, 5], list(range(8))], ids=str)
def test_what_a_bias_of_minus_infinity_hides_may_hold_anything(env, size, hidden):
    B, H, D, cap, window, sinks, _ = size
    q, k, v, lengths = data(size, 2)
    starts = R.bucket_starts(8, 64)
    bias = np.random.default_rng(6).standard_normal((H, 8), dtype=np.float32)
    bias[:, hidden] = -np.inf
    want = R.step(q, k, v, lengths, D**-0.5, window, sinks, bias, starts)
    for b, n in enumerate(lengths):
        j = np.arange(n)
        j = j[np.isin(np.searchsorted(starts, n - 1 - j, side="right") - 1, hidden)]
        k[b][:, j[::2]] = np.nan
        k[b][:, j[1::2]] = np.inf
        v[b][:, j[::3]] = np.nan
        v[b][:, j[1::3]] = -np.inf
    got = run(env, size, q, k, v, lengths, bias, starts)
    assert max_abs_rel(got, want) < TOL
    if len(hidden) == 8:
        assert not got.any()
