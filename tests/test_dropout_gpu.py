"""Dropout through the C ABI against the generator's definition (tests/attention_rule.py).  The mask has to be exact; a kept value is one
multiplication by a rounded 1 / (1 - p) and one addition: three roundings of at most 2^-24 each."""
import numpy as np
import pytest

from tests import attention_rule as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch

    from gradcraft_b200 import capi

    ctx = capi.Context(0)
    yield ctx, torch, capi
    ctx.sync()
    ctx.close()


@pytest.mark.parametrize("seed,offset", [(0, 0), (12345678901234, 7), (-1, (1 << 32) - 2), (1 << 62, -3)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.999, 1.0])
@pytest.mark.parametrize("n,shift", [(1, 0), (3, 0), (4, 0), (1023, 0), (4096, 0), (4097, 1), (257, 3)])
def test_mask_and_values(env, n, shift, p, seed, offset):
    ctx, torch, capi = env
    rng = np.random.default_rng(n)
    x, res = rng.standard_normal(n + shift, dtype=np.float32), rng.standard_normal(n + shift, dtype=np.float32)
    X, RES, out = torch.from_numpy(x).cuda()[shift:], torch.from_numpy(res).cuda()[shift:], torch.full((n + shift + 4,), 7.0, device="cuda")
    keep = R.kept(n, p, seed % 2**64, offset % 2**64)
    with np.errstate(divide="ignore", invalid="ignore"):
        want = np.where(keep, x[shift:].astype(np.float64) / (1.0 - float(np.float32(p))), 0.0)
    for residual in (None, RES):
        ctx.dropout_fwd_f32(out[shift:], X, residual, n, p, seed, offset)
        ctx.sync()
        got, ref = out[shift:shift + n].cpu().numpy().astype(np.float64), want + (0.0 if residual is None else res[shift:].astype(np.float64))
        assert (out[:shift] == 7).all() and (out[shift + n:] == 7).all()
        assert (np.abs(got - ref) <= 3 * 2.0**-24 * (np.abs(want) + np.abs(ref))).all()
        if residual is None:
            assert ((got != 0) == (keep & (x[shift:] != 0))).all()
    dx = RES.clone()
    ctx.dropout_bwd_f32(dx, X, n, p, seed, offset, 1)  # gradient: the same mask and factor, added to what is there
    ctx.sync()
    assert torch.equal(dx, out[shift:shift + n])
    ctx.dropout_bwd_f32(dx, X, n, p, seed, offset, 0)
    ctx.dropout_fwd_f32(X, X, None, n, p, seed, offset)  # in place
    ctx.sync()
    assert torch.equal(dx, X)


def test_large_call_continues_where_a_smaller_one_ends(env):
    """The mask hangs on the element's number alone: a call over everything equals calls over its parts."""
    ctx, torch, capi = env
    n, cut = 148 * 4096 + 4 * 1234 + 3, 4 * 1000
    x = torch.randn(n, device="cuda")
    whole, parts = torch.empty_like(x), torch.empty_like(x)
    ctx.dropout_fwd_f32(whole, x, None, n, 0.3, 5, 100)
    ctx.dropout_fwd_f32(parts, x, None, cut, 0.3, 5, 100)
    ctx.dropout_fwd_f32(parts[cut:], x[cut:], None, n - cut, 0.3, 5, 100 + cut // 4)
    ctx.sync()
    assert torch.equal(whole, parts)
    keep = R.kept(4096, 0.3, 5, 100)
    assert ((whole[:4096] != 0).cpu().numpy() == keep).all()
    kept = float((whole != 0).double().mean())  # four standard deviations of n draws
    assert abs(kept - 0.7) < 4 * (0.21 / n) ** 0.5


def test_dropped_values_are_not_looked_at(env):
    ctx, torch, capi = env
    n = 1000
    keep = torch.from_numpy(R.kept(n, 0.5, 3, 9)).cuda()
    x = torch.where(keep, torch.ones(n, device="cuda"), torch.full((n,), float("nan"), device="cuda"))
    out = torch.empty(n, device="cuda")
    ctx.dropout_fwd_f32(out, x, None, n, 0.5, 3, 9)
    ctx.sync()
    assert torch.equal(out, torch.where(keep, 2.0, 0.0))


def test_refusals_and_empty_calls(env):
    ctx, torch, capi = env
    x = torch.zeros(8, device="cuda")
    ctx.dropout_fwd_f32(None, None, None, 0, 0.5, 0, 0)
    for bad in (lambda: ctx.dropout_fwd_f32(None, x, None, 8, 0.5, 0, 0), lambda: ctx.dropout_fwd_f32(x, None, None, 8, 0.5, 0, 0), lambda: ctx.dropout_fwd_f32(x, x, None, -1, 0.5, 0, 0),
                lambda: ctx.dropout_fwd_f32(x, x, None, 8, 1.1, 0, 0), lambda: ctx.dropout_bwd_f32(x, x, 8, -0.1, 0, 0, 0)):
        with pytest.raises(capi.GcbError) as e:
            bad()
        assert e.value.status == capi.INVALID_ARG
    ctx.sync()
