"""Attention under a visibility rule where scores are large, and where a query is not a number."""
import numpy as np
import pytest

from tests import attention_rule as R
from tests.helpers import max_abs_rel
from tests.test_window_attention_gpu import TOL, Case, env  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("engine", [0, 1])
@pytest.mark.parametrize("buckets", [0, 8])
@pytest.mark.parametrize("T,D,top", [(200, 16, 8.0), (400, 64, 8.0), (150, 96, 4.0)])
def test_gradients_of_large_scores(env, T, D, top, buckets, engine):  # noqa: F811
    """Scores up to top^2 D, growing along the sequence.

    A score s is off by at most e = 2^-19 |s| (its terms have one sign) plus what a logarithm and a product of its size add in the backward pass,
    8 x 2^-24 |s|: below 2^-18 |s| together.  A probability is e^(s - log-sum), both of them off by that: a factor of 1 +- d, d = 2 x 2^-18 max |s|.
    With A = |P| (|dP| + |dO| |O|), where dP = dO V^T: G = P (dP - dO O) is off by d A, and by d' |P| |dO| |O|, d' = d for O's own probabilities; each product after it by 2^-19
    of its terms.  So dQ is off by (2 d + 2^-18) scale A |K|, dK by the same of A^T |Q|, dV by (d + 2^-18) |P|^T |dO|, dbias by (2 d + 2^-18) of the sum of A.
    A bucket's part of a block of 32 x 16 elements of G is a difference of two running sums over its diagonals, 16 + 5 + 1 additions each, so that it is also off by
    2 x 22 + 1 half steps of the sizes of all G around it: 45 x 2^-24 of the sum of A over all buckets."""
    ctx, torch, capi = env
    c = Case(torch, 1, 1, T, D, buckets, 40)
    for name in "qk":
        x = np.full((1, 1, T, D), 1.0, np.float32) * np.linspace(0.1, top, T, dtype=np.float32)[None, None, :, None]
        c.host[name] = x
        c.dev[name] = c.place(x)
    ctx.ctx_set_gemm_engine(engine)
    try:
        c.forward(ctx, 90, 1, 1.0)
        c.backward(ctx)
        ctx.sync()
    finally:
        ctx.ctx_set_gemm_engine(0)
    q, k, v, g = (c.host[n][0, 0].astype(np.float64) for n in ("q", "k", "v", "dout"))
    want = R.attention(c.host["q"], c.host["k"], c.host["v"], 1.0, 90, 1, c.bias, c.starts, c.host["dout"])
    i = np.arange(T)
    dist = i[:, None] - i[None, :]
    s = q @ k.T + (R.bias_of(c.bias.astype(np.float64), c.starts, dist)[0] if buckets else 0.0)
    d = 4 * 2.0**-19 * np.abs(s).max()
    s = np.where(R.visible(i[:, None], i[None, :], 90, 1), s, -np.inf)
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    a = p * (np.abs(g) @ np.abs(v).T + (np.abs(g) * (p @ np.abs(v))).sum(1, keepdims=True))
    small, twice = d + 2.0**-18, 2 * d + 2.0**-18
    bounds = [small * (p @ np.abs(v)), twice * (a @ np.abs(k)), twice * (a.T @ np.abs(q)), small * (p.T @ np.abs(g))]
    for got, ref, bound in zip([c.out] + c.grads, want, bounds):
        assert (np.abs(got.cpu().numpy()[0, 0] - ref[0, 0]) <= bound).all()
    if buckets:
        n = np.searchsorted(c.starts, np.maximum(dist, 0), side="right") - 1
        assert all(abs(c.dbias[0, b].item() - want[4][0, b]) <= twice * a[n == b].sum() + 45 * 2.0**-24 * a.sum() for b in range(buckets))


@pytest.mark.parametrize("engine", [0, 1])
@pytest.mark.parametrize("buckets", [0, 8])
@pytest.mark.parametrize("T,D", [(40, 16), (300, 64), (90, 96), (150, 7)])
def test_a_query_that_is_not_a_number_stays_one_row(env, T, D, buckets, engine):  # noqa: F811
    """Its row of out and dq holds no numbers; the other rows are what they were, but for the moments at which a tile of them moves to a new maximum."""
    ctx, torch, capi = env
    ctx.ctx_set_gemm_engine(engine)
    try:
        c = Case(torch, 2, 2, T, D, buckets, 16)
        c.forward(ctx, 24, 3, 0.3)
        c.backward(ctx)
        before = [c.out.clone(), c.grads[0].clone()]
        c.dev["q"][0][1, 0, T // 2] = float("nan")
        c.forward(ctx, 24, 3, 0.3)
        c.backward(ctx)
        ctx.sync()
    finally:
        ctx.ctx_set_gemm_engine(0)
    for was, now in zip(before, [c.out, c.grads[0]]):
        assert now[1, 0, T // 2].isnan().all()
        now[1, 0, T // 2] = was[1, 0, T // 2]
        assert max_abs_rel(now.cpu().numpy(), was.cpu().numpy()) < TOL
