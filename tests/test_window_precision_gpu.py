"""Attention under a visibility rule on values, keys and gradients that share a large common part, as those of a trained model do (a bias, a direction
that all positions have): sums of one sign, in which what a tensor core cuts off adds up, and gradients that are small differences of large ones.

What is allowed, with all operands positive, so that every sum is as large as its terms:
  A product of split operands is off by less than u = 2^-17: two cross products whose factors are rounded to 8 bits, 2^-9 each of at most 2^-10,
  and a product of two remainders left out.  The signs are random: a sum of n such terms has 4 u / sqrt(n) of its size.
  An addition on the tensor core cuts off less than 2^-23 of the sum.  Scores, dP and a block's share of O are at most 16 additions, of which the
  first eight are of remainders 2^-10 as large: b = 9 x 2^-23.  Sums over a sequence move on every four blocks, 64 additions: 64 x 2^-23.
  G = P (dP - dO . O): off by b and 4 u / sqrt(D) of A = P (dP + dO . O); sums of G over n pairs keep b, and 1 / sqrt(n) of the rest."""
import numpy as np
import pytest

from tests import attention_rule as R
from tests.test_window_attention_gpu import Case, env  # noqa: F401

pytestmark = pytest.mark.gpu
U, B16, B64 = 2.0**-17, 9 * 2.0**-23, 64 * 2.0**-23


def rms(x, axis):
    """4 / sqrt(the number of terms that carry a sum of positive ones), at most 1"""
    total = x.sum(axis)
    return np.minimum(1.0, 4 * np.sqrt((x * x).sum(axis)) / np.where(total > 0, total, 1.0))


@pytest.mark.parametrize("buckets", [0, 15])
@pytest.mark.parametrize("T,window,sinks,D", [(600, 0, 0, 64), (1500, 700, 3, 64), (700, 130, 0, 32), (400, 0, 0, 40)])
def test_a_large_common_part(env, T, window, sinks, D, buckets):  # noqa: F811
    ctx, torch, capi = env
    c = Case(torch, 1, 2, T, D, buckets, 200)
    rng = np.random.default_rng(4)
    for name, low, high in (("q", 0.0, 0.1), ("k", 0.8, 1.2), ("v", 0.7, 1.3), ("dout", 0.7, 1.3)):
        x = rng.uniform(low, high, (1, 2, T, D)).astype(np.float32)
        c.host[name] = x
        c.dev[name] = c.place(x)
    if buckets:
        c.bias *= 0.1
    scale = D**-0.5
    before = ctx.ctx_launch_count_named(b"window_attention_tc")
    c.forward(ctx, window, sinks, scale)
    c.backward(ctx)
    ctx.sync()
    assert ctx.ctx_launch_count_named(b"window_attention_tc") == before + 3
    want = R.attention(*(c.host[n] for n in "qkv"), scale, window, sinks, c.bias, c.starts, c.host["dout"])
    i = np.arange(T)
    dist = i[:, None] - i[None, :]
    seen = R.visible(i[:, None], i[None, :], window, sinks)
    for h in range(2):
        q, k, v, g = (c.host[n][0, h].astype(np.float64) for n in ("q", "k", "v", "dout"))
        s = np.where(seen, scale * q @ k.T + (R.bias_of(c.bias.astype(np.float64), c.starts, dist)[h] if buckets else 0.0), -np.inf)
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        dp = g @ v.T
        a = p * (dp + (p * dp).sum(1, keepdims=True))  # G is its two parts' difference
        one = U * 4 / np.sqrt(D)  # random part of an element of G, of A
        rows, cols = rms(p, 1)[:, None], rms(p, 0)[:, None]
        flat = dict(out=(B16 + U * rows) * (p @ v), dv=(B64 + U * cols) * (p.T @ g),
                    dq=scale * ((B16 + one * rms(a, 1)[:, None]) * (a @ k) + (B64 + U) * (np.abs(p * (dp - (p * dp).sum(1, keepdims=True))) @ k)),
                    dk=scale * ((B16 + one * rms(a, 0)[:, None]) * (a.T @ q) + (B64 + U) * (np.abs(p * (dp - (p * dp).sum(1, keepdims=True))).T @ q)))
        for name, got, ref in zip(("out", "dq", "dk", "dv"), [c.out] + c.grads, want):
            worst = (np.abs(got.cpu().numpy()[0, h] - ref[0, h]) / flat[name]).max()
            assert worst <= 1, (name, worst)
        if buckets:
            n = np.searchsorted(c.starts, np.maximum(dist, 0), side="right") - 1
            for b in range(buckets):
                pairs = a[(n == b) & seen]
                if pairs.size:
                    bound = (B16 + one * rms(pairs, 0)) * pairs.sum()
                    assert abs(c.dbias[h, b].item() - want[4][h, b]) <= bound, (b, abs(c.dbias[h, b].item() - want[4][h, b]) / bound)
