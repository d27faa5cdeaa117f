"""Attention under a visibility rule (window, first positions, bias by distance bucket) and its single-token form against the definitions
in 64 bits (tests/attention_rule.py).

Tolerance: a product of up to 128 terms is off by about 2^-19 of its terms' size with split operands, 16 x 2^-24 in fp32; an output passes
through at most six such products and exponentials one after another, which comes to 1.2e-5 of the largest value; 2e-5 is used.  The bias
gradient adds up to 10^5 terms that each carry such an error, of either sign, and is held to 4e-5 of the largest."""
import numpy as np
import pytest

from tests import attention_rule as R
from tests.helpers import max_abs_rel

pytestmark = pytest.mark.gpu
TOL, TOL_BIAS = 2e-5, 4e-5


@pytest.fixture(scope="module")
def env():
    import torch

    from gradcraft_b200 import capi

    ctx = capi.Context(0)
    yield ctx, torch, capi
    ctx.sync()
    ctx.close()


class Case:
    """Operands in one of several layouts, all seen as (B, H, T, D): "bthd" and "bhtd" by the order in memory, "wide" in rows with room between
    them, "odd" off 16-byte boundaries, "shared" one k and v for all heads (stride 0)."""

    def __init__(self, torch, B, H, T, D, buckets=0, reach=0, layout="bthd", seed=0):
        self.torch, self.size = torch, (B, H, T, D)
        rng = np.random.default_rng(seed)
        self.host, self.dev, self.layout = {}, {}, layout
        for name in ("q", "k", "v", "dout"):
            x = rng.standard_normal((B, 1 if layout == "shared" and name in "kv" else H, T, D), dtype=np.float32)
            self.host[name] = np.broadcast_to(x, (B, H, T, D))
            self.dev[name] = self.place(x)
        self.starts = R.bucket_starts(buckets, reach) if buckets else None
        self.bias = rng.standard_normal((H, buckets), dtype=np.float32) if buckets else None
        self.dbias = torch.full((H, buckets), float("nan"), device="cuda") if buckets else None

    def place(self, x=None):
        """(view seen as (B, H, T, D), strides of row, sequence, head); without x: an output full of NaN"""
        torch, (B, H, T, D) = self.torch, self.size
        heads = H if x is None else x.shape[1]
        order = {"bhtd": (0, 1, 2)}.get(self.layout, (0, 2, 1))
        ext = [B, heads, T]
        room = D + 8 if self.layout == "wide" else D + 3 if self.layout == "odd" else D
        flat = torch.full((ext[order[0]] * ext[order[1]] * ext[order[2]] * room + 1,), float("nan"), device="cuda")
        flat = flat[1:] if self.layout == "odd" else flat[:-1]
        view = flat.view([ext[o] for o in order] + [room])[..., :D].permute(*[order.index(d) for d in range(3)], 3)
        if x is not None:
            view.copy_(torch.from_numpy(x))
        st = view.stride()
        return view, (st[2], st[0], st[1] if heads == H else 0)

    def forward(self, ctx, window, sinks, scale):
        B, H, T, D = self.size
        self.rule = (scale, window, sinks, self.bias_dev(), 0 if self.bias is None else self.bias.shape[1], self.starts)
        self.stats = self.torch.full((max(1, ctx.lib.attention_stats_floats(B, H, T)),), float("nan"), device="cuda")
        self.out, self.out_at = self.place()
        ctx.window_attention_fwd_f32(B, H, T, D, self.out, *self.out_at, self.stats, *self.arg("q"), *self.arg("k"), *self.arg("v"), *self.rule)

    def bias_dev(self):
        return None if self.bias is None else self.torch.from_numpy(self.bias).cuda()

    def arg(self, name):
        return (self.dev[name][0], *self.dev[name][1])

    def backward(self, ctx, accumulate=0):
        B, H, T, D = self.size
        grads = [self.place() for _ in range(3)]
        self.grads = [g for g, _ in grads]
        ctx.window_attention_bwd_f32(B, H, T, D, *self.grads, *grads[0][1], self.dbias, accumulate, *self.arg("dout"), self.out, *self.out_at, self.stats, *self.arg("q"), *self.arg("k"), *self.arg("v"), *self.rule)

    def check(self, ctx, window, sinks, scale):
        self.forward(ctx, window, sinks, scale)
        self.backward(ctx)
        ctx.sync()
        want = R.attention(self.host["q"], self.host["k"], self.host["v"], scale, window, sinks, self.bias, self.starts, self.host["dout"])
        for name, got, ref in zip(("out", "dq", "dk", "dv"), [self.out] + self.grads, want):
            self.close(name, got, ref, TOL, scale)
        if self.bias is not None:
            self.close("dbias", self.dbias, want[4], TOL_BIAS, scale)

    def close(self, name, got, ref, tol, scale):
        got = got.cpu().numpy()
        if np.abs(ref).max() > 1e-10:
            assert max_abs_rel(got, ref) < tol, name
            return
        # A query that sees one key (a table of one bucket, all of them together) has no gradient: dO . v - dO . O is the difference of two equal
        # sums of D terms, each off by at most (2^-19 + D 2^-24) of the sum of their sizes, and probabilities add up to one.
        (B, H, T, D), d = self.size, {n: np.abs(x).astype(np.float64) for n, x in self.host.items()}
        most = 2 * (2.0**-19 + D * 2.0**-24) * d["dout"].sum(3).max() * d["v"].max()
        assert np.abs(got).max() <= most * (B * T if name == "dbias" else abs(scale) * d["k"].max() if name == "dq" else abs(scale) * T * d["q"].max()), name


SIZES = [
    # B, H, T, D, window, sinks, buckets, reach
    (2, 3, 1, 16, 0, 0, 0, 0),
    (2, 3, 1, 16, 1, 1, 4, 8),
    (1, 2, 2, 4, 1, 0, 0, 0),
    (1, 2, 5, 8, 1, 2, 0, 0),  # beyond the first two positions a query sees itself and those
    (3, 2, 31, 12, 7, 0, 8, 16),
    (2, 2, 64, 64, 64, 3, 0, 0),  # the window just covers the sequence
    (2, 2, 65, 32, 64, 1, 32, 128),  # one key of one query is beyond it, and stays visible
    (1, 3, 127, 64, 63, 64, 0, 0),  # more first positions than the window reaches
    (1, 2, 128, 40, 65, 5, 1, 1),
    (2, 2, 129, 64, 100, 33, 32, 64),
    (1, 4, 200, 64, 0, 0, 32, 128),
    (2, 2, 331, 64, 100, 3, 32, 128),
    (1, 2, 513, 64, 130, 4, 64, 400),
    (1, 1, 1000, 64, 1, 4, 0, 0),  # a window of one
    (1, 2, 1025, 64, 256, 0, 0, 0),
    (1, 1, 1537, 32, 700, 17, 32, 1000),
    (1, 2, 700, 48, 5000, 9, 16, 128),  # a window beyond the sequence
    (1, 2, 300, 96, 70, 4, 32, 128),
    (1, 1, 260, 128, 64, 40, 8, 32),
    (1, 1, 150, 72, 0, 0, 0, 0),
]


@pytest.mark.parametrize("engine", [0, 1])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_gradients(env, size, engine):
    ctx, torch, capi = env
    B, H, T, D, window, sinks, buckets, reach = size
    ctx.ctx_set_gemm_engine(engine)
    try:
        Case(torch, B, H, T, D, buckets, reach).check(ctx, window, sinks, D**-0.5)
    finally:
        ctx.ctx_set_gemm_engine(0)


@pytest.mark.parametrize("size", [s for s in SIZES if s[2] <= 128], ids=lambda s: "x".join(map(str, s)))
def test_short_sequences_on_the_tensor_cores(env, size):
    """Where the choice between the kernels goes the other way by itself."""
    ctx, torch, capi = env
    B, H, T, D, window, sinks, buckets, reach = size
    ctx.ctx_set_gemm_engine(2)
    try:
        before = ctx.ctx_launch_count_named(b"window_attention_tc")
        Case(torch, B, H, T, D, buckets, reach).check(ctx, window, sinks, D**-0.5)
        assert ctx.ctx_launch_count_named(b"window_attention_tc") == before + 3
    finally:
        ctx.ctx_set_gemm_engine(0)


@pytest.mark.parametrize("D", [40, 33, 128])
@pytest.mark.parametrize("T, window, sinks, buckets", [(65, 20, 3, 8), (64, 0, 0, 0), (300, 100, 5, 32), (129, 1, 1, 0)])
def test_enough_heads_for_tiles_of_64_rows(env, T, window, sinks, buckets, D):
    ctx, torch, capi = env
    ctx.ctx_set_gemm_engine(1)
    try:
        Case(torch, 8, 14, T, D, buckets, 64).check(ctx, window, sinks, D**-0.5)
    finally:
        ctx.ctx_set_gemm_engine(0)


@pytest.mark.parametrize("engine", [0, 2])
def test_one_position_with_a_stride_that_no_tensor_map_holds(env, engine):
    ctx, torch, capi = env
    ctx.ctx_set_gemm_engine(engine)
    try:
        c = Case(torch, 1, 3, 1, 16)
        for name in c.dev:
            view, (_, so, si) = c.dev[name]
            c.dev[name] = (view, (1 << 40, so, si))
        c.check(ctx, 4, 1, 0.25)
    finally:
        ctx.ctx_set_gemm_engine(0)


@pytest.mark.parametrize("D", [64, 20, 7])
@pytest.mark.parametrize("layout", ["bhtd", "wide", "odd", "shared"])
def test_layouts(env, layout, D):
    ctx, torch, capi = env
    Case(torch, 2, 3, 150, D, 8, 40, layout=layout).check(ctx, 50, 2, 0.3)


@pytest.mark.parametrize("scale", [-0.5, 0.0, 3.0])
def test_scales(env, scale):
    ctx, torch, capi = env
    Case(torch, 1, 2, 140, 32).check(ctx, 60, 1, scale)


def test_many_heads_of_few_positions_and_few_of_many(env):
    ctx, torch, capi = env
    Case(torch, 40, 16, 17, 16, 4, 8).check(ctx, 5, 1, 0.25)
    Case(torch, 1, 1, 2500, 64, 32, 512).check(ctx, 1024, 4, 0.125)


@pytest.mark.parametrize("hidden", [[0], [1], [3], [0, 1, 2, 3]], ids=str)
@pytest.mark.parametrize("T,D", [(40, 16), (300, 64), (90, 96)])
def test_a_bias_of_minus_infinity_hides_a_bucket(env, T, D, hidden):
    """Rows that see nothing (the first one does where bucket 0 is hidden) give zeros and no gradient."""
    ctx, torch, capi = env
    c = Case(torch, 2, 2, T, D, 4, 16)
    c.bias[:, hidden] = -np.inf
    c.forward(ctx, 24, 3, 0.3)
    c.backward(ctx)
    ctx.sync()
    want = R.attention(c.host["q"], c.host["k"], c.host["v"], 0.3, 24, 3, c.bias, c.starts, c.host["dout"])
    for got, ref in zip([c.out] + c.grads + [c.dbias], want):
        assert max_abs_rel(got.cpu().numpy(), ref) < TOL_BIAS
    if len(hidden) == 4:
        assert not any(t.any() for t in [c.out] + c.grads + [c.dbias])


def test_a_bias_of_the_lowest_value_leaves_a_row_its_only_key(env):
    """Row 0 sees itself alone, under a bias of the type's lowest value: its probability is one."""
    ctx, torch, capi = env
    for T, D in ((50, 16), (200, 64)):
        c = Case(torch, 1, 2, T, D, 4, 16)
        c.bias[:, 0] = np.finfo(np.float32).min
        c.check(ctx, 0, 0, 0.3)


def test_large_scores_neither_overflow_nor_vanish(env):
    """Scores between -4000 and 4000, growing along the sequence, so that the running maximum moves with every tile; probabilities are held to
    what 2^-19 of a score of that size leaves of them."""
    ctx, torch, capi = env
    for T, D in ((200, 16), (400, 64)):
        c = Case(torch, 1, 1, T, D)
        for name in "qk":
            x = np.full((1, 1, T, D), 1.0, np.float32) * np.linspace(0.1, 8.0, T, dtype=np.float32)[None, None, :, None]
            c.host[name] = x
            c.dev[name] = c.place(x)
        c.forward(ctx, 90, 1, 1.0)
        ctx.sync()
        want = R.attention(c.host["q"], c.host["k"], c.host["v"], 1.0, 90, 1)
        assert max_abs_rel(c.out.cpu().numpy(), want) < 64 * D * 2.0**-19


def test_bias_gradient_is_added_and_may_be_left_out(env):
    ctx, torch, capi = env
    for T, D in ((100, 16), (300, 64), (90, 96)):
        c = Case(torch, 2, 2, T, D, 8, 32)
        c.forward(ctx, 40, 2, 0.2)
        c.backward(ctx)
        first, grads = c.dbias.clone(), [g.clone() for g in c.grads]
        c.backward(ctx, accumulate=1)
        ctx.sync()
        assert torch.equal(c.dbias, first + first)
        c.dbias = None
        c.backward(ctx)
        ctx.sync()
        assert all(torch.equal(a, b) for a, b in zip(c.grads, grads))


def test_two_runs_agree_to_the_bit(env):
    ctx, torch, capi = env
    got = []
    for _ in range(2):
        c = Case(torch, 2, 3, 700, 64, 32, 128)
        c.forward(ctx, 200, 4, 0.125)
        c.backward(ctx)
        ctx.sync()
        got.append([c.out.clone(), c.dbias.clone()] + [g.clone() for g in c.grads])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_room_between_rows_and_behind_the_last_one_is_left_alone(env):
    ctx, torch, capi = env
    for D in (64, 7, 96):
        c = Case(torch, 2, 2, 70, D, 4, 8, layout="wide")
        c.forward(ctx, 30, 1, 0.2)
        c.backward(ctx)
        ctx.sync()
        for t in [c.out] + c.grads:
            whole = t.permute(0, 2, 1, 3)
            room = torch.as_strided(whole, (2, 70, 2, 8), whole.stride(), whole.storage_offset() + D)
            assert room.isnan().all() and not whole.isnan().any()


def test_settings_that_change_between_forward_and_backward(env):
    """The row statistics are the same whichever kernels fill and read them."""
    ctx, torch, capi = env
    for first, second in ((0, 1), (1, 0)):
        c = Case(torch, 1, 2, 300, 64, 8, 64)
        ctx.ctx_set_gemm_engine(first)
        c.forward(ctx, 100, 2, 0.125)
        ctx.ctx_set_gemm_engine(second)
        c.backward(ctx)
        ctx.ctx_set_gemm_engine(0)
        ctx.sync()
        want = R.attention(c.host["q"], c.host["k"], c.host["v"], 0.125, 100, 2, c.bias, c.starts, c.host["dout"])
        for got, ref in zip(c.grads, want[1:4]):
            assert max_abs_rel(got.cpu().numpy(), ref) < TOL


def test_captured_and_replayed_with_other_values(env):
    ctx0, torch, capi = env
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = capi.Context(0)
        c = Case(torch, 1, 2, 300, 64, 8, 64)
        c.forward(ctx, 100, 2, 0.125)  # first calls look functions up and let the arena grow
        c.backward(ctx)
        stream.synchronize()
        bias = c.rule[3]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            B, H, T, D = c.size
            ctx.window_attention_fwd_f32(B, H, T, D, c.out, *c.out_at, c.stats, *c.arg("q"), *c.arg("k"), *c.arg("v"), *c.rule)
            ctx.window_attention_bwd_f32(B, H, T, D, *c.grads, *c.out_at, c.dbias, 0, *c.arg("dout"), c.out, *c.out_at, c.stats, *c.arg("q"), *c.arg("k"), *c.arg("v"), *c.rule)
        other = Case(torch, 1, 2, 300, 64, 8, 64, seed=9)
        for n in c.dev:
            c.dev[n][0].copy_(other.dev[n][0])
        bias.copy_(torch.from_numpy(other.bias))
        graph.replay()
        stream.synchronize()
        want = R.attention(*(other.host[n] for n in "qkv"), 0.125, 100, 2, other.bias, other.starts, other.host["dout"])
        for got, ref in zip([c.out] + c.grads + [c.dbias], want):
            assert max_abs_rel(got.cpu().numpy(), ref) < TOL_BIAS
        del graph
        ctx.close()


def test_empty_calls(env):
    ctx, torch, capi = env
    x = torch.zeros(64, device="cuda")
    dbias, starts, at = torch.full((2, 2), 3.0, device="cuda"), np.array([0, 1]), (8, 8, 8)
    for B, H, T in ((0, 2, 4), (1, 2, 0)):
        ctx.window_attention_fwd_f32(B, H, T, 8, x, *at, x, x, *at, x, *at, x, *at, 1.0, 2, 1, dbias, 2, starts)
        ctx.window_attention_bwd_f32(B, H, T, 8, x, x, x, *at, dbias, 1, x, *at, x, *at, x, x, *at, x, *at, x, *at, 1.0, 2, 1, x, 2, starts)
        assert (dbias == 3).all()
    ctx.window_attention_bwd_f32(0, 2, 4, 8, x, x, x, *at, dbias, 0, x, *at, x, *at, x, x, *at, x, *at, x, *at, 1.0, 2, 1, x, 2, starts)
    ctx.sync()
    assert not dbias.any()


def test_refusals(env):
    ctx, torch, capi = env
    x, at = torch.zeros(4096, device="cuda"), (8, 64, 32)

    def fwd(D=8, out=x, stats=x, q=x, at=at, T=4):
        ctx.window_attention_fwd_f32(1, 2, T, D, out, *at, stats, q, *at, x, *at, x, *at, 1.0, 2, 1, None, 0, None)

    for bad, status in ((dict(D=129), capi.UNSUPPORTED), (dict(T=1 << 25), capi.UNSUPPORTED), (dict(out=None), capi.INVALID_ARG), (dict(stats=None), capi.INVALID_ARG), (dict(q=None), capi.INVALID_ARG),
                        (dict(at=(4, 64, 32)), capi.INVALID_ARG), (dict(at=(8, 64, 0)), capi.INVALID_ARG)):
        with pytest.raises(capi.GcbError) as e:
            fwd(**bad)
        assert e.value.status == status, bad
    with pytest.raises(capi.GcbError) as e:  # a gradient of a bias that is not there
        ctx.window_attention_bwd_f32(1, 2, 4, 8, x, x, x, *at, x, 0, x, *at, x, *at, x, x, *at, x, *at, x, *at, 1.0, 2, 1, None, 0, None)
    assert e.value.status == capi.INVALID_ARG
    ctx.sync()


# ---- one new position -----------------------------------------------------------------------------------------------------
STEPS = [
    # B, H, D, cap, window, sinks, buckets, reach
    (1, 1, 64, 1, 0, 0, 0, 0),
    (3, 2, 16, 5, 2, 1, 4, 8),
    (1, 12, 64, 385, 0, 0, 32, 128),
    (4, 3, 40, 200, 64, 4, 0, 0),
    (7, 2, 64, 1000, 1, 0, 0, 0),
    (5, 4, 96, 777, 300, 64, 64, 500),
    (2, 1, 128, 3001, 0, 0, 8, 2000),
    (3, 2, 7, 130, 50, 3, 3, 60),  # rows off 16-byte boundaries
    (1, 2, 32, 9000, 8000, 2, 0, 0),
    # enough keys for the streaming kernel
    (6, 4, 64, 3000, 0, 0, 32, 512),
    (9, 8, 40, 2000, 1500, 64, 16, 128),
    (6, 8, 128, 1200, 700, 4, 0, 0),
    (150, 7, 32, 333, 100, 33, 8, 64),
    (600, 1, 64, 129, 0, 0, 0, 0),
    (5, 1, 64, 16384, 0, 0, 0, 0),
]


@pytest.mark.parametrize("size", STEPS, ids=lambda s: "x".join(map(str, s)))
def test_single_positions(env, size):
    ctx, torch, capi = env
    B, H, D, cap, window, sinks, buckets, reach = size
    rng = np.random.default_rng(1)
    q, k, v = rng.standard_normal((B, H, D), dtype=np.float32), rng.standard_normal((B, H, cap, D), dtype=np.float32), rng.standard_normal((B, H, cap, D), dtype=np.float32)
    lengths = rng.integers(1, cap + 1, B)
    lengths[0], lengths[-1] = cap, 0 if B > 2 else cap
    starts = R.bucket_starts(buckets, reach) if buckets else None
    bias = rng.standard_normal((H, buckets), dtype=np.float32) if buckets else None
    out = torch.full((B, H, D), float("nan"), device="cuda")
    kd, vd = (torch.from_numpy(x).cuda().transpose(1, 2).contiguous() for x in (k, v))
    for b in range(B):  # what lies beyond a length is not read
        kd[b, lengths[b]:] = float("nan")
        vd[b, lengths[b]:] = float("inf")
        if window and lengths[b] - window > sinks:  # nor what the rule hides
            kd[b, sinks:lengths[b] - window] = float("nan")
            vd[b, sinks:lengths[b] - window] = float("nan")
    at = (H * D, cap * H * D, D)
    ctx.window_attention_step_f32(B, H, D, out, H * D, D, torch.from_numpy(q).cuda(), H * D, D, kd, *at, vd, *at, cap, torch.from_numpy(lengths).cuda(), D**-0.5, window, sinks,
                                  None if bias is None else torch.from_numpy(bias).cuda(), buckets, starts)
    ctx.sync()
    assert max_abs_rel(out.cpu().numpy(), R.step(q, k, v, lengths, D**-0.5, window, sinks, bias, starts)) < TOL


@pytest.mark.parametrize("lengths", [[5, 0, 0, 130, 0], [0] * 7, [1] * 9, [64, 65, 63, 1, 0, 4096], [70, 4096], [4096, 0, 3]], ids=lambda x: "-".join(map(str, x)))
def test_streamed_positions_of_uneven_lengths(env, lengths):
    """Few tiles, or all of them in one sequence: heads that lie in several CTAs, CTAs without a tile."""
    ctx, torch, capi = env
    B, H, D, cap = len(lengths), 12, 64, 4096  # so many heads that two sequences reach the streaming kernel
    rng = np.random.default_rng(4)
    q, k, v = rng.standard_normal((B, H, D), dtype=np.float32), rng.standard_normal((B, H, cap, D), dtype=np.float32), rng.standard_normal((B, H, cap, D), dtype=np.float32)
    out, kd, vd = torch.full((B, H, D), float("nan"), device="cuda"), torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
    for b, n in enumerate(lengths):
        kd[b, :, n:] = float("nan")
        vd[b, :, n:] = float("nan")
    before = ctx.ctx_launch_count_named(b"window_attention_stream")
    at = (D, H * cap * D, cap * D)
    got = []
    for _ in range(2):
        ctx.window_attention_step_f32(B, H, D, out, H * D, D, torch.from_numpy(q).cuda(), H * D, D, kd, *at, vd, *at, cap, torch.tensor(lengths, device="cuda"), 0.125, 3000, 5, None, 0, None)
        ctx.sync()
        got.append(out.clone())
    assert ctx.ctx_launch_count_named(b"window_attention_stream") == before + 2
    assert torch.equal(*got)
    assert max_abs_rel(out.cpu().numpy(), R.step(q, k, v, lengths, 0.125, 3000, 5)) < TOL


def test_a_cache_beyond_32_bits_of_offsets(env):
    """The last sequence's rows lie more than 2^32 elements behind the first one's."""
    ctx, torch, capi = env
    rows, D, gap = 300, 64, (1 << 32) + 64
    k = torch.empty(gap + rows * D, device="cuda")
    rng = np.random.default_rng(2)
    data = rng.standard_normal((2, 1, rows, D), dtype=np.float32)
    for b in range(2):
        k[b * gap:b * gap + rows * D] = torch.from_numpy(data[b].reshape(-1)).cuda()
    q, lengths, out = rng.standard_normal((2, 1, D), dtype=np.float32), np.array([rows, rows - 7]), torch.empty(2, 1, D, device="cuda")
    ctx.window_attention_step_f32(2, 1, D, out, D, D, torch.from_numpy(q).cuda(), D, D, k, D, gap, 0, k, D, gap, 0, rows, torch.from_numpy(lengths).cuda(), 0.125, 100, 1, None, 0, None)
    ctx.sync()
    assert max_abs_rel(out.cpu().numpy(), R.step(q, data, data, lengths, 0.125, 100, 1)) < TOL


def test_a_length_outside_its_cache_is_reported(env):
    ctx, torch, capi = env
    x, out = torch.ones(2, 4, 1, 8, device="cuda"), torch.full((2, 1, 8), 5.0, device="cuda")
    big, big_out, at = torch.ones(2, 40000, 1, 64, device="cuda"), torch.full((2, 1, 64), 5.0, device="cuda"), (64, 40000 * 64, 64)
    ctx.window_attention_step_f32(2, 1, 64, big_out, 64, 64, big_out, 64, 64, big, *at, big, *at, 40000, torch.tensor([40001, 4000], device="cuda"), 1.0, 0, 0, None, 0, None)
    with pytest.raises(capi.GcbError) as e:
        ctx.sync()
    assert e.value.status == capi.INVALID_ARG
    assert (big_out[0] == 0).all() and ((big_out[1] - 1).abs() < 1e-6).all()
    for bad in (5, -1, 1 << 40):
        ctx.window_attention_step_f32(2, 1, 8, out, 8, 8, x, 8, 8, x, 8, 32, 8, x, 8, 32, 8, 4, torch.tensor([3, bad], device="cuda"), 1.0, 0, 0, None, 0, None)
        with pytest.raises(capi.GcbError) as e:
            ctx.sync()
        assert e.value.status == capi.INVALID_ARG
        assert (out[0] == 1).all() and (out[1] == 0).all()
    for kw in (dict(D=129), dict(cap=1 << 30)):
        with pytest.raises(capi.GcbError) as e:
            ctx.window_attention_step_f32(2, 1, kw.get("D", 8), out, 8, 8, x, 8, 8, x, 8, 32, 8, x, 8, 32, 8, kw.get("cap", 4), torch.tensor([3, 3], device="cuda"), 1.0, 0, 0, None, 0, None)
        assert e.value.status == capi.UNSUPPORTED


def test_single_positions_continue_what_a_forward_pass_began(env):
    """Row t of a forward pass over a sequence is the single-token form at length t + 1, over the same keys and values."""
    ctx, torch, capi = env
    B, H, T, D = 2, 3, 150, 64
    c = Case(torch, B, H, T, D, 16, 64)
    c.forward(ctx, 40, 2, 0.125)
    out = torch.empty(B, H, D, device="cuda")
    for t in (0, 1, 41, 42, 149):
        ctx.window_attention_step_f32(B, H, D, out, H * D, D, c.dev["q"][0][:, :, t].contiguous(), H * D, D, *c.arg("k"), *c.arg("v"), T, torch.full((B,), t + 1, device="cuda"), *c.rule)
        ctx.sync()
        assert max_abs_rel(out.cpu().numpy(), c.out[:, :, t].cpu().numpy()) < TOL


def test_two_contexts_at_once(env):
    """Calls of two contexts on streams of their own, queued in turn without waiting, give what each gives alone."""
    _, torch, capi = env
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [capi.Context(0, s.cuda_stream) for s in streams]
    sizes = [(4, 8, 700, 64), (2, 6, 300, 128)]
    cases = [Case(torch, *size, 16, 64, seed=i) for i, size in enumerate(sizes)]
    rng = np.random.default_rng(8)
    n, H, cap, D = 8, 16, 4096, 64
    lengths = torch.from_numpy(rng.integers(1, cap, n)).cuda()
    caches = [torch.randn(2, n, cap, H, D, device="cuda") for _ in range(2)]
    q = torch.randn(n, H, D, device="cuda")
    outs = [torch.empty(n, H, D, device="cuda") for _ in range(2)]

    def calls(i):
        with torch.cuda.stream(streams[i]):
            cases[i].forward(ctxs[i], 100, 3, 0.125)
            cases[i].backward(ctxs[i])
            at = (H * D, cap * H * D, D)
            ctxs[i].window_attention_step_f32(n, H, D, outs[i], H * D, D, q, H * D, D, caches[i][0], *at, caches[i][1], *at, cap, lengths, 0.125, 0, 0, None, 0, None)

    def results(i):
        return [t.clone() for t in [cases[i].out, cases[i].dbias, outs[i]] + cases[i].grads]

    torch.cuda.synchronize()
    alone = []
    for i in range(2):
        calls(i)
        torch.cuda.synchronize()
        alone.append(results(i))
    for _ in range(5):
        for i in range(2):
            calls(i)
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(results(i), alone[i]))
        ctxs[i].sync()
        ctxs[i].close()
