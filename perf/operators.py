"""The work that attention under a visibility rule and dropout are timed on, case by case.

Three kinds of pass, each through the C ABI (`gradcraft_b200.capi.Context`) where `own` is set and in elementary torch operations
where it is not:

  attention   causal attention with a sliding window, a few first positions that stay visible (sinks) and a learned bias by distance
              bucket: forward, or forward and backward with the gradients of q, k, v and the bias table
  step        the same for the newest position of every sequence, over keys and values in a cache
  dropout     residual + dropout(x) with a mask that follows from a seed and a counter, and its backward

`listed()` gives the fixed cases, `draw()` further ones of the same ranges; `prepare()` makes everything from the seed, `run()` makes
one pass, `exact()` gives the same outputs from the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False


def _attention(name, B, H, T, D, window, sinks, buckets=0, reach=0, train=True):
    """`buckets`: rows of the bias table a head (0: no bias), `reach`: the distance from which on all are in the last bucket."""
    return dict(name=name, kind="attention", B=B, H=H, T=T, D=D, window=window, sinks=sinks, buckets=buckets, reach=reach, train=train)


def _step(name, B, H, D, cap, window, sinks, buckets=0, reach=0, full=True):
    return dict(name=name, kind="step", B=B, H=H, D=D, cap=cap, window=window, sinks=sinks, buckets=buckets, reach=reach, full=full)


def listed():
    return [
        # ---- attention: q, k and v as the projections leave them, (B, T, H, D) in memory
        # a step of the two-layer model a user tries things out on: launches and latency are what counts
        _attention("attention_tiny", 4, 4, 64, 32, 16, 2),
        # document lengths that are no multiple of anything, bias and window together
        _attention("attention_odd_sizes", 5, 6, 331, 64, 100, 3, 32, 128),
        # the sizes that GPTConfig has by default with a bias by distance instead of a window
        _attention("attention_bias_default_config", 8, 12, 512, 64, 0, 0, 32, 128),
        # heads of the 180M-parameter model that look back 256 positions
        _attention("attention_window_180m", 16, 16, 1024, 64, 256, 4),
        # a long document, the length at which a window is what makes training possible
        _attention("attention_long", 1, 16, 8192, 64, 1024, 4, 32, 512),
        # evaluating a prompt: forward alone
        _attention("attention_prompt", 1, 12, 4099, 64, 512, 16, train=False),
        # ---- one token of every sequence against its cache
        # one conversation with a small model
        _step("step_small", 1, 12, 64, 385, 0, 0),
        # long conversations of different lengths, everything visible, bias by distance
        _step("step_long_ragged", 8, 16, 64, 16384, 0, 0, 32, 512, full=False),
        # a batch of long streams of which a window and the first positions are looked at
        _step("step_window_batch", 64, 16, 64, 4096, 1024, 4),
        # ---- dropout on a residual branch, forward and backward
        # 256 tokens of the two-layer model
        dict(name="dropout_tiny", kind="dropout", rows=256, cols=128, p=0.1, residual=True),
        # 32 sequences of 1024 tokens, the 180M-parameter model
        dict(name="dropout_180m", kind="dropout", rows=32768, cols=1024, p=0.1, residual=True),
        # a width that is no multiple of four, no residual
        dict(name="dropout_odd_width", kind="dropout", rows=1655, cols=771, p=0.25, residual=False),
    ]


# ---- drawing further cases ------------------------------------------------------------------------------------------------
def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _rule(rng, T):
    window = rng.choice([0, _log_int(rng, min(2, T), T), _log_int(rng, min(2, T), T)])
    return dict(window=window, sinks=rng.choice([0, 1, 4, rng.randint(0, 64)]) if window else 0)


def _table(rng):
    buckets = rng.choice([0, 0, 8, 32, rng.randint(1, 64)])
    return dict(buckets=buckets, reach=_log_int(rng, max(2, buckets), 1024) if buckets else 0)


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "step", "step", "dropout"])
    if kind == "attention":
        while True:
            T = _log_int(rng, 1, 8192)
            c = dict(kind=kind, B=_log_int(rng, 1, 32), H=rng.randint(1, 16), T=T, D=rng.choice([16, 24, 32, 40, 64, 64, 64, 96, 128]), train=rng.random() < 0.7)
            c.update(_rule(rng, T), **_table(rng))
            if c["train"] and (T == 1 or c["window"] == 1 or c["buckets"] == 1):
                continue  # a query that sees one key, or a table of one value, has no gradient but rounding noise
            if c["B"] * c["H"] * T * T <= (1 << 28) and work(c)["flops"] < 5e10:
                return c
    if kind == "step":
        while True:
            cap = _log_int(rng, 1, 16384)
            c = dict(kind=kind, B=_log_int(rng, 1, 64), H=rng.randint(1, 16), D=rng.choice([16, 32, 40, 64, 64, 96, 128]), cap=cap, full=rng.random() < 0.5)
            c.update(_rule(rng, cap), **_table(rng))
            if c["B"] * c["H"] * c["D"] * cap <= (1 << 26):
                return c
    cols = _log_int(rng, 1, 4096)
    return dict(kind=kind, rows=_log_int(rng, 1, max(1, (1 << 25) // cols)), cols=cols, p=rng.choice([0.0, 0.05, 0.1, 0.5, round(rng.uniform(0.01, 0.9), 3)]), residual=rng.random() < 0.6)


# ---- state ----------------------------------------------------------------------------------------------------------------
def _bucket_starts(buckets, reach):
    """First distance of every bucket: the first half holds one distance each, the others grow by a constant factor up to `reach`.
    Bucket e + k of e + m starts at the least n with n >= e (reach / e)^(k / m), found in whole numbers."""
    e = max(1, buckets // 2)
    m = buckets - e
    starts = list(range(min(e, buckets)))
    for k in range(m):
        n = max(1, int(e * (max(reach, e) / e) ** (k / m)) - 2)
        while n**m * e**k < max(reach, e) ** k * e**m:
            n += 1
        starts.append(n)
    return starts


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda") * scale

    s = dict(case=case)
    if case["kind"] == "dropout":
        s["x"], s["dy"] = normal(case["rows"], case["cols"]), normal(case["rows"], case["cols"])
        s["residual"] = normal(case["rows"], case["cols"]) if case["residual"] else None
        s["seed"], s["offset"] = seed * 0x9E3779B97F4A7C15 % (1 << 62), (seed * 7919 % (1 << 20)) + (1 << 32) - 5000
        s["out"], s["dx"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
        return s
    B, H, D = case["B"], case["H"], case["D"]
    s["scale"] = 1.0 / math.sqrt(D)
    s["bias"] = normal(H, case["buckets"], scale=0.5) if case["buckets"] else None
    s["starts"] = np.array(_bucket_starts(case["buckets"], case["reach"]), np.int64) if case["buckets"] else None
    if case["kind"] == "step":
        cap = case["cap"]
        s["q"], s["k"], s["v"], s["out"] = normal(B, H, D), normal(B, cap, H, D), normal(B, cap, H, D), torch.empty(B, H, D, device="cuda")
        s["lengths"] = torch.full((B,), cap, dtype=torch.int64, device="cuda") if case["full"] else torch.randint(1, cap + 1, (B,), generator=g, device="cuda")
        return s
    T = case["T"]
    for name in ("q", "k", "v", "dout"):
        s[name] = normal(B, T, H, D)
    for name in ("out", "dq", "dk", "dv"):
        s[name] = torch.empty(B, T, H, D, device="cuda")
    s["dbias"] = torch.empty_like(s["bias"]) if case["buckets"] else None
    return s


# ---- the framework's calls ------------------------------------------------------------------------------------------------
_contexts = {}


def _context():
    """One context for every stream a program launches on.  The default stream's handle is 0 on every device, and a stream that is gone may leave its
    handle to another one: contexts go by device and stream, and hold on to the stream."""
    from gradcraft_b200 import capi

    device, stream = torch.cuda.current_device(), torch.cuda.current_stream()
    key = device, stream.cuda_stream
    if key not in _contexts:
        _contexts[key] = capi.Context(device, stream.cuda_stream), stream
    return _contexts[key][0]


def _own_attention(s):
    c, ctx = s["case"], _context()
    B, H, T, D = c["B"], c["H"], c["T"], c["D"]
    at = (H * D, T * H * D, D)  # strides of a row, a sequence, a head
    rule = (s["scale"], c["window"], c["sinks"], s["bias"], c["buckets"], s["starts"])
    stats = torch.empty(ctx.lib.attention_stats_floats(B, H, T), device="cuda")
    ctx.window_attention_fwd_f32(B, H, T, D, s["out"], *at, stats, s["q"], *at, s["k"], *at, s["v"], *at, *rule)
    if not c["train"]:
        return s["out"]
    ctx.window_attention_bwd_f32(B, H, T, D, s["dq"], s["dk"], s["dv"], *at, s["dbias"], 0, s["dout"], *at, s["out"], *at, stats, s["q"], *at, s["k"], *at, s["v"], *at, *rule)
    return [s[n] for n in ("out", "dq", "dk", "dv") + (("dbias",) if c["buckets"] else ())]


def _own_step(s):
    c = s["case"]
    B, H, D, cap = c["B"], c["H"], c["D"], c["cap"]
    at = (H * D, cap * H * D, D)
    _context().window_attention_step_f32(B, H, D, s["out"], H * D, D, s["q"], H * D, D, s["k"], *at, s["v"], *at, cap, s["lengths"], s["scale"], c["window"], c["sinks"], s["bias"], c["buckets"], s["starts"])
    return s["out"]


def _own_dropout(s):
    c, ctx, n = s["case"], _context(), s["x"].numel()
    ctx.dropout_fwd_f32(s["out"], s["x"], s["residual"], n, c["p"], s["seed"], s["offset"])
    ctx.dropout_bwd_f32(s["dx"], s["dy"], n, c["p"], s["seed"], s["offset"], 0)
    return [s["out"], s["dx"]]


# ---- plain forms ----------------------------------------------------------------------------------------------------------
def _buckets(s, distance):
    starts = torch.from_numpy(s["starts"]).to(distance.device)
    return torch.searchsorted(starts, distance.clamp(min=0), right=True) - 1


def _plain_attention(s):
    c = s["case"]
    q, k, v, dout = (s[n].transpose(1, 2) for n in ("q", "k", "v", "dout"))  # (B, H, T, D)
    i = torch.arange(c["T"], device=q.device)
    distance = i[:, None] - i[None, :]
    seen = distance >= 0
    if c["window"]:
        seen = seen & ((distance < c["window"]) | (i[None, :] < c["sinks"]))
    scores = q @ k.transpose(2, 3) * s["scale"]
    if c["buckets"]:
        scores += s["bias"][:, _buckets(s, distance)]
    scores.masked_fill_(~seen, -math.inf)
    scores -= scores.amax(3, keepdim=True)
    p = scores.exp_()
    p /= p.sum(3, keepdim=True)
    out = p @ v
    if not c["train"]:
        return out.transpose(1, 2)
    dv = p.transpose(2, 3) @ dout
    ds = dout @ v.transpose(2, 3)
    ds -= (dout * out).sum(3, keepdim=True)
    ds *= p
    dq, dk = ds @ k * s["scale"], ds.transpose(2, 3) @ q * s["scale"]
    got = [t.transpose(1, 2) for t in (out, dq, dk, dv)]
    if c["buckets"]:
        # a bucket's keys lie side by side in a row: differences of running sums, in 64 bits as they cancel
        upto = torch.nn.functional.pad(ds.sum(0, dtype=torch.float64).cumsum(2), (1, 0))
        edges = torch.tensor([*s["starts"].tolist(), max(c["T"], int(s["starts"][-1]))], device=q.device)
        count = (i[:, None] + 1 - edges).clamp(min=0)
        at = upto.gather(2, count.expand(c["H"], -1, -1)).sum(1)
        got.append((at[:, :-1] - at[:, 1:]).float())
    return got


def _plain_step(s):
    c = s["case"]
    last = s["lengths"][:, None] - 1
    j = torch.arange(c["cap"], device=last.device)[None, :]
    distance = last - j
    seen = distance >= 0
    if c["window"]:
        seen = seen & ((distance < c["window"]) | (j < c["sinks"]))
    scores = (s["q"][:, None] * s["k"]).sum(3).transpose(1, 2) * s["scale"]  # (B, H, cap)
    if c["buckets"]:
        scores = scores + s["bias"][:, _buckets(s, distance)].transpose(0, 1)
    scores = scores.masked_fill(~seen[:, None], -math.inf)
    p = (scores - scores.amax(2, keepdim=True)).exp()
    p = p / p.sum(2, keepdim=True)
    return (p.transpose(1, 2)[..., None] * s["v"]).sum(1)


def _philox(blocks, seed):
    """Philox4x32-10 on the 64-bit counters `blocks`: (n, 4) words in int64."""
    low = 0xFFFFFFFF
    c0, c1, c2, c3 = blocks & low, (blocks >> 32) & low, torch.zeros_like(blocks), torch.zeros_like(blocks)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], 1)


def _plain_dropout(s):
    x, n = s["x"], s["x"].numel()
    p = float(np.float32(s["case"]["p"]))
    words = _philox(s["offset"] + torch.arange((n + 3) // 4, device=x.device), s["seed"]).flatten()[:n]
    factor = (words >= int(p * 2.0**32)).view_as(x).float() * (1.0 / (1.0 - p))
    out = x * factor
    if s["residual"] is not None:
        out = s["residual"] + out
    return [out, s["dy"] * factor]


def run(state):
    if own:
        return dict(attention=_own_attention, step=_own_step, dropout=_own_dropout)[state["case"]["kind"]](state)
    return dict(attention=_plain_attention, step=_plain_step, dropout=_plain_dropout)[state["case"]["kind"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def _pairs(last, window, sinks):
    """Visible keys of a query at position `last`."""
    if not window or last < window:
        return last + 1
    return window + min(sinks, last + 1 - window)


def work(case):
    if case["kind"] == "dropout":
        n = case["rows"] * case["cols"]
        return dict(bytes=n * (20 if case["residual"] else 16), flops=3 * n)
    B, H, D = case["B"], case["H"], case["D"]
    if case["kind"] == "step":
        # lengths are spread evenly over the cache where they differ: half of it is looked at on average
        seen = _pairs(case["cap"] - 1, case["window"], case["sinks"]) if case["full"] else sum(_pairs(case["cap"] * (2 * i + 1) // 32, case["window"], case["sinks"]) for i in range(16)) / 16
        return dict(bytes=int(B * H * D * 4 * (2 * seen + 2)), flops=int(4 * B * H * D * seen))
    T = case["T"]
    full = min(T, case["window"]) if case["window"] else T  # rows below this see everything before them
    pairs = full * (full + 1) // 2 + sum(_pairs(t, case["window"], case["sinks"]) for t in range(full, T))
    tensors = 8 if case["train"] else 4  # q k v dout in, out dq dk dv out
    return dict(bytes=4 * tensors * B * H * T * D, flops=(14 if case["train"] else 4) * B * H * D * pairs)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------
def _exact_bias(s, h, distance):
    if s["bias"] is None:
        return 0.0
    edges = torch.tensor([int(x) for x in s["starts"]] + [1 << 62], device=distance.device)
    return sum(s["bias"][h, n].double() * ((distance >= edges[n]) & (distance < edges[n + 1])) for n in range(len(edges) - 1))


def _exact_dropout(s):
    n, p = s["x"].numel(), float(np.float32(s["case"]["p"]))
    block = np.uint64(s["offset"]) + np.arange((n + 3) // 4, dtype=np.uint64)
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    ctr = [block & low, block >> half, np.zeros_like(block), np.zeros_like(block)]
    key = [s["seed"] % 2**32, s["seed"] // 2**32]
    for _ in range(10):
        left, right = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(right >> half) ^ ctr[1] ^ np.uint64(key[0]), right & low, (left >> half) ^ ctr[3] ^ np.uint64(key[1]), left & low]
        key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
    kept = torch.from_numpy((np.stack(ctr, 1).reshape(-1)[:n] >= np.uint64(int(p * 2.0**32)))).to(s["x"].device).view_as(s["x"])
    out, dx = (torch.where(kept, t.double() / (1.0 - p), torch.zeros_like(t, dtype=torch.float64)) for t in (s["x"], s["dy"]))
    return [out if s["residual"] is None else out + s["residual"].double(), dx]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "dropout":
        return _exact_dropout(s)
    B, H, D, W, S = (case[n] for n in ("B", "H", "D", "window", "sinks"))
    if case["kind"] == "step":
        out = torch.empty(B, H, D, dtype=torch.float64, device="cuda")
        for b in range(B):
            last = int(s["lengths"][b]) - 1
            j = torch.arange(last + 1, device="cuda")
            j = j[(j > last - W) | (j < S)] if W else j
            for h in range(H):
                z = s["k"][b, j, h].double() @ s["q"][b, h].double() / math.sqrt(D) + _exact_bias(s, h, last - j)
                out[b, h] = torch.softmax(z, 0) @ s["v"][b, j, h].double()
        return out
    T = case["T"]
    out = torch.empty(B, T, H, D, dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.empty_like(out) for _ in range(3))
    dbias = torch.zeros(H, case["buckets"], dtype=torch.float64, device="cuda")
    i = torch.arange(T, device="cuda")
    distance = i[:, None] - i[None, :]
    hidden = (distance < 0) | ((distance >= W) & (i >= S)[None, :]) if W else distance < 0
    edges = [int(x) for x in s["starts"]] + [1 << 62] if case["buckets"] else []
    for h in range(H):
        bias = _exact_bias(s, h, distance)
        total = torch.zeros(T, T, dtype=torch.float64, device="cuda") if edges and case["train"] else None
        for b in range(B):
            q, k, v, do = (s[n][b, :, h].double() for n in ("q", "k", "v", "dout"))
            p = torch.softmax(((q @ k.T) / math.sqrt(D) + bias).masked_fill(hidden, -math.inf), 1)
            out[b, :, h] = p @ v
            if not case["train"]:
                continue
            dv[b, :, h] = p.T @ do
            dp = do @ v.T
            ds = p * (dp - (p * dp).sum(1, keepdim=True))
            dq[b, :, h], dk[b, :, h] = ds @ k / math.sqrt(D), ds.T @ q / math.sqrt(D)
            if edges:
                total += ds
        if total is not None:
            dbias[h] = torch.stack([total[(distance >= edges[n]) & (distance < edges[n + 1])].sum() for n in range(case["buckets"])])
    if not case["train"]:
        return out
    return [out, dq, dk, dv] + ([dbias] if case["buckets"] else [])
