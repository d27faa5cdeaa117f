"""Attention under a visibility rule, its gradients and its single-token form, in 64 bits from the definitions, and dropout's mask."""
import numpy as np


def bucket_starts(buckets, reach):
    """The first half of the buckets one distance each, then a constant factor up to `reach`: bucket e + k of e + m starts at the least n
    with (n / e)^m >= (reach / e)^k, in whole numbers."""
    e = max(1, buckets // 2)
    m, far = buckets - e, max(reach, e)
    out = list(range(e))
    for k in range(m):
        lo, hi = 0, far
        while hi - lo > 1:
            mid = (lo + hi) // 2
            if mid**m * e**k < far**k * e**m:
                lo = mid
            else:
                hi = mid
        out.append(hi)
    return np.array(out, np.int64)


def visible(i, j, window, sinks):
    return (j <= i) & ((i - j < window) | (j < sinks) if window else True)


def bias_of(bias, starts, distance):
    """(H, ...) bias of an array of distances (those below zero: anything finite)."""
    return bias[:, np.maximum(np.searchsorted(starts, np.maximum(distance, 0), side="right") - 1, 0)]


def attention(q, k, v, scale, window=0, sinks=0, bias=None, starts=None, dout=None):
    """(B, H, T, D) arrays -> out, or (out, dq, dk, dv, dbias) with `dout`."""
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    i = np.arange(q.shape[2])
    dist = i[:, None] - i[None, :]
    s = scale * (q @ k.swapaxes(2, 3))
    if bias is not None:
        s = s + bias_of(bias.astype(np.float64), starts, dist)[None]
    s = np.where(visible(i[:, None], i[None, :], window, sinks), s, -np.inf)
    m = s.max(3, keepdims=True)
    p = np.exp(s - np.where(np.isfinite(m), m, 0.0))
    total = p.sum(3, keepdims=True)
    p = np.divide(p, total, out=np.zeros_like(p), where=total > 0)
    out = p @ v
    if dout is None:
        return out
    g = dout.astype(np.float64)
    ds = p * (g @ v.swapaxes(2, 3) - (g * out).sum(3, keepdims=True))
    dbias = None
    if bias is not None:
        n = np.searchsorted(starts, np.maximum(dist, 0), side="right") - 1
        dbias = np.stack([[ds[:, h][:, n == b].sum() for b in range(len(starts))] for h in range(q.shape[1])])
    return out, scale * (ds @ k), scale * (ds.swapaxes(2, 3) @ q), p.swapaxes(2, 3) @ g, dbias


def step(q, k, v, lengths, scale, window=0, sinks=0, bias=None, starts=None):
    """q (B, H, D), caches (B, H, cap, D) -> (B, H, D)."""
    out = np.zeros(q.shape)
    for b, n in enumerate(lengths):
        j = np.arange(n)
        j = j[visible(n - 1, j, window, sinks)]
        if not len(j):
            continue
        s = scale * np.einsum("hd,hjd->hj", q[b].astype(np.float64), k[b][:, j].astype(np.float64))
        if bias is not None:
            s = s + bias_of(bias.astype(np.float64), starts, n - 1 - j)
        m = s.max(1, keepdims=True)
        p = np.exp(s - np.where(np.isfinite(m), m, 0.0))
        total = p.sum(1, keepdims=True)
        out[b] = np.einsum("hj,hjd->hd", np.divide(p, total, out=np.zeros_like(p), where=total > 0), v[b][:, j].astype(np.float64))
    return out


def philox_words(n, seed, offset):
    """The first n words of Philox4x32-10 from the counter `offset` on, one block after another."""
    out = []
    for block in range((n + 3) // 4):
        at = (offset + block) % 2**64
        c, k = [at % 2**32, at >> 32, 0, 0], [seed % 2**32, (seed >> 32) % 2**32]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b % 2**32, (a >> 32) ^ c[3] ^ k[1], a % 2**32]
            k = [(k[0] + 0x9E3779B9) % 2**32, (k[1] + 0xBB67AE85) % 2**32]
        out += c
    return np.array(out[:n], np.uint64)


def kept(n, p, seed, offset):
    return philox_words(n, seed, offset) >= np.uint64(int(float(np.float32(p)) * 2.0**32)) if p < 1 else np.zeros(n, bool)
