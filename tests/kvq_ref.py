"""The quantised key/value cache in numpy and 64 bits: what is held for given rows, and attention over it, with a bound
on what an implementation in fp32 sums and bfloat16 products may differ by."""
import numpy as np

GROUP = 32


def hold(x, bits):
    """(codes from 0, scales) of x [..., D] (float32 values): the definition, decided exactly."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    most = np.abs(g).max(-1)
    top = 7 if bits == 4 else 127
    with np.errstate(all="ignore"):
        t = most * (np.float32(1) / np.float32(top))
    cut = 20 if bits == 4 else 23
    s = (((t.view(np.uint32).astype(np.uint64) + (1 << cut) - 1) >> cut) << cut).astype(np.uint32).view(np.float32)
    fine = most < np.float32(2.0) ** 100          # False for NaN
    s = np.where(fine, s, np.float32(np.nan))
    with np.errstate(all="ignore"):
        c = np.rint(g.astype(np.float64) / s.astype(np.float64)[..., None])
    c = np.where((s > 0)[..., None], c, 0.0)
    assert np.abs(c).max(initial=0) <= top
    return (c.reshape(x.shape) + 2 ** (bits - 1)).astype(np.uint8), s


def pack(u, bits):
    return u if bits == 8 else (u[..., 0::2] | (u[..., 1::2] << 4)).astype(np.uint8)


def values(u, s, bits):
    c = u.astype(np.float64) - 2 ** (bits - 1)
    return (c.reshape(*c.shape[:-1], -1, GROUP) * s.astype(np.float64)[..., None]).reshape(c.shape)


def sees(i, n, window, sinks):
    """[n] truth values: what a query at position i sees of positions 0 .. n - 1."""
    j = np.arange(n)
    ok = j <= i
    if window:
        ok &= (i - j < window) | (j < sinks)
    return ok


def attention(q, k, v, pos, count, window=0, sinks=0, scale=None, split_q=True, out_bits=24):
    """q [T, H, D], k, v [Hk, n, D] of one sequence (float64). Returns (out [T, H, D], bound of the difference).

    The bound, with u = 2^-24: a score is off by scale * sum|q k| * (2^-16 where q is split into two bfloat16 terms, D * 2u for
    the sum) and by 8u of its size in the log2 domain's arithmetic; twice that moves the weights (numerator and
    denominator); a probability is off by 2^-16 (two terms, half a step of 2^-8 each) or 2^-8 (one), its exponential by 2^-21; sums over n positions go
    in steps of 16, off by 2u each, and through at most 64 joins; what is below 2^-126
    (before it meets a value) may be zero, and fp16 probabilities, held times 2^7 relative to a maximum that is at most the
    row's (so that the sum is 1 or more), are off by half of fp16's smallest step: 2^-25 / 2^7; the result is rounded to its type."""
    T, H, D = q.shape
    Hk, n, _ = k.shape
    u = 2.0 ** -24
    scale = D ** -0.5 if scale is None else scale
    out, tol = np.zeros((T, H, D)), np.zeros((T, H, D))
    for t in range(min(T, count)):
        i = pos + t
        if i < 0 or i >= n:
            continue
        ok = sees(i, n, window, sinks)
        for h in range(H):
            kk, vv = k[h * Hk // H][ok], v[h * Hk // H][ok]
            z = kk @ q[t, h] * scale
            size = np.abs(kk) @ np.abs(q[t, h]) * scale
            w = np.exp(z - z.max())
            w /= w.sum()
            out[t, h] = w @ vv
            m = len(z)
            off = (size * ((2.0 ** -16 if split_q else 0.0) + 2 * D * u) + 8 * u * (np.abs(z) + np.abs(z).max())).max()
            rel = np.expm1(2 * off) + (2.0 ** -16 if split_q else 2.0 ** -8) + 2.0 ** -21 + 2 * u * (m / 16 + 64)
            tol[t, h] = (1 + 2.0 ** -out_bits) * rel * (w @ np.abs(vv)) + 2.0 ** -out_bits * np.abs(out[t, h]) + (2.0 ** -126 + 2.0 ** -32) * np.abs(vv).sum(0)
    return out, tol
