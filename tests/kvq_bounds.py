"""What attention over the quantised cache may differ by from 64 bits, from the kernels' terms: a bound a position, so that it
holds, and stays narrow, where one position's score is far larger than the others'."""
import numpy as np

from tests import kvq_ref as R


def lse(z):
    m = z.max()
    return m + np.log(np.exp(z - m).sum())


def attention(q, k, v, pos, count, window=0, sinks=0, scale=None, fp32=True, few_rows=True):
    """q [T, H, D], k, v [Hk, n, D] of one sequence (float64). Returns (out [T, H, D], bound of the difference); few_rows: at most 16
    query rows a key/value head (the token kernel), else the prompt kernel.

    With u = 2^-24, all bounds are sums of:
    a score: queries in two fp16 terms are off by 2^-22 of their own size, or by 2^-31 of the row's largest (half of fp16's smallest
    step, 2^-25, beside a largest value of 64 or more); the tensor cores cut sums of 16 products off, by 2^-23 of the sum of magnitudes,
    in 2 D / 16 steps at most, and no more of them than there are products that are not zero, in two terms; the way into the log2 domain and the distance from the reference point round a few times, by u of either;
    what that does to the weights is formed position by position, from the scores moved up and down;
    a probability: the exponential is off by 2^-22 and its terms by 2^-22 (two of fp16, three of bfloat16 are less), in bfloat16 outputs
    by 2^-16 (two bfloat16 terms, few rows) or 2^-11 (one of fp16, many rows); fp16 terms, held times 2^7 beside a sum of 1 or more, lose
    half a step of 2^-24 each where they are subnormal: 2^-25 / 2^7 = 2^-32 with one term; of two terms, the first is cut to 11 bits and
    what is left is formed from that cut number, so that the rounding of neither makes up for the other's: 2^-31; what is below
    2^-126 may be zero;
    sums over positions: of 16 products, in two or three terms, cut off by 2^-23 each; a new accumulator after 64 of them
    (fp32 outputs), then fp32 additions, through 64 joins at most and no more than there are steps; the same number of them for the sum of the probabilities;
    the result: half a step of its type."""
    T, H, D = q.shape
    Hk, n, _ = k.shape
    u = 2.0 ** -24
    scale = D ** -0.5 if scale is None else scale
    out, tol = np.zeros((T, H, D)), np.zeros((T, H, D))
    p_off = 2.0 ** -21 if fp32 else 2.0 ** -16 + 2.0 ** -22 if few_rows else 2.0 ** -11 + 2.0 ** -22
    half = 2.0 ** -24 if fp32 else 2.0 ** -8
    for t in range(min(T, count)):
        i = pos + t
        if i < 0 or i >= n:
            continue
        ok = R.sees(i, n, window, sinks)
        for h in range(H):
            kk, vv, qq = k[h * Hk // H][ok], v[h * Hk // H][ok], q[t, h]
            z = kk @ qq * scale
            size = np.abs(kk) @ np.abs(qq) * abs(scale)
            top = np.abs(qq).max(initial=0.0) * np.abs(kk).sum(1) * abs(scale)
            cuts = np.minimum(D / 8, 2 * np.count_nonzero(kk * qq, axis=1))
            w = np.exp(z - lse(z))
            out[t, h] = w @ vv
            off = size * (2.0 ** -22 + cuts * 2.0 ** -23) + 2.0 ** -31 * top + 4 * u * (np.abs(z) + abs(z.max()))
            hi, lo = z + off, z - off
            up = np.minimum(np.exp(np.minimum(hi - lse(lo), 0.0)), 1.0) - w
            down = w - np.exp(lo - lse(hi))
            steps = -(-len(z) // 16)
            sums = (min(3 * steps, 64) if fp32 else 3 * steps) * 2.0 ** -23 + 2 * u * (steps / 64 + min(steps, 64))
            tol[t, h] = (np.maximum(np.maximum(up, down), 0.0) @ np.abs(vv) + (p_off + sums) * (w @ np.abs(vv))
                         + ((2.0 ** -31 if fp32 else 2.0 ** -32) + 2.0 ** -126) * np.abs(vv).sum(0)) * (1 + half) + half * np.abs(out[t, h])
    return out, tol


def compare(K, cache, q, pos, count=None, window=0, sinks=0, scale=None, n=None):
    """As check() of test_kvq_gpu.py, by this bound; pos and count: ints, or lists of one a sequence."""
    import torch

    from tests.test_kvq_gpu import host_values

    B, T, H = q.shape[:3]
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda") if isinstance(x, list) else x  # noqa: E731
    got = K.kvq_attention(q, cache, dev(pos), count=dev(count), window=window, sinks=sinks, scale=scale).double().cpu().numpy()
    ps = pos if isinstance(pos, list) else [pos] * B
    cs = count if isinstance(count, list) else [T] * B
    n = n or min(cache.capacity, max([p + c for p, c in zip(ps, cs)] + [1]))
    k, v = host_values(cache, n)
    qq = q.double().cpu().numpy()
    for b in range(B):
        want, tol = attention(qq[b], k[b], v[b], ps[b], cs[b], window, sinks, scale, fp32=q.dtype == torch.float32,
                              few_rows=T * H // cache.Hk <= 16)
        over = np.abs(got[b] - want) - tol
        assert over.max(initial=-1.0) <= 0, (b, over.max(), np.abs(got[b] - want).max(), tol.max())
        assert not got[b][cs[b]:].any()
    return got
