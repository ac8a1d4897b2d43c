"""The quantised cache at the edges of what its calls take, on the GPU; against numpy in 64 bits (tests/kvq_ref.py) where there are values."""
import numpy as np
import pytest
import torch

from tests import kvq_bounds as B
from tests.test_kvq_gpu import K, _status_clean, check, rnd  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("T,H", [(1, 4), (16, 4), (40, 6)])
def test_an_empty_batch(K, T, H):  # noqa: F811
    cache = K.kvq_cache(0, 2, 100, 64, 4)
    rows = torch.empty(0, T, 2, 64, device="cuda")
    K.kvq_write(cache, rows, rows, 0)
    assert K.kvq_attention(torch.empty(0, T, H, 64, device="cuda"), cache, 0).shape == (0, T, H, 64)
    assert K.kvq_read(cache, 0, 8)[0].shape == (0, 2, 8, 64)


# ---- values and keys of very different sizes ------------------------------------------------------
def wrote(K, k, v, bits):  # noqa: F811
    """A cache of exactly these rows [B, n, Hk, D]; what lies behind them is NaN."""
    batch, n, Hk, D = k.shape
    cache = K.kvq_cache(batch, Hk, n, D, bits)
    for i in (0, 2):
        cache.tensors[i].fill_(0xFF)
        cache.tensors[i + 1].fill_(float("nan"))
    K.kvq_write(cache, k.cuda(), v.cuda(), 0)
    return cache


SHAPES = [(1, 4, 2, 64), (3, 4, 2, 128), (40, 4, 2, 64), (129, 2, 2, 128), (150, 3, 1, 64)]   # T, H, Hk, D


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,H,Hk,D", SHAPES)
@pytest.mark.parametrize("lo,hi", [(-30, 30), (30, -30), (0, 20), (20, 0), (-90, 0)])
def test_values_that_grow_and_shrink_along_the_sequence(K, bits, dtype, T, H, Hk, D, lo, hi):  # noqa: F811
    """By powers of two that fit one range of fp16 (the sums are rescaled on the way) and by ones that do not."""
    n = 600
    k, v = rnd((1, n, Hk, D), 11, 0.3), rnd((1, n, Hk, D), 12)
    v = v * torch.exp2(torch.linspace(lo, hi, n).round()).reshape(1, n, 1, 1)
    cache, q = wrote(K, k, v, bits), rnd((1, T, H, D), 13, 1.0, dtype).cuda()
    check(K, cache, q, n - T)
    check(K, cache, q, 0, n=n)
    check(K, cache, q, 300 - T // 2, window=90, sinks=3, n=n)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("power", [20, 24, 25, 26, 27, 28, 40, 97])
def test_a_row_does_not_depend_on_sizes_that_it_cannot_see(K, bits, dtype, power):  # noqa: F811
    """One group of values, then one of keys, far larger than the others: the rows before it, and the ones whose window has left it,
    are as without it."""
    n, H, Hk, D, at = 256, 4, 2, 64, 100
    q = rnd((1, n, H, D), 21, 1.0, dtype).cuda()
    for which in (0, 1):
        x = [rnd((1, n, Hk, D), 22, 0.5), rnd((1, n, Hk, D), 23)]
        plain = wrote(K, *x, bits)
        x[which][0, at, 1, 32:] *= 2.0 ** power
        cache = wrote(K, *x, bits)
        for window, sinks in ((0, 0), (40, 2)):
            got = B.compare(K, cache, q, 0, window=window, sinks=sinks)
            want = K.kvq_attention(q, plain, 0, window=window, sinks=sinks).double().cpu().numpy()
            blind = [t for t in range(n) if t < at or (window and t >= at + window)]
            # both are within that bound of the same numbers; what they may differ by is twice that, and 2^-8 (2^-15) is more
            tol = 2.0 ** -7 if dtype == BF16 else 2.0 ** -14
            assert np.abs(got[0, blind] - want[0, blind]).max() <= tol * np.abs(want).max()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,H,Hk,D", SHAPES)
def test_keys_of_all_sizes(K, bits, dtype, T, H, Hk, D):  # noqa: F811
    """Positions whose keys are far larger, in columns in which the queries are zeros: their scores come from the small ones."""
    n = 500
    k, v = rnd((2, n, Hk, D), 31, 0.5), rnd((2, n, Hk, D), 32)
    q = rnd((2, T, H, D), 33, 1.0, dtype)
    q[..., 32:] = 0
    k[:, ::3, :, 32:] *= 2.0 ** 50
    k[:, 1::7, :, 32:] *= 2.0 ** -60
    cache = wrote(K, k, v, bits)
    check(K, cache, q.cuda(), [n - T, 100], n=n)
    check(K, cache, q.cuda(), [n - T, 200], [T, T // 2], window=130, sinks=2, n=n)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sizes_that_differ_beside_split_work_and_nan(K, bits, dtype):  # noqa: F811
    """Few row tiles over a long cache (parts that are joined), some sequences even and some not, and a NaN on top."""
    n, T, H, Hk, D = 3000, 20, 2, 1, 64
    k, v = rnd((3, n, Hk, D), 41, 0.3), rnd((3, n, Hk, D), 42)
    v[1] *= torch.exp2(torch.linspace(-40, 40, n).round()).reshape(n, 1, 1)
    v[2, 1500, 0, :32] *= 2.0 ** 60
    v[2, 2990, 0, 40] = float("nan")
    cache = wrote(K, k, v, bits)
    q = rnd((3, T, H, D), 43, 1.0, dtype).cuda()
    check(K, cache, q, n - T)
    check(K, cache, q, [n - T, 1495, 2400], [T, 11, T], n=n)


# ---- scores of all sizes --------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,H,Hk,D", SHAPES)
@pytest.mark.parametrize("power", [18, 22, 24, 26, 28, 31, 45, 80])
def test_large_scores(K, bits, dtype, T, H, Hk, D, power):  # noqa: F811
    """Scores far beyond the 24 bits in which fp32 holds a difference of one: one position has all the weight, or, where two keys are
    alike, both have half of it, whatever sign the scores have."""
    n = 400
    k, v = rnd((2, n, Hk, D), 61, 0.7), rnd((2, n, Hk, D), 62)
    k[:, 1::2] = k[:, ::2]
    q = rnd((2, T, H, D), 63) * 2.0 ** power
    cache = wrote(K, k, v, bits)
    B.compare(K, cache, q.to(dtype).cuda(), n - T)
    B.compare(K, cache, q.to(dtype).cuda(), [n - T, 150], window=70, sinks=2, n=n)
    low = wrote(K, k.abs() + 0.1, v, bits)            # all scores far below zero
    B.compare(K, low, -q.abs().to(dtype).cuda(), n - T)


# ---- queries of all sizes -------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,H,Hk,D", [(1, 4, 2, 64), (2, 6, 2, 128), (4, 6, 2, 64), (40, 4, 2, 128), (40, 4, 2, 64)])
@pytest.mark.parametrize("power", [-120, -90, 99, 107, 113, 119, 125])
def test_large_and_small_queries(K, bits, dtype, T, H, Hk, D, power):  # noqa: F811
    """Finite queries up to the type's largest: over keys as small (or large) as they are large, with ordinary scores, and one huge head beside
    ordinary ones."""
    n = 300
    k, v = rnd((2, n, Hk, D), 51, 0.7), rnd((2, n, Hk, D), 52)
    q = rnd((2, T, H, D), 53, 1.0, F32).clamp(-3.5, 3.5)
    cache = wrote(K, k * 2.0 ** -max(power, -90), v, bits)
    B.compare(K, cache, (q * 2.0 ** power).to(dtype).cuda(), n - T)
    if 0 < power < 120:
        q[:, :, 1] *= 2.0 ** power
        B.compare(K, wrote(K, k, v, bits), q.to(dtype).cuda(), n - T, window=100, sinks=3)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,H,Hk,D", [(1, 4, 2, 64), (5, 4, 2, 128), (40, 4, 2, 64)])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30, 1e30])
def test_scales_of_all_sizes(K, bits, dtype, T, H, Hk, D, scale):  # noqa: F811
    """Also where a factor of a row would overflow: its scores are zeros, queries and keys have no column in common."""
    n = 200
    k, v = rnd((1, n, Hk, D), 71, 0.7), rnd((1, n, Hk, D), 72)
    q = rnd((1, T, H, D), 73)
    if scale == 1e30:
        k[..., 32:] = 0
        q[..., :32] = 0
        q *= 2.0 ** 100
    B.compare(K, wrote(K, k, v, bits), q.to(dtype).cuda(), n - T, scale=scale)


# ---- sizes at which work is shared out differently ------------------------------------------------
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_more_parts_than_the_join_holds_at_a_time(K, bits, dtype):  # noqa: F811
    """One long sequence of one head on every CTA: more than 128 parts (the join takes them in rounds), with scores that grow."""
    n, H, D = 150000, 4, 64
    k, v = rnd((1, n, 1, D), 81, 0.4), rnd((1, n, 1, D), 82)
    k *= torch.linspace(0.5, 6, n).reshape(1, n, 1, 1)
    cache = wrote(K, k, v, bits)
    B.compare(K, cache, rnd((1, 1, H, D), 83, 1.0, dtype).cuda(), n - 1)
    B.compare(K, cache, rnd((1, 3, H, D), 84, 1.0, dtype).cuda(), n - 3)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_more_sequences_than_a_block_has_threads(K, dtype):  # noqa: F811
    """700 ragged sequences, some empty, in a cache long enough for the work to be shared."""
    batch, H, Hk, D = 700, 4, 2, 64
    capacity = 1536
    cache = K.kvq_cache(batch, Hk, capacity, D, 8)
    g = torch.Generator().manual_seed(91)
    lengths = torch.randint(0, 200, (batch,), generator=g)
    lengths[::7] = 0
    lengths[511], lengths[255], lengths[256] = 1500, 1100, 0
    k, v = rnd((batch, 200, Hk, D), 92).cuda(), rnd((batch, 200, Hk, D), 93).cuda()
    for at in range(0, capacity - 200, 200):
        K.kvq_write(cache, k, v, at)
    q = rnd((batch, 1, H, D), 94, 1.0, dtype).cuda()
    pos = [int(n) - 1 for n in lengths]
    got = K.kvq_attention(q, cache, torch.tensor(pos, dtype=torch.int32, device="cuda"))
    for b in list(range(0, 30)) + [254, 255, 256, 257, 510, 511, 512, 513, 698, 699]:
        one = K.KvqCache(*[t[b:b + 1].contiguous() for t in cache.tensors])
        alone = B.compare(K, one, q[b:b + 1], [pos[b]], n=max(pos[b] + 1, 1))
        assert torch.equal(got[b] == 0, torch.from_numpy(alone[0] == 0).cuda())
    # every sequence against the others' way of being shared out: fp32 to its bound's size, a few roundings
    far = (got.double() - torch.cat([K.kvq_attention(q[b:b + 1], K.KvqCache(*[t[b:b + 1].contiguous() for t in cache.tensors]), pos[b] if pos[b] >= 0 else
                                                      torch.tensor([-1], dtype=torch.int32, device="cuda")) for b in range(batch)]).double()).abs().max()
    assert far <= (2.0 ** -18 if dtype == F32 else 2.0 ** -6) * float(v.abs().max())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,Hk,D", [(17, 1, 64), (32, 1, 128), (40, 2, 64), (160, 1, 64)])
def test_one_token_of_many_heads(K, bits, dtype, H, Hk, D):  # noqa: F811
    """More than 16 query heads a key/value head: single tokens go to the prompt kernel."""
    n = 700
    cache = wrote(K, rnd((2, n, Hk, D), 101, 0.5), rnd((2, n, Hk, D), 102), bits)
    q = rnd((2, 1, H, D), 103, 1.0, dtype).cuda()
    B.compare(K, cache, q, n - 1)
    B.compare(K, cache, q, [0, 130], window=60, sinks=2, n=n)
