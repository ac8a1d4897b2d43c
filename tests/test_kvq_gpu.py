"""The key/value cache of 4 or 8 bits and attention over it, against numpy in 64 bits (tests/kvq_ref.py)."""
import numpy as np
import pytest
import torch

from tests import kvq_ref as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def K():
    from emberlm_b200 import ops
    return ops


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    from emberlm_b200 import lib
    torch.cuda.synchronize()
    w = (lib.C.c_int * 4)()
    assert lib.raw().ctdk_device_status(None, w) == 0, lib.last_error()


def rnd(shape, seed, spread=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * spread).to(dtype)


def held(cache):
    """(k codes, k scales, v codes, v scales) on the host."""
    return [t.cpu() for t in cache.tensors]


def host_values(cache, n):
    """Keys and values [B, Hk, n, D] that the cache stands for, from its bytes."""
    out = []
    for codes, scales in (cache.tensors[:2], cache.tensors[2:]):
        u = codes[:, :, :n].cpu().numpy()
        if cache.bits == 4:
            u = np.stack((u & 15, u >> 4), -1).reshape(*u.shape[:-1], -1)
        out.append(R.values(u, scales[:, :, :n].float().cpu().numpy(), cache.bits))
    return out


def filled(K, B, Hk, n, D, bits, seed, capacity=None, spread=1.0):
    """A cache whose first n positions hold random rows; what lies behind them is NaN."""
    cache = K.kvq_cache(B, Hk, capacity or n, D, bits)
    for t in (cache.tensors[0], cache.tensors[2]):
        t.fill_(0xFF)
    for t in (cache.tensors[1], cache.tensors[3]):
        t.fill_(float("nan"))
    k, v = rnd((B, n, Hk, D), seed, 0.7 * spread).cuda(), rnd((B, n, Hk, D), seed + 1).cuda()
    k[..., 3::32] *= 4
    if n:
        K.kvq_write(cache, k, v, 0)
    return cache


def check(K, cache, q, pos, count=None, window=0, sinks=0, scale=None, n=None):
    """Runs attention and compares every row; pos and count: ints, or lists of one a sequence."""
    B, T = q.shape[:2]
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda") if isinstance(x, list) else x  # noqa: E731
    got = K.kvq_attention(q, cache, dev(pos), count=dev(count), window=window, sinks=sinks, scale=scale)
    assert got.dtype == q.dtype and got.shape == q.shape
    got = got.double().cpu().numpy()
    ps = pos if isinstance(pos, list) else [pos] * B
    cs = count if isinstance(count, list) else [T] * B
    n = n or min(cache.capacity, max([p + c for p, c in zip(ps, cs)] + [1]))
    k, v = host_values(cache, n)
    qq = q.double().cpu().numpy()
    for b in range(B):
        m = max(1, min(n, ps[b] + max(cs[b], 0)))
        want, tol = R.attention(qq[b], k[b][:, :m], v[b][:, :m], ps[b], cs[b], window, sinks, scale, split_q=q.dtype == F32,
                                out_bits=24 if q.dtype == F32 else 8)
        assert np.array_equal(np.isnan(got[b]), np.isnan(want)), b
        fine = ~np.isnan(want)
        over = (np.abs(got[b] - want) - tol)[fine]
        assert over.size == 0 or over.max() <= 0, (b, over.max(), np.abs(got[b] - want)[fine].max(), tol[fine].max())
        assert not got[b][cs[b]:].any()
    return got


# ---- writing and reading ------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,Hk,pos", [(1, 1, 1, 0), (2, 1, 3, 70), (3, 17, 5, 40), (1, 130, 8, 1)])
def test_write_holds_the_definition_and_read_gives_it_back(K, bits, D, dtype, B, T, Hk, pos):
    cache = K.kvq_cache(B, Hk, pos + T, D, bits)
    before = held(cache)
    k, v = rnd((B, T, Hk, D), 1, 3.0, dtype), rnd((B, T, Hk, D), 2, 1e-3, dtype)
    K.kvq_write(cache, k.cuda(), v.cuda(), pos)
    after = held(cache)
    back = K.kvq_read(cache, pos, T)
    for x, codes, scales, b0, s0, got in ((k, after[0], after[1], before[0], before[1], back[0]), (v, after[2], after[3], before[2], before[3], back[1])):
        u, s = R.hold(x.float().permute(0, 2, 1, 3).numpy(), bits)
        assert np.array_equal(codes[:, :, pos:pos + T].numpy(), R.pack(u, bits))
        assert np.array_equal(scales[:, :, pos:pos + T].float().numpy(), s)
        assert np.array_equal(got.cpu().numpy(), R.values(u, s, bits).astype(np.float32))
        for a, b in ((codes, b0), (scales, s0)):      # nothing else is touched
            assert torch.equal(a[:, :, :pos], b[:, :, :pos]) and torch.equal(a[:, :, pos + T:], b[:, :, pos + T:])


@pytest.mark.parametrize("bits", [4, 8])
def test_write_decides_halves_small_and_not_finite_groups_exactly(K, bits):
    """Values on and next to the half between two codes, zeros, denormals, the largest held magnitude, infinities and NaN."""
    top = 7 if bits == 4 else 127
    rows = []
    for s in (1.0, 1.125, 1.875, 0.4375) if bits == 4 else (1.0, 2.0 ** -9):
        for c in (0, 1, 2, 5, 6):
            x = np.full(32, (c + 0.5) * s, np.float32)
            x[1::4] = np.nextafter(x[1::4], np.float32(0))
            x[2::4] = np.nextafter(x[2::4], np.float32(100))
            x[3::4] *= -1
            x[0] = top * s
            rows.append(x)
    for m in (0.0, 1e-45, 3e-44, 1e-40, 1.2e-38, 1e-36, 1e-30, 2.0 ** -103, 2.0 ** -98, 1e29, 2.0 ** 100, 1e38, np.inf, np.nan):
        x = np.linspace(-1, 1, 32).astype(np.float32)
        with np.errstate(all="ignore"):
            rows.append(np.where(x == -1, m, x * np.float32(0 if not np.isfinite(m) else m)).astype(np.float32))
    if len(rows) % 2:
        rows.append(rows[0])
    x = torch.from_numpy(np.stack(rows).reshape(1, 1, len(rows) // 2, 64))
    cache = K.kvq_cache(1, x.shape[2], 1, 64, bits)
    K.kvq_write(cache, x.cuda(), (-x).cuda(), 0)
    after = held(cache)
    for y, codes, scales, got in ((x, after[0], after[1], K.kvq_read(cache, 0, 1)[0]), (-x, after[2], after[3], K.kvq_read(cache, 0, 1)[1])):
        u, s = R.hold(y[0, 0].numpy(), bits)
        assert np.array_equal(codes[0, :, 0].numpy(), R.pack(u, bits))
        assert np.array_equal(scales[0, :, 0].float().numpy(), s, equal_nan=True)
        assert np.array_equal(got.cpu().numpy()[0, :, 0], R.values(u, s, bits).astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("bits", [4, 8])
def test_write_leaves_padding_and_positions_outside_alone(K, bits):
    B, T, Hk, D = 5, 6, 2, 64
    cache = filled(K, B, Hk, 64, D, bits, 3)
    before = held(cache)
    k, v = rnd((B, T, Hk, D), 5), rnd((B, T, Hk, D), 6)
    pos, count = [10, 62, -3, 64, 20], [6, 6, 6, 6, 2]
    K.kvq_write(cache, k.cuda(), v.cuda(), torch.tensor(pos, dtype=torch.int32, device="cuda"), torch.tensor(count, dtype=torch.int32, device="cuda"))
    want = [t.clone() for t in before]
    for x, i in ((k, 0), (v, 2)):
        u, s = R.hold(x.permute(0, 2, 1, 3).numpy(), bits)
        for b in range(B):
            for t in range(count[b]):
                if 0 <= pos[b] + t < 64:
                    want[i][b, :, pos[b] + t] = torch.from_numpy(R.pack(u, bits)[b, :, t])
                    want[i + 1][b, :, pos[b] + t] = torch.from_numpy(s[b, :, t]).bfloat16()
    for a, b in zip(held(cache), want):
        assert torch.equal(a, b)


def test_write_from_a_packed_projection_and_read_repeats_heads(K):
    B, T, H, Hk, D = 2, 9, 4, 2, 64
    qkv = rnd((B, T, H + 2 * Hk, D), 7).cuda()
    a, b = K.kvq_cache(B, Hk, T, D, 8), K.kvq_cache(B, Hk, T, D, 8)
    K.kvq_write(a, qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:], 0)
    K.kvq_write(b, qkv[:, :, H:H + Hk].contiguous(), qkv[:, :, H + Hk:].contiguous(), 0)
    assert all(torch.equal(x, y) for x, y in zip(a.tensors, b.tensors))
    one, three = K.kvq_read(a, 2, 5), K.kvq_read(a, 2, 5, group=3)
    for x, y in zip(one, three):
        assert torch.equal(x.repeat_interleave(3, 1), y)
    for x, y in zip(one, K.kvq_read(a, 2, 5, dtype=BF16)):
        assert torch.equal(x, y.float())


# ---- attention ----------------------------------------------------------------------------------
LAYOUTS = [(3, 1, 64), (9, 3, 64), (4, 4, 128), (16, 8, 128), (8, 1, 64), (12, 1, 128)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,Hk,D", LAYOUTS)
@pytest.mark.parametrize("n", [1, 15, 16, 17, 64, 65, 127, 500])
def test_single_tokens(K, bits, dtype, H, Hk, D, n):
    B = 2
    cache = filled(K, B, Hk, n, D, bits, n)
    check(K, cache, rnd((B, 1, H, D), 9, 1.0, dtype).cuda(), n - 1)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,Hk,D", [(9, 3, 64), (16, 8, 128), (12, 1, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 4), (1, 0), (77, 100)])
def test_long_caches_are_split_over_the_device(K, bits, dtype, H, Hk, D, window, sinks):
    """Sequences of very different lengths, among them an empty one, whose work CTAs share unevenly."""
    lengths = [2600, 1, 0, 1025, 64, 2111]
    cache = filled(K, len(lengths), Hk, 2600, D, bits, 21, capacity=4096)
    q = rnd((len(lengths), 1, H, D), 22, 1.0, dtype).cuda()
    check(K, cache, q, [n - 1 for n in lengths], window=window, sinks=sinks)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("H,Hk,D", [(9, 3, 64), (16, 8, 128)])
@pytest.mark.parametrize("lengths", [[1, 1], [31, 32], [33, 130], [0, 450], [0, 0]])
def test_short_sequences_in_a_large_cache(K, bits, H, Hk, D, lengths):
    """The host sees the capacity only: far more CTAs than there is work."""
    cache = filled(K, 2, Hk, 450, D, bits, 25, capacity=8192)
    for dtype in (F32, BF16):
        check(K, cache, rnd((2, 1, H, D), 26, 1.0, dtype).cuda(), [n - 1 for n in lengths], n=450)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,Hk,D,T", [(4, 4, 64, 5), (16, 8, 128, 3), (8, 2, 64, 5), (15, 5, 64, 16), (4, 2, 128, 40), (3, 1, 64, 129)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3), (1, 0)])
def test_several_tokens(K, bits, dtype, H, Hk, D, T, window, sinks):
    cache = filled(K, 2, Hk, 200, D, bits, 31)
    q = rnd((2, T, H, D), 32, 1.0, dtype).cuda()
    check(K, cache, q, 200 - T, window=window, sinks=sinks)
    check(K, cache, q, [0, 31], window=window, sinks=sinks, n=200)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("T", [1, 4, 37])
def test_padding_empty_rows_and_positions_outside(K, bits, T):
    B, H, Hk, D = 6, 4, 2, 64
    cache = filled(K, B, Hk, 192, D, bits, 41)
    q = rnd((B, T, H, D), 42).cuda()
    q[1, T // 2:] = float("nan")                      # padding may hold anything
    check(K, cache, q, [0, 5, -2, 190, 300, -100], [T, T // 2, T, T, T, 0], n=192)
    check(K, cache, q, [0, 5, -2, 190, 300, -100], [T, T // 2, T, T, T, 0], window=3, sinks=1, n=192)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("D,T", [(64, 1), (128, 4), (64, 70)])
def test_not_finite_values_reach_the_rows_that_see_them_and_no_other(K, bits, D, T):
    """A key and a value that are NaN or infinite, at positions that some rows see, that the window has left, and behind all."""
    n, H, Hk = 150, 4, 2
    for at in (n - 1, n - T, n - T // 2 - 1, 10, 2):
        for which in (0, 1):
            cache = filled(K, 1, Hk, n, D, bits, 51)
            x = [rnd((1, 1, Hk, D), 52).cuda(), rnd((1, 1, Hk, D), 53).cuda()]
            x[which][0, 0, 1, D - 5] = float("inf") if at % 2 else float("nan")
            K.kvq_write(cache, x[0], x[1], at)
            for window, sinks in ((0, 0), (40, 4)):
                got = check(K, cache, rnd((1, T, H, D), 54).cuda(), n - T, window=window, sinks=sinks)
                assert np.isfinite(got[0, :, :H // 2]).all()     # the other head's


def test_large_scores_move_the_reference_point(K):
    """Scores that grow along the sequence by far more than the slack, and rows in which one position has all the weight."""
    n, D = 700, 64
    for bits in (4, 8):
        cache = K.kvq_cache(1, 1, n, D, bits)
        k, v = rnd((1, n, 1, D), 61), rnd((1, n, 1, D), 62)
        k *= torch.linspace(0.1, 30, n).reshape(1, n, 1, 1)
        K.kvq_write(cache, k.cuda(), v.cuda(), 0)
        check(K, cache, rnd((1, 1, 8, D), 63, 3.0).cuda(), n - 1)
        check(K, cache, rnd((1, 30, 8, D), 63, 3.0).cuda(), n - 30)


def test_scale_and_strided_queries(K):
    B, T, H, Hk, D = 2, 3, 4, 2, 64
    cache = filled(K, B, Hk, 100, D, 4, 71)
    qkv = rnd((B, T, H + 2 * Hk, D), 72).cuda()
    a = check(K, cache, qkv[:, :, :H], 97, scale=0.3)
    b = K.kvq_attention(qkv[:, :, :H].contiguous(), cache, 97, scale=0.3).cpu().numpy()
    assert np.array_equal(a.astype(np.float32), b)


@pytest.mark.parametrize("bits", [4, 8])
def test_offsets_past_32_bits(K, bits):
    """A cache of more than 4 GB a tensor: its last sequence and last positions."""
    B, Hk, D = 72 if bits == 4 else 36, 8, 128
    capacity, n = 131072, 70
    cache = K.kvq_cache(B, Hk, capacity, D, bits)
    assert cache.tensors[0].numel() > 2 ** 32
    k, v, q = rnd((1, n, Hk, D), 81).cuda(), rnd((1, n, Hk, D), 82).cuda(), rnd((B, 1, 16, D), 83).cuda()
    pos = torch.full((B,), -1, dtype=torch.int32, device="cuda")
    pos[-1] = capacity - n
    count = torch.tensor([0] * (B - 1) + [n], dtype=torch.int32, device="cuda")
    K.kvq_write(cache, k.expand(B, n, Hk, D), v.expand(B, n, Hk, D), pos, count)
    u, s = R.hold(k[0].permute(1, 0, 2).cpu().numpy(), bits)
    assert np.array_equal(K.kvq_read(cache, capacity - n, n, dtype=BF16)[0][-1].float().cpu().numpy(), R.values(u, s, bits).astype(np.float32))
    pos[-1] = capacity - 1
    got = K.kvq_attention(q, cache, pos, window=n)
    assert not got[:-1].any()
    small = K.kvq_cache(1, Hk, n, D, bits)
    K.kvq_write(small, k, v, 0)
    kk, vv = host_values(small, n)
    want, tol = R.attention(q[-1].double().cpu().numpy(), kk[0], vv[0], n - 1, 1)
    assert (np.abs(got[-1].double().cpu().numpy() - want) <= tol).all()


# ---- as they are used ---------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [4, 8])
def test_a_prompt_then_single_tokens(K, bits):
    """A padded batch of prompts is written and attended, then each sequence goes on by itself, one token at a time."""
    B, H, Hk, D, T = 3, 6, 2, 64, 90
    cache = K.kvq_cache(B, Hk, T + 8, D, bits)
    count = [90, 33, 1]
    qkv = rnd((B, T, H + 2 * Hk, D), 91).cuda()
    at = torch.zeros(B, dtype=torch.int32, device="cuda")
    cnt = torch.tensor(count, dtype=torch.int32, device="cuda")
    K.kvq_write(cache, qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:], at, cnt)
    check(K, cache, qkv[:, :, :H], [0] * B, count, n=T)
    for step in range(4):
        new = rnd((B, 1, H + 2 * Hk, D), 92 + step).cuda()
        pos = [c + step for c in count]
        K.kvq_write(cache, new[:, :, H:H + Hk], new[:, :, H + Hk:], torch.tensor(pos, dtype=torch.int32, device="cuda"))
        check(K, cache, new[:, :, :H], pos, window=0 if step % 2 else 50, sinks=2)


def test_a_captured_step_follows_positions_on_the_device(K):
    B, H, Hk, D, n = 4, 8, 2, 64, 1500
    cache = filled(K, B, Hk, n, D, 4, 101, capacity=2048)
    new, pos = rnd((B, 1, H + 2 * Hk, D), 102).cuda(), torch.tensor([700, 3, 1499, 0], dtype=torch.int32, device="cuda")

    def step():
        K.kvq_write(cache, new[:, :, H:H + Hk], new[:, :, H + Hk:], pos)
        return K.kvq_attention(new[:, :, :H], cache, pos)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        pos.add_(1)
        new.copy_(rnd(new.shape, 110 + i))
        graph.replay()
        torch.cuda.synchronize()
        want = K.kvq_attention(new[:, :, :H], cache, pos)
        assert torch.equal(got, want)
        check(K, cache, new[:, :, :H], pos.tolist(), n=n + 8)


def test_two_streams_at_once(K):
    """Calls on two streams, each with its own workspace, give what they give alone, every time."""
    caches = [filled(K, 2, 3, 3000, 64, bits, 121) for bits in (4, 8)]
    q = rnd((2, 1, 9, 64), 122).cuda()
    want = [K.kvq_attention(q, c, 2999) for c in caches]
    streams = [torch.cuda.Stream() for _ in caches]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(K.kvq_attention(q, caches[i], 2999))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        assert all(torch.equal(w, g) for g in gs)


def test_nothing_to_do(K):
    cache = filled(K, 2, 2, 64, 64, 4, 131)
    before = held(cache)
    empty = torch.empty(2, 0, 2, 64, device="cuda")
    K.kvq_write(cache, empty, empty, 64)
    assert all(torch.equal(a, b) for a, b in zip(before, held(cache)))
    assert K.kvq_attention(empty, cache, 64).shape == (2, 0, 2, 64)
    assert K.kvq_read(cache, 64, 0)[0].shape == (2, 2, 0, 64)


def test_refusals(K):
    cache = K.kvq_cache(2, 2, 100, 64, 4)
    assert cache.capacity == 128
    x, i32 = torch.zeros(2, 3, 2, 64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    bad = [
        lambda: K.kvq_cache(1, 1, 64, 96, 4), lambda: K.kvq_cache(1, 1, 64, 64, 6),
        lambda: K.KvqCache(*[t[:, :, :100].contiguous() for t in cache.tensors]),
        lambda: K.KvqCache(cache.tensors[0], cache.tensors[1], cache.tensors[0], cache.tensors[1].float()),
        lambda: K.kvq_write(cache, x, x, 126), lambda: K.kvq_write(cache, x, x, -1),
        lambda: K.kvq_write(cache, x.half(), x.half(), 0), lambda: K.kvq_write(cache, x, x.bfloat16(), 0),
        lambda: K.kvq_write(cache, x.cpu(), x.cpu(), 0), lambda: K.kvq_write(cache, x[:1], x[:1], 0),
        lambda: K.kvq_write(cache, x.transpose(1, 2).contiguous().transpose(1, 2), x, 0),
        lambda: K.kvq_write(cache, x, x, i32.long()), lambda: K.kvq_write(cache, x, x, 0, count=3),
        lambda: K.kvq_read(cache, 120, 9), lambda: K.kvq_read(cache, 0, 4, group=0), lambda: K.kvq_read(cache, 0, 4, dtype=torch.half),
        lambda: K.kvq_attention(x[:, :, :1].expand(2, 3, 3, 64), cache, 0), lambda: K.kvq_attention(torch.zeros(2, 1, 3, 64, device="cuda"), cache, 0),
        lambda: K.kvq_attention(x, cache, 126), lambda: K.kvq_attention(x, cache, i32[:1]),
        lambda: K.kvq_attention(x, cache, 0, window=-1), lambda: K.kvq_attention(x, cache, 0, sinks=-1),
        lambda: K.kvq_attention(torch.zeros(2 * 3 * 2 * 64 + 1, device="cuda")[1:].view(2, 3, 2, 64), cache, 0),
    ]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()


# ---- what long sums cost, and prompts as they are replayed ----------------------------------------
@pytest.mark.parametrize("bits,D", [(4, 128), (8, 64)])
@pytest.mark.parametrize("T,H", [(1, 4), (2, 8), (3, 48)])
def test_fp32_sums_over_long_rows(K, bits, D, T, H):
    """Values of one sign, so that what the tensor cores cut off an accumulator (2^-23 of it at most, every sum) adds up. An
    accumulator takes 64 sums at most (four tiles of 128 positions, 16 a product, in two terms) before fp32 addition takes over;
    probabilities and scores in two terms leave 2^-20. Sums kept in one accumulator would be off by up to 2048 * 2^-23."""
    n, Hk = 16384, 1
    cache = K.kvq_cache(1, Hk, n, D, bits)
    v = 1 + 0.05 * rnd((1, n, Hk, D), 131)
    K.kvq_write(cache, rnd((1, n, Hk, D), 132, 0.05).cuda(), v.cuda(), 0)
    q = rnd((1, T, H, D), 133)
    got = K.kvq_attention(q.cuda(), cache, n - T).double().cpu().numpy()
    kk, vv = host_values(cache, n)
    want, _ = R.attention(q[0].double().numpy(), kk[0], vv[0], n - T, T)
    assert np.linalg.norm(got[0] - want) <= (64 * 2.0 ** -23 + 2.0 ** -20) * np.linalg.norm(want)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_prompts_replayed_and_on_two_streams(K, dtype):
    """A captured prompt follows positions and counts on the device; two graphs' prompts run at once with a workspace each."""
    B, T, H, Hk, D = 2, 70, 6, 2, 64
    caches = [filled(K, B, Hk, 1200, D, bits, 141, capacity=1280) for bits in (4, 8)]
    q = rnd((B, T, H, D), 142, dtype=dtype).cuda()
    pos = torch.tensor([0, 900], dtype=torch.int32, device="cuda")
    count = torch.tensor([70, 9], dtype=torch.int32, device="cuda")
    streams, graphs, outs = [torch.cuda.Stream() for _ in caches], [], []
    for c in caches:
        K.kvq_attention(q, c, pos, count=count)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(K.kvq_attention(q, c, pos, count=count))
        graphs.append(g)
    for i in range(3):
        pos.copy_(torch.tensor([60 * i, 900 + i], dtype=torch.int32))
        count.copy_(torch.tensor([70 - 30 * i, 9 + 20 * i], dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(5):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for c, out in zip(caches, outs):
            want = check(K, c, q, pos.tolist(), count.tolist())
            assert np.array_equal(out.double().cpu().numpy(), want)
