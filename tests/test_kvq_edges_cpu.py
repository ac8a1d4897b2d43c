"""The quantised cache at the edges of what its calls take, as far as that needs no GPU."""
import ctypes as C
import subprocess
import sys

import pytest

from emberlm_b200 import lib


def desc(**k):
    a = dict(k_codes=4096, k_scales=4096, v_codes=4096, v_scales=4096, B=2, capacity=128, Hk=2, D=64, bits=4)
    a.update(k)
    return lib.KvqCacheDesc(**a)


@pytest.mark.parametrize("T,H", [(1, 4), (8, 4), (9, 4), (64, 4), (1, 64), (0, 4)])
def test_an_empty_batch_needs_nothing(T, H):
    """In a process of its own: a division by the number of rows would end it."""
    code = (f"import ctypes as C; from emberlm_b200 import lib; L = lib.raw()\n"
            f"d = lib.KvqCacheDesc(B=0, capacity=128, Hk=2, D=64, bits=4); p = C.addressof(d)\n"
            f"assert L.ctdk_kvq_attn_workspace_bytes(p, {T}, {H}) == 0\n"
            f"assert L.ctdk_kvq_attn(p, None, 0, 0, 0, {T}, {H}, None, 0, None, 0, 0, 0.125, None, None, 0, None) == 0\n"
            f"assert L.ctdk_kvq_write(p, None, None, 0, 0, 0, {T}, None, 0, None, None) == 0\n"
            f"assert L.ctdk_kvq_read(p, 0, 8, 1, 0, None, None, None) == 0\n")
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, (res.returncode, res.stderr[-2000:])


def test_no_rows_need_no_workspace():
    d = desc()
    assert lib.raw().ctdk_kvq_attn_workspace_bytes(C.addressof(d), 0, 4) == 0
    assert lib.raw().ctdk_kvq_attn_workspace_bytes(C.addressof(d), 0, 64) == 0


def test_positions_and_lengths_at_the_end_of_64_bits_are_refused():
    L, d = lib.raw(), desc()
    p = C.addressof(d)
    for at in (2 ** 63 - 1, 2 ** 63 - 64, 127):
        assert L.ctdk_kvq_write(p, 4096, 4096, 0, 128, 128, 64, None, at, None, None) == lib.CTDK_EINVAL
        assert L.ctdk_kvq_attn(p, 4096, 0, 128, 128, 64, 4, None, at, None, 0, 0, 0.125, 4096, 4096, 1 << 30, None) == lib.CTDK_EINVAL
    for T in (2 ** 63 - 1, 2 ** 62, 2 ** 40, -1):
        assert L.ctdk_kvq_attn_workspace_bytes(p, T, 4) == lib.CTDK_EINVAL
        assert L.ctdk_kvq_attn(p, 4096, 0, 128, 128, T, 4, 4096, 0, None, 0, 0, 0.125, 4096, 4096, 1 << 30, None) == lib.CTDK_EINVAL


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_a_scale_that_is_not_finite_is_refused(scale):
    L, d = lib.raw(), desc()
    for T in (1, 64):                                  # few and many rows
        assert L.ctdk_kvq_attn(C.addressof(d), 4096, 0, 128, 128, T, 4, None, 0, None, 0, 0, scale, 4096, 4096, 1 << 30, None) == lib.CTDK_EINVAL


@pytest.mark.parametrize("value", [2 ** 64, 2 ** 63, -2 ** 63 - 1, 2 ** 64 + 5, 3.5, float("nan"), float("inf")])
def test_numbers_that_a_call_would_change_are_refused(value):
    """ctypes keeps the low 64 bits of a number: position 2^64 would be position 0, a window of 2^64 + 5 one of 5."""
    from emberlm_b200 import ops

    cache = type("Cache", (), {"B": 2, "device": None, "capacity": 64})()
    with pytest.raises(RuntimeError, match="whole number"):
        ops._kvq_places(value, None, cache, "kvq_write")
    assert ops._kvq_places(7.0, None, cache, "kvq_write") == [None, 7, None]
    assert ops._kvq_places(2 ** 62, None, cache, "kvq_write") == [None, 2 ** 62, None]


def test_windows_and_groups_that_a_call_would_change_are_refused():
    import torch

    from emberlm_b200 import ops

    cache = type("Cache", (), {"B": 2, "device": torch.device("cpu"), "capacity": 64, "Hk": 2, "D": 64})()
    q = torch.zeros(2, 1, 4, 64)
    for kw in ({"window": 2 ** 64 + 5}, {"sinks": 2 ** 64 + 5}, {"window": 2.5}):
        with pytest.raises(RuntimeError, match="whole number"):
            ops.kvq_attention(q, cache, 0, **kw)
    for args in ((0, 1, 2 ** 32 + 1), (0.5, 1, 1), (0, 1, 2 ** 31)):
        with pytest.raises(RuntimeError):
            ops.kvq_read(cache, *args)
