"""The quantised cache without a GPU: refusals of the C entry points, and the definition's own properties."""
import ctypes as C

import numpy as np
import pytest

from emberlm_b200 import lib
from tests import kvq_ref as R


def desc(**k):
    a = dict(k_codes=4096, k_scales=4096, v_codes=4096, v_scales=4096, B=2, capacity=128, Hk=2, D=64, bits=4)
    a.update(k)
    return lib.KvqCacheDesc(**a)


@pytest.mark.parametrize("change", [dict(bits=3), dict(D=96), dict(capacity=100), dict(capacity=0), dict(Hk=0), dict(B=-1),
                                    dict(k_codes=None), dict(v_scales=4100), dict(capacity=2 ** 31)])
def test_entry_points_refuse_a_bad_cache(change):
    L, d = lib.raw(), desc(**change)
    p = C.addressof(d)
    assert L.ctdk_kvq_write(p, 4096, 4096, 0, 128, 128, 1, None, 0, None, None) == lib.CTDK_EINVAL
    assert L.ctdk_kvq_read(p, 0, 1, 1, 0, 4096, 4096, None) == lib.CTDK_EINVAL
    assert L.ctdk_kvq_attn(p, 4096, 0, 128, 128, 1, 4, None, 0, None, 0, 0, 0.125, 4096, 4096, 1 << 30, None) == lib.CTDK_EINVAL
    assert L.ctdk_kvq_attn_workspace_bytes(p, 1, 4) == lib.CTDK_EINVAL
    assert b"kvq" in L.ctdk_last_error()
    assert L.ctdk_kvq_write(None, 4096, 4096, 0, 128, 128, 1, None, 0, None, None) == lib.CTDK_EINVAL


def test_entry_points_refuse_bad_arguments():
    L, d = lib.raw(), desc()
    p = C.addressof(d)
    ok = (4096, 4096, 0, 128, 128)
    for args in ((4096, 4096, 2, 128, 128), (None, 4096, 0, 128, 128), (4100, 4096, 0, 128, 128), (4096, 4096, 0, 130, 128), (4096, 4096, 1, 132, 128)):
        assert L.ctdk_kvq_write(p, *args, 1, None, 0, None, None) == lib.CTDK_EINVAL
    for T, at in ((1, 128), (129, 0), (1, -1), (-1, 0)):
        assert L.ctdk_kvq_write(p, *ok, T, None, at, None, None) == lib.CTDK_EINVAL
        assert L.ctdk_kvq_attn(p, 4096, 0, 128, 128, T, 4, None, at, None, 0, 0, 0.125, 4096, 4096, 1 << 30, None) == lib.CTDK_EINVAL
    for start, n, group in ((0, 129, 1), (128, 1, 1), (-1, 1, 1), (0, -1, 1), (0, 1, 0)):
        assert L.ctdk_kvq_read(p, start, n, group, 0, 4096, 4096, None) == lib.CTDK_EINVAL
    for H, window, sinks, q, out in ((3, 0, 0, 4096, 4096), (0, 0, 0, 4096, 4096), (4, -1, 0, 4096, 4096), (4, 0, -1, 4096, 4096), (4, 0, 0, None, 4096),
                                     (4, 0, 0, 4096, 4104)):
        assert L.ctdk_kvq_attn(p, q, 0, 128, 128, 1, H, None, 0, None, window, sinks, 0.125, out, 4096, 1 << 30, None) == lib.CTDK_EINVAL
    # nothing to do is no error, whatever the pointers
    assert L.ctdk_kvq_write(p, None, None, 0, 0, 0, 0, None, 128, None, None) == lib.CTDK_OK
    assert L.ctdk_kvq_read(p, 128, 0, 1, 0, None, None, None) == lib.CTDK_OK
    assert L.ctdk_kvq_attn(p, None, 0, 0, 0, 0, 4, None, 128, None, 0, 0, 0.125, None, None, 0, None) == lib.CTDK_OK


@pytest.mark.parametrize("bits", [4, 8])
def test_what_is_held_is_exact_in_bfloat16_and_within_half_a_step(bits):
    x = (np.random.default_rng(1).standard_normal((500, 64)) * np.exp(np.random.default_rng(2).uniform(-20, 20, (500, 1)))).astype(np.float32)
    u, s = R.hold(x, bits)
    v = R.values(u, s, bits)
    assert np.array_equal(v, (v.astype(np.float32).view(np.uint32) & 0xffff0000).view(np.float32).astype(np.float64))
    assert (np.abs(v - x) <= np.repeat(s, 32, -1).reshape(x.shape) / 2).all()
