"""How many bits of queries and probabilities attention over the quantised cache keeps, from sums of so few products that nothing else
shows: against 64 bits by the bound of kvq_bounds.py."""
import pytest
import torch

from tests import kvq_bounds as B
from tests.test_kvq_gpu import K, _status_clean  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def cache_of(K, k, v, bits):  # noqa: F811
    cache = K.kvq_cache(k.shape[0], k.shape[2], k.shape[1], k.shape[3], bits)
    K.kvq_write(cache, k.cuda(), v.cuda(), 0)
    return cache


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 2, 3, 5, 40])      # 2 query heads a key/value head: up to four rows, eight, sixteen, a prompt
def test_probabilities(K, bits, dtype, D, T):  # noqa: F811
    """Two positions count, one of them with values of zero: an output is one probability over a sum of two."""
    batch, Hk, H, n = 6, 8, 16, T + 1
    k, v = torch.zeros(batch, n, Hk, D), torch.zeros(batch, n, Hk, D)
    k[:, 1:, :, 0] = -1.0
    k[:, 2:, :, 0] = -1024.0
    v[:, 1] = 1.0
    v[:, 2:] = -1.0
    cache = cache_of(K, k, v, bits)
    q = torch.zeros(batch, T, H, D)
    q[..., 0] = torch.rand(q.shape[:-1], generator=torch.Generator().manual_seed(3)) * 3.5 + 0.25
    B.compare(K, cache, q.to(dtype).cuda(), 1, scale=1.0)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 2, 3, 5, 40])      # 2 query heads a key/value head: up to four rows, eight, sixteen, a prompt
def test_queries(K, bits, dtype, D, T):  # noqa: F811
    """Large scores of two positions, each from one column of the query alone: their difference shows the columns' last bits."""
    batch, Hk, H, n = 6, 8, 16, T + 1
    k, v = torch.zeros(batch, n, Hk, D), torch.zeros(batch, n, Hk, D)
    k[:, 0, :, 5] = 7.0
    k[:, 1, :, 40] = 7.0
    k[:, 2:, :, 5] = -7.0
    v[:, 1] = 1.0
    cache = cache_of(K, k, v, bits)
    q = torch.zeros(batch, T, H, D)
    g = torch.Generator().manual_seed(4)
    q[..., 5] = 9 + torch.rand(q.shape[:-1], generator=g) * 0.2
    q[..., 40] = 9 + torch.rand(q.shape[:-1], generator=g) * 0.2
    B.compare(K, cache, q.to(dtype).cuda(), 1, scale=1.0)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 5, 40])
@pytest.mark.parametrize("power", [10, 14, 17, 18, 19, 20, 22, 23, 24, 25, 26, 27, 30])
def test_small_values_beside_large_ones(K, bits, dtype, D, T, power):  # noqa: F811
    """Columns in which only the small values are not zero keep their bits, and so do scores from columns in which only the small keys are."""
    batch, Hk, H, n = 3, 4, 8, T + 1
    k, v = torch.zeros(batch, n, Hk, D), torch.zeros(batch, n, Hk, D)
    k[:, 1:, :, 0] = -1.0
    k[:, 2:, :, 0] = -1024.0
    v[:, 0, :, 7::32] = 1.0
    v[:, 1] = 2.0 ** -power                            # (one or two steps of its group)
    v[:, 1, :, 9::32] = (4.0 if bits == 4 else 64.0) * 2.0 ** -power
    v[:, 1, :, 7::32] = 0.0
    q = torch.zeros(batch, T, H, D)
    q[..., 0] = torch.rand(q.shape[:-1], generator=torch.Generator().manual_seed(5)) * 3.5 + 0.25
    B.compare(K, cache_of(K, k, v, bits), q.to(dtype).cuda(), 1, scale=1.0)
    k[:, 0, :, 40] = 2.0 ** (power + 6)                # large keys in a column that no query has
    k[:, 1:, :, 9] = 4.0 if bits == 4 else 64.0        # (and the others of one or two steps)
    B.compare(K, cache_of(K, k, v, bits), q.to(dtype).cuda(), 1, scale=1.0)
