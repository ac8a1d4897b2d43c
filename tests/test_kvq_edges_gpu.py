"""The quantised cache at the edges of what its calls take, on the GPU; against numpy in 64 bits (tests/kvq_ref.py) where there are values."""
import pytest
import torch

from tests.test_kvq_gpu import K, _status_clean  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("T,H", [(1, 4), (16, 4), (40, 6)])
def test_an_empty_batch(K, T, H):  # noqa: F811
    cache = K.kvq_cache(0, 2, 100, 64, 4)
    rows = torch.empty(0, T, 2, 64, device="cuda")
    K.kvq_write(cache, rows, rows, 0)
    assert K.kvq_attention(torch.empty(0, T, H, 64, device="cuda"), cache, 0).shape == (0, T, H, 64)
    assert K.kvq_read(cache, 0, 8)[0].shape == (0, 2, 8, 64)
