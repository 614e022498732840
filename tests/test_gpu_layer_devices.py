"""The decoder-layer calls run on their tensors' device."""
import pytest
import torch

from q4rdna._lib import Q4RdnaError
from test_gpu_kv_attend import filled
from test_gpu_kv_cache import normal, step

pytestmark = pytest.mark.gpu


def test_a_device_that_is_not_there(cuda):
    """Refused, and the current device stays."""
    cache, table, slots = filled(1, 64, [70], 90)
    batch = step([69], [1], table, slots)
    q, k = normal((1, 2, 64), "f32", 91), normal((1, 1, 64), "f32", 92)
    want = cache.attend(batch, q)
    for bad in (torch.cuda.device_count(), 1000, -3):
        cache.raw.device = bad
        for call in (lambda: cache.attend(batch, q), lambda: cache.append(batch, k, k), lambda: cache.read(batch, 1)):
            with pytest.raises(Q4RdnaError, match="device"):
                call()
    cache.raw.device = 0
    assert torch.cuda.current_device() == 0 and torch.equal(cache.attend(batch, q), want)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device_than_the_current_one(cuda):
    from q4rdna import api
    cache = api.KVCache.empty(2, 1, 2, 64, device=1)
    past, table, cu = (torch.tensor(x, dtype=torch.int32, device="cuda:1") for x in ([0], [[0, 1]], [0, 70]))
    k, q = torch.randn((70, 2, 64), device="cuda:1"), torch.randn((70, 4, 64), device="cuda:1")
    batch = api.KVBatch(past, table, cu, max_tokens=70)
    results = []
    for current in (1, 0):
        with torch.cuda.device(current):
            cache.append(batch, k, k)
            results.append((cache.attend(batch, q), *cache.read(batch, 70), *api.add_norm(k[:, 0], k[:, 1], torch.ones(64, device="cuda:1"))))
            assert torch.cuda.current_device() == current
    torch.cuda.synchronize(1)
    assert all(torch.equal(a, b) for a, b in zip(*results))
