"""Outputs that the calls of the decoder-layer operators allocate."""
import pytest
import torch

from test_gpu_kv_attend import filled
from test_gpu_kv_cache import normal, rotary_table, step

pytestmark = pytest.mark.gpu


def test_rows_of_a_sliding_window(cuda):
    """Inputs whose rows overlap in memory, each one number further on."""
    from q4rdna import api
    cache, table, slots = filled(1, 64, [70], 50)
    base = normal((5000,), "f32", 51)
    for shape, stride in (((5, 4, 64), (1, 64, 1)), ((5, 4, 64), (64, 1, 1)), ((5, 4, 64), (1, 1, 1)), ((5, 4, 64), (0, 0, 1))):
        q = base.as_strided(shape, stride)
        batch = step([65], [5], table, slots)
        for x, y in zip(cache.attend(batch, q, lse=True), cache.attend(batch, q.contiguous(), lse=True)):
            assert torch.equal(x, y)
        k = normal((5, 1, 64), "f32", 52)
        cos, sin = rotary_table(80, 64)
        assert torch.equal(cache.append(batch, k, k, q=q, cos=cos, sin=sin), cache.append(batch, k, k, q=q.contiguous(), cos=cos, sin=sin))
    x, y = base.as_strided((50, 64), (1, 1)), normal((50, 64), "f32", 53)
    for a, b in zip(api.add_norm(x, y, base[:64].contiguous()), api.add_norm(x.contiguous(), y, base[:64].contiguous())):
        assert torch.equal(a, b)
    # read: v in the manner of a given k
    k = torch.zeros((70 * 64 + 70,), device="cuda").as_strided((70, 1, 64), (65, 1, 1))
    batch = step([0], [70], table, slots)
    assert all(torch.equal(a, b) for a, b in zip(cache.read(batch, 70, k=k), cache.read(batch, 70)))
