"""attend_tree's dealing of blocks to workgroups, against the definition."""
import numpy as np
import pytest
import torch

from test_gpu_attend_tree import chains, check, drafted
from test_gpu_kv_attend import filled
from test_gpu_kv_cache import ints, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [64, 65, 256, 257])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_sequences_than_a_scan_or_than_are_dealt(cuda, n, dtype):
    """Tables of more than 13 blocks, so that parts are worth it: sequences are
    looked at 64 at a time, and up to 256 of them are dealt by their lengths."""
    from q4rdna import api
    past = [(i * 37) % 200 for i in range(n)]
    past[3], past[n // 2], past[n - 1] = 1500, 0, 1100
    counts = [i % 3 for i in range(n)]
    counts[3], counts[n - 1] = 20, 9
    cache, table, slots = filled(1, 64, past, 70)
    assert table.shape[1] > 13
    total = sum(counts)
    q, k, v = (normal((total, h, 64), dtype, s) for s, h in ((71, 2), (72, 1), (73, 1)))
    batch = drafted(past, counts, table, slots)
    _, seen = api.tree(batch, ints(chains(counts, 9)))
    out, lse = cache.attend_tree(batch, q, k, v, seen, lse=True)
    check(cache, table, slots, past, counts, q, k, v, seen, out, dtype, lse)
    assert torch.equal(cache.attend_tree(batch, q, k, v, seen), out) and cache.faults() == 0


@pytest.mark.parametrize("dtype,past,count,window", [("bf16", 2048, 33, 900), ("f32", 3000, 64, 1025), ("f16", 1700, 5, 1500)])
def test_parts_of_a_window(cuda, dtype, past, count, window):
    """A window of so many blocks that they are split, its first ones masked."""
    from q4rdna import api
    cache, table, slots = filled(2, 128, [past], 74)
    q, k, v = (normal((count, h, 128), dtype, s, 1.5) for s, h in ((75, 4), (76, 2), (77, 2)))
    batch = drafted([past], [count], table, slots)
    _, seen = api.tree(batch, ints(chains([count], 5)))
    out, lse = cache.attend_tree(batch, q, k, v, seen, lse=True, window=window)
    check(cache, table, slots, [past], [count], q, k, v, seen, out, dtype, lse, window=window)
