"""Small things at the edges of the decoder-layer calls."""
import pytest
import torch

from test_gpu_kv_attend import check, filled
from test_gpu_kv_cache import ints, normal, step

pytestmark = pytest.mark.gpu


def test_a_refused_sequence_counts_once(cuda):
    """In a step that both attention kernels take part in, and in each of them alone."""
    for past, counts in (([300, 0, 20], [1, 150, 1]), ([300, 60], [1, 1]), ([0, 10], [150, 90]), ([5], [150])):
        cache, table, slots = filled(1, 64, [p + c for p, c in zip(past, counts)], 70)
        q = normal((sum(counts), 4, 64), "bf16", 71)
        for bad in range(len(past)):
            for other, at in (([-5 if i == bad else p for i, p in enumerate(past)], slots),
                              (past, [99 if i == bad else s for i, s in enumerate(slots)])):
                before = cache.faults()
                cache.attend(step(other, counts, table, at), q)
                assert cache.faults() == before + 1
