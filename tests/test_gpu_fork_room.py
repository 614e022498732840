"""What KVBatch.fork gives pages for with a room of nothing: open blocks."""
import pytest
import torch

from test_gpu_fork import state
from test_gpu_kv_cache import ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 300])  # in one launch, and with the plan in one of its own
@pytest.mark.parametrize("free", [0, 2])
def test_room_of_nothing(cuda, n, free):
    """A block that holds tokens gets a page, and adds a fault where none is left;
    a sequence that ends with a full block, or is empty, gets none and adds none."""
    past_of = [130, 128, 0, 63] * n
    full = sum(p // 64 for p in past_of)
    caches, batch, past, table, slots = state(past_of, 4, full + free, len(past_of), layers=1, kv_heads=1)
    before = table.clone()
    batch.fork(torch.arange(len(past_of), dtype=torch.int32, device="cuda"), caches, room=0)
    held = set(before[before >= 0].tolist())
    left = [p for p in range(full + free) if p not in held]
    want = before.tolist()
    for i, p in enumerate(past_of):
        if p % 64 and left:
            want[i][p // 64] = left.pop(0)
    assert torch.equal(table, ints(want)) and past.tolist() == past_of
    assert caches[0].faults() == 2 * n - free
