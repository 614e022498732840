"""attend_tree at the ends of what its arguments may be."""
import numpy as np
import pytest
import torch

from test_gpu_attend_tree import bits, check, drafted
from test_gpu_kv_attend import filled
from test_gpu_kv_cache import normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("past", [0, 65, 200])
@pytest.mark.parametrize("window", [63, 64, 65])
def test_windows_about_as_long_as_the_drafts(cuda, dtype, past, window):
    """64 drafts, of which one sees all and stands 64 after one that sees none."""
    cache, table, slots = filled(2, 64, [past], 60)
    r = np.random.RandomState(past)
    masks = [int(r.randint(0, 2 ** 31)) | int(r.randint(0, 2 ** 31)) << 33 for _ in range(64)]
    masks[5] = masks[40] = 0
    masks[20] = masks[63] = 2 ** 64 - 1
    masks[62] = 2 ** 64 - 2
    seen = bits(masks)
    q, k, v = (normal((64, h, 64), dtype, s) for s, h in ((61, 4), (62, 2), (63, 2)))
    batch = drafted([past], [64], table, slots)
    out, lse = cache.attend_tree(batch, q, k, v, seen, lse=True, window=window)
    check(cache, table, slots, [past], [64], q, k, v, seen, out, dtype, lse, window=window)
    # what the window hides may be anything
    v[5], k[40] = float("nan"), float("inf")
    got = cache.attend_tree(batch, q, k, v, seen, window=window)
    hidden = window <= 64
    assert torch.isfinite(got[[20, 63]]).all() == hidden
    if hidden:
        assert torch.equal(got[[20, 63]], out[[20, 63]])
