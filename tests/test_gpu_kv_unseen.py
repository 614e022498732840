"""A block that cannot be read, in a step where some rows see it and others, in
the same wave of the kernel, do not."""
import pytest
import torch

from test_gpu_kv_attend import check, filled
from test_gpu_kv_cache import normal, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("what", ["k", "v", "page"])
@pytest.mark.parametrize("past,tokens,window", [(41, 110, 0), (41, 110, 23), (126, 4, 2)])
def test_only_rows_that_see_a_block_are_nan(cuda, dim, dtype, what, past, tokens, window):
    kv_heads, group = 2, 2
    cache, table, slots = filled(kv_heads, dim, [past + tokens], 40)
    q = normal((tokens, kv_heads * group, dim), dtype, 41)
    want = cache.attend(step([past], [tokens], table, slots), q, window=window)
    check(cache, table, slots, [past], [tokens], q, want, dtype, window=window)
    if what == "page":
        table[0, 1] = -1
    else:
        cache.scales[int(table[0, 1]), :, 0 if what == "k" else 1] = float("nan")
    out, lse = cache.attend(step([past], [tokens], table, slots), q, window=window, lse=True)
    position = torch.arange(past, past + tokens, device="cuda")
    sees = position >= 64
    if window:
        sees &= position - window < 127
    # the same sums, up to the roundings that the block's scale may have moved: a last place of the output's type or
    # some 32 of fp32
    near = {"f32": 2.0 ** -18, "bf16": 2.0 ** -8}[dtype]
    assert torch.isnan(out[sees]).all() and (out[~sees] - want[~sees]).abs().max() <= near * want.abs().max()
    assert torch.isfinite(lse[~sees]).all() and (cache.faults() > 0) == (what == "page" and bool(sees.any()))
