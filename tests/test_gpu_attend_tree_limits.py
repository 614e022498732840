"""attend_tree at the ends of what its arguments may be."""
import numpy as np
import pytest
import torch

import branch_reference as B
import layer_reference as R
from test_gpu_attend_tree import bits, check, drafted, unsigned
from test_gpu_kv_attend import OUT_ROUND, filled
from test_gpu_kv_cache import f64, ints, make_cache, normal, snapshot, step

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


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("q_size,k_size", [(0, 118), (0, 125), (-100, 124), (60, 60), (120, -20), (100, -100), (-60, -60)])
@pytest.mark.parametrize("past", [0, 40, 64, 168])
@pytest.mark.parametrize("scale", [0.125, 0.0])
def test_loud_keys_whose_scores_are_numbers(cuda, dtype, q_size, k_size, past, scale):
    """Queries of 2^q_size and keys of 2^k_size, drafted, in the open block and in
    full ones: where the scores are fp32 numbers the rows are too.  q and k have one
    small whole number each, so products are exact, tokens tie exactly or are a 16th
    of 2^(q_size + k_size) apart, and a score is off by 2^-22 of itself."""
    from q4rdna import api
    dim, count, r = 64, 12, np.random.RandomState(7)
    cache, table = make_cache(1, dim, 4, 1), ints([[1, 3, 0]])

    def first(numbers, size, heads=1):
        x = torch.zeros((len(numbers), heads, dim), dtype=torch.float64)
        x[..., 0] = torch.tensor(numbers, dtype=torch.float64).view(len(numbers), -1) * 2.0 ** size
        return x.to({"f32": torch.float32, "bf16": torch.bfloat16}[dtype]).cuda()

    if past:
        cache.append(step([0], [past], table), first(r.choice([-3, -1, 1], past), k_size), normal((past, 1, dim), dtype, 64))
    q = first(r.randint(1, 4, (count, 2)), q_size, 2)
    k = first(r.choice([-4, -2, 2, 4], count), k_size)
    v = normal((count, 1, dim), dtype, 65, 300.0)
    batch = drafted([past], [count], table)
    _, seen = api.tree(batch, ints([-1] + [int(r.randint(max(-1, j - 4), j)) for j in range(1, count)]))
    out, lse = cache.attend_tree(batch, q, k, v, seen, lse=True, scale=scale)
    snap = snapshot(cache)
    keys = np.concatenate((R.tokens_of(snap, [1, 3, 0], 0, past, 0, 0), f64(k)[:, 0]))
    values = np.concatenate((R.tokens_of(snap, [1, 3, 0], 0, past, 0, 1), f64(v)[:, 0]))
    sees = np.repeat(B.visible(past, count, unsigned(seen), 0), 2, axis=0)
    x = f64(q).reshape(-1, dim)
    want, want_lse = B.attend(x, keys, values, sees, scale)
    reach = scale * np.abs(x @ keys.T).max()
    noise = 2.0 ** -22 * reach if reach < 64 else 0.0  # (the best ones alone count otherwise)
    top = np.where(sees, np.abs(values).max(-1)[None], 0).max(-1, keepdims=True)
    bound = OUT_ROUND[dtype] * np.abs(want) + (2.0 ** -20 + 2 * noise) * top
    assert (np.abs(f64(out).reshape(-1, dim) - want) <= bound).all()
    assert (np.abs(f64(lse).reshape(-1) - want_lse) <= 2.0 ** -21 * (1 + np.abs(want_lse)) + noise).all()
