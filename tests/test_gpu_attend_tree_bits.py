"""attend_tree's precision with 16-bit queries and drafts: scores as in fp32."""
import numpy as np
import pytest

import branch_reference as B
import layer_reference as R
from test_gpu_attend_tree import chains, drafted, unsigned
from test_gpu_kv_cache import f64, ints, make_cache, normal, snapshot, step

pytestmark = pytest.mark.gpu


def check_lse(cache, table, slots, past, counts, q, k, v, seen, lse, window=0):
    """fp16 and bf16 numbers of q and k, and codes, are exact in the products, so
    what is left are fp32 roundings: of a score, a chain of under 16 of 2^-24 of
    the largest products' sum, and exp2's own."""
    snap, rows = snapshot(cache), table.cpu().numpy()
    kv_heads, dim = cache.kv_heads, cache.head_dim
    group, scale = q.shape[1] // kv_heads, dim ** -0.5
    q64, k64, v64, masks = f64(q), f64(k), f64(v), unsigned(seen)
    at = 0
    for i, (p, c) in enumerate(zip(past, counts)):
        sees = np.repeat(B.visible(p, c, masks[at:at + c], window), group, axis=0)
        for head in range(kv_heads if c else 0):
            keys = np.concatenate((R.tokens_of(snap, rows[i], slots[i], p, head, 0), k64[at:at + c, head]))
            values = np.concatenate((R.tokens_of(snap, rows[i], slots[i], p, head, 1), v64[at:at + c, head]))
            heads = slice(head * group, (head + 1) * group)
            x = q64[at:at + c, heads].reshape(-1, dim)
            _, want_lse = B.attend(x, keys, values, sees, scale)
            reach = scale * np.where(sees, np.abs(x) @ np.abs(keys).T, 0).max(-1, keepdims=True)
            noise = 2.0 ** -24 * (16 * reach + 16)
            off = np.abs(f64(lse)[at:at + c, heads].reshape(-1) - want_lse)
            assert (off <= noise[:, 0] + 2.0 ** -22 * (1 + np.abs(want_lse))).all(), (i, head, off.max())
        at += c


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("signs", ["same", "halves"])
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_of_quiet_tokens_beside_a_loud_one(cuda, dtype, signs, dim):
    """A token that is loud in a number of which q has nothing sets its block's
    scale; the others' codes are small, while q's numbers share a sign, or are
    positive in one half and negative in the other."""
    from q4rdna import api
    past, count, heads = 256, 5, 2
    cache, table = make_cache(1, dim, 5, 1), ints([[3, 0, 4, 1]])
    k0, v0 = normal((past, 1, dim), "f32", 50, 0.4), normal((past, 1, dim), "f32", 51)
    k0[..., 0] = 0
    k0[::64, 0, 0] = 100.0
    cache.append(step([0], [past], table), k0, v0)
    q = normal((count, heads, dim), dtype, 52).abs() + 0.5
    q[..., 0] = 0
    if signs == "halves":
        q[..., dim // 2:] *= -1
    k, v = (normal((count, 1, dim), dtype, s) for s in (53, 54))
    batch = drafted([past], [count], table)
    _, seen = api.tree(batch, ints(chains([count])))
    _, lse = cache.attend_tree(batch, q, k, v, seen, lse=True)
    check_lse(cache, table, [0], [past], [count], q, k, v, seen, lse)
