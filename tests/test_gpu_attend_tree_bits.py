"""attend_tree's precision with 16-bit queries, drafts and outputs: scores and
weights as in fp32, nothing but the output itself in 16 bits."""
import numpy as np
import pytest
import torch

import branch_reference as B
import layer_reference as R
from test_gpu_attend_tree import chains, drafted, unsigned
from test_gpu_kv_attend import OUT_ROUND, filled
from test_gpu_kv_cache import f64, ints, make_cache, normal, snapshot, step

pytestmark = pytest.mark.gpu


def check_as_fp32(cache, table, slots, past, counts, q, k, v, seen, out, lse, dtype, window=0):
    """fp16 and bf16 numbers of q and k, and codes, are exact in the products, so
    what is left are fp32 roundings: of a score, a chain of under 16 of 2^-24 of
    the largest products' sum, and exp2's own; weights that two fp16 parts hold to
    2^-22, the log of V's scale to as much; and the output's half step."""
    snap, rows = snapshot(cache), table.cpu().numpy()
    kv_heads, dim = cache.kv_heads, cache.head_dim
    group, scale = q.shape[1] // kv_heads, dim ** -0.5
    q64, k64, v64, got, masks = f64(q), f64(k), f64(v), f64(out), unsigned(seen)
    at = 0
    for i, (p, c) in enumerate(zip(past, counts)):
        sees = np.repeat(B.visible(p, c, masks[at:at + c], window), group, axis=0)
        for head in range(kv_heads if c else 0):
            keys = np.concatenate((R.tokens_of(snap, rows[i], slots[i], p, head, 0), k64[at:at + c, head]))
            values = np.concatenate((R.tokens_of(snap, rows[i], slots[i], p, head, 1), v64[at:at + c, head]))
            heads = slice(head * group, (head + 1) * group)
            x = q64[at:at + c, heads].reshape(-1, dim)
            want, want_lse = B.attend(x, keys, values, sees, scale)
            reach = scale * np.where(sees, np.abs(x) @ np.abs(keys).T, 0).max(-1, keepdims=True)
            noise = 2.0 ** -24 * (16 * reach + 16)
            top = np.where(sees, np.abs(values).max(-1)[None], 0).max(-1, keepdims=True)
            err = np.abs(got[at:at + c, heads].reshape(-1, dim) - want)
            assert (err <= OUT_ROUND[dtype] * np.abs(want) + (2.0 ** -21 + 2 * noise) * top).all(), (i, head, err.max())
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
    out, lse = cache.attend_tree(batch, q, k, v, seen, lse=True)
    check_as_fp32(cache, table, [0], [past], [count], q, k, v, seen, out, lse, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kv_heads,group,dim", [(1, 1, 64), (2, 4, 128), (2, 7, 64), (1, 33, 128)])
@pytest.mark.parametrize("window", [0, 70])
def test_weights_keep_more_than_16_bits(cuda, dtype, kv_heads, group, dim, window):
    """Short and split sequences, drafts alone, full and open blocks: each row to
    the output's rounding."""
    from q4rdna import api
    past, counts = [0, 5, 60, 64, 190, 127, 2900, 65], [1, 3, 40, 0, 2, 64, 6, 20]
    cache, table, slots = filled(kv_heads, dim, past, 55)
    n = sum(counts)
    q, k, v = (normal((n, h, dim), dtype, s, 1.5) for s, h in ((56, kv_heads * group), (57, kv_heads), (58, kv_heads)))
    batch = drafted(past, counts, table, slots)
    _, seen = api.tree(batch, ints(chains(counts)))
    out, lse = cache.attend_tree(batch, q, k, v, seen, lse=True, window=window)
    check_as_fp32(cache, table, slots, past, counts, q, k, v, seen, out, lse, dtype, window)
    assert torch.equal(cache.attend_tree(batch, q, k, v, seen, window=window), out)
