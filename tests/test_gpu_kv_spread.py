"""kv_attend where the values of one block are far larger than another's: every
row is held to what its own weights give, not to the sequence's largest value."""
import math

import numpy as np
import pytest
import torch

import layer_reference as R
from test_gpu_kv_attend import OUT_ROUND, WEIGHT_ROUND
from test_gpu_kv_cache import f64, ints, make_cache, normal, snapshot, step

pytestmark = pytest.mark.gpu


def largest(cache, snap, row, slot, length, head):
    """The largest number that each token's V codes can hold: 127 of the block's
    steps, or 32512 of the token's own in the open block."""
    out = np.empty(length)
    for t in range(length):
        if (t // 64 + 1) * 64 <= length:
            out[t] = 127 * float(snap["scales"][row[t // 64], head, 1])
        else:
            out[t] = R.CODE16 * float(snap["open_scales"][slot, t // 64 % 2, head, 1, t % 64])
    return out


def check_rows(cache, row, slot, past, q, out, dtype, window=0):
    """Every number of every row of one sequence, by elements:

    * half a last place of the output's type;
    * relative to sum_t p_t |v_t|: the weights' own rounding; the scores' fp32
      roundings (a chain of under 16 of 2^-24 of the largest sum |q k|, an
      absolute error of the exponent, twice for the sum of weights); a rounding
      or two for each matrix product that adds into a number (8 a block, with
      two parts of each weight);
    * the weights' last place: 2^-31 at most of the largest weight that one of
      the row's blocks carries, for each of its tokens.
    """
    snap = snapshot(cache)
    kv_heads, dim = cache.kv_heads, cache.head_dim
    group, count = q.shape[1] // kv_heads, q.shape[0]
    length = past + count
    token, position = np.arange(length), np.repeat(past + np.arange(count), group)
    seen = token[None] <= position[:, None]
    if window:
        seen &= token[None] > position[:, None] - window
    block, whole = token // 64, (token // 64 + 1) * 64 <= length
    blocks = np.array([len(np.unique(block[row])) for row in seen])
    for head in range(kv_heads):
        heads = slice(head * group, (head + 1) * group)
        x, got = f64(q)[:, heads].reshape(-1, dim), f64(out)[:, heads].reshape(-1, dim)
        keys, values = (R.tokens_of(snap, row, slot, length, head, which) for which in (0, 1))
        top = largest(cache, snap, row, slot, length, head)
        s = np.where(seen, dim ** -0.5 * (x @ keys.T), -np.inf)
        w = np.exp(s - s.max(axis=1, keepdims=True))
        w /= w.sum(axis=1, keepdims=True)
        want, mass = w @ values, w @ np.abs(values)
        carried = np.max([w[:, block == b].max(axis=1) * top[block == b].max() if whole[block == b].all()
                          else (w * top)[:, block == b].max(axis=1) for b in range(block[-1] + 1)], axis=0)
        reach = np.where(seen, dim ** -0.5 * (np.abs(x) @ np.abs(keys).T), 0).max(axis=1)
        relative = WEIGHT_ROUND[dtype] + 2 * 2.0 ** -24 * (16 * reach + 16) + 2.0 ** -24 * (16 * blocks + 32)
        last = seen.sum(axis=1) * 2.0 ** -31 * carried
        bound = OUT_ROUND[dtype] * np.abs(want) + relative[:, None] * mass + last[:, None]
        off = np.abs(got - want) / bound
        n = int(off.max(axis=1).argmax())
        assert (off <= 1).all(), (head, n // group, n % group, off[n].max(), got[n, :4], want[n, :4])


def spread_cache(dim, length, loud, spread, nats, seed):
    """A sequence whose tokens in `loud` have values `spread` times the others'
    and scores `nats` below theirs for the queries of `toward`."""
    kv_heads, blocks = 2, (length + 63) // 64
    row = [blocks - i for i in range(blocks)]
    cache = make_cache(kv_heads, dim, blocks + 1, 2, seed)
    g = torch.Generator().manual_seed(seed)
    side = torch.randn((kv_heads, dim), generator=g).cuda()
    side /= side.norm(dim=-1, keepdim=True)
    k, v = normal((length, kv_heads, dim), "f32", seed + 1, 0.2), normal((length, kv_heads, dim), "f32", seed + 2)
    sign = torch.ones(length, device="cuda")
    sign[loud] = -1.0
    k += sign[:, None, None] * side * (nats / 2 / 10 * dim ** 0.5)
    v[loud] *= spread
    cache.append(step([0], [length], ints([row]), [1]), k, v)
    return cache, row, side


def toward(side, tokens, group, dtype, seed):
    kv_heads, dim = side.shape
    q = normal((tokens, kv_heads, group, dim), "f32", seed, 0.2) + 10 * side[:, None]
    return q.reshape(tokens, kv_heads * group, dim).to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype,spread", [("f32", 1e3), ("f32", 1e6), ("f32", 1e24), ("bf16", 1e6), ("bf16", 1e24), ("f16", 1e3)])
@pytest.mark.parametrize("loud", [slice(0, 64), slice(128, 192), slice(192, 256)])
@pytest.mark.parametrize("hidden", [False, True])
def test_a_quiet_block_beside_a_loud_one(cuda, dim, dtype, spread, loud, hidden):
    """A prompt, so that some rows see the loud block and others, in the same
    wave, do not.  Its part of a row is as large as the quiet blocks', or
    (`hidden`) far below their rounding."""
    length, past = 256, 19
    cache, row, side = spread_cache(dim, length, loud, spread, math.log(spread) + (35 if hidden else 0), 1)
    q = toward(side, length - past, 3, dtype, 7)
    out = cache.attend(step([past], [length - past], ints([row]), [1]), q)
    check_rows(cache, row, 1, past, q, out, dtype)


@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("spread", [1e6, 1e24])
def test_parts_of_a_long_row_with_references_of_their_own(cuda, tokens, spread):
    """A long sequence is cut into parts, which are joined; the loud blocks lie
    in some of them."""
    length = 64 * 100
    loud = torch.zeros(length, dtype=torch.bool)
    for b in (3, 40, 41, 97):
        loud[64 * b:64 * b + 64] = True
    for nats in (math.log(spread), math.log(spread) + 35):
        cache, row, side = spread_cache(64, length, loud.cuda(), spread, nats, 2)
        past = length - tokens
        q = toward(side, tokens, 2, "f32", 8)
        out = cache.attend(step([past], [tokens], ints([row]), [1]), q)
        check_rows(cache, row, 1, past, q, out, "f32")
