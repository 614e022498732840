"""The append's roundings, number by number."""
from fractions import Fraction

import numpy as np
import pytest
import torch

import layer_reference as R
from test_gpu_kv_cache import DTYPES, f64, ints, make_cache, normal, snapshot, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("length", [5, 64, 130])
def test_numbers_up_to_the_type_s_largest(cuda, dtype, length):
    """Keys and values of 2^126 and more, whose reciprocal is subnormal, are kept
    like others."""
    cache, row = make_cache(2, 64, 4, 1), [2, 0, 3]
    k, v = normal((length, 2, 64), dtype, 1), normal((length, 2, 64), dtype, 2)
    k[1] *= 2.0 ** 126 / k[1].abs().max()
    v[2, 0] *= 3e38 / v[2, 0].abs().max()
    k[3, 1, 7] = torch.finfo(DTYPES[dtype]).max
    cache.append(step([0], [length], ints([row])), k, v)
    got = cache.read(step([0], [length], ints([row])), length)
    snap = snapshot(cache)
    for x, y, which in ((got[0], k, 0), (got[1], v, 1)):
        for head in range(2):
            for t in range(length):
                want = f64(y)[t, head]
                top = np.abs(want).max()
                step8 = float(snap["scales"][row[t // 64], head, which]) if (t // 64 + 1) * 64 <= length else 0.0
                # half a 16-bit step, half an 8-bit step, fp32 arithmetic before them
                bound = 0.5 * top / R.CODE16 + 0.5 * step8 + 2.0 ** -20 * top
                assert np.abs(f64(x)[t, head] - want).max() <= bound, (which, head, t)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_codes_are_the_nearest_to_the_scaled_numbers(cuda, dtype, dim):
    """code16 = rint(x * f), f = 32512 / (the token's largest) rounded to fp32, in
    every place of an open block; the product of two fp32 numbers is exact in 64 bits."""
    length, kv_heads = 63, 8
    cache = make_cache(kv_heads, dim, 1, 1)
    k, v = normal((length, kv_heads, dim), dtype, 3, 2.0), normal((length, kv_heads, dim), dtype, 4)
    cache.append(step([0], [length], ints([[0]])), k, v)
    o = snapshot(cache)["open"].astype(np.int64)
    for which, x in ((0, k), (1, v)):
        x = x.float().cpu().numpy()
        f = np.float32(R.CODE16) / np.abs(x).max(axis=-1, keepdims=True)
        want = np.rint(x.astype(np.float64) * f.astype(np.float64))
        token, number = R.codes(which, dim)
        got = np.zeros((64, kv_heads, dim))
        got[token, :, number] = (256 * o[0, 0, :, 2 * which] + o[0, 0, :, 2 * which + 1]).T
        assert np.array_equal(got[:length], want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_full_blocks_round_the_product_of_code_and_ratio(cuda, dtype):
    """code8 = rint(fl(code16 * r)), r = fl(token scale / block scale), with token
    scale = fl(largest / 32512) and block scale 256 times the largest of them:
    each in fp32, bit by bit.  Numbers of few bits make many exact products lie
    midway; rounded first, most of those go to the even code as they should."""
    kv_heads, dim = 8, 128
    cache = make_cache(kv_heads, dim, 1, 1)
    k, v = normal((64, kv_heads, dim), dtype, 5, 2.0), normal((64, kv_heads, dim), dtype, 6)
    cache.append(step([0], [64], ints([[0]])), k, v)
    snap = snapshot(cache)
    wrong = {"once": 0, "fused": 0}
    for which, x in ((0, k), (1, v)):
        x = x.float().cpu().numpy()
        largest = np.abs(x).max(axis=-1, keepdims=True)
        code = np.rint(x.astype(np.float64) * (np.float32(R.CODE16) / largest).astype(np.float64))
        scale = largest / np.float32(R.CODE16)
        whole = np.float32(256) * scale.max(axis=0, keepdims=True)
        ratio = scale / whole
        want = np.rint(code.astype(np.float32) * ratio)
        token, number = R.codes(which, dim)
        got = np.zeros((64, kv_heads, dim))
        got[token, :, number] = snap["pages"][0, :, which].T
        assert np.array_equal(snap["scales"][0, :, which], whole[0, :, 0]) and np.array_equal(got, want)
        b = largest.max(axis=0, keepdims=True)
        exact = np.array([[[nearest(c, l, t) for c in row] for row, l, t in zip(rows, ls[:, 0], b[0, :, 0])] for rows, ls in zip(code, largest)])
        wrong["once"] += int((want != exact).sum())
        wrong["fused"] += int((np.rint(code * ratio.astype(np.float64)) != exact).sum())
    assert wrong["once"] <= wrong["fused"]


def nearest(code, largest, top):
    """rint(code * largest / (256 * top)) of exact numbers, ties to the even."""
    return round(Fraction(int(code)) * Fraction(float(largest)) / (256 * Fraction(float(top))))
