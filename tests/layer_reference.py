"""The decoder-layer operators in 64 bits on the CPU, written from their
definitions in include/q4rdna.h: a cache that stores numbers by the two
rounding rules, attention over it, and the norms."""
import numpy as np

BLOCK = 64
CODE16 = 32512


def rotate(x, position, cos, sin, interleaved):
    """x [..., dim] (float64) by the row `position` of cos and sin."""
    half = cos.shape[1]
    out = x.copy()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = float(cos[position, i]), float(sin[position, i])
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def rms(x, weight, eps):
    x = np.asarray(x, dtype=np.float64)
    return x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + eps) * np.asarray(weight, dtype=np.float64)


def codes(which, dim):
    """(token, number) of each of a block's 64 * dim codes, K (0) or V (1)."""
    token, number = np.empty(BLOCK * dim, dtype=np.int64), np.empty(BLOCK * dim, dtype=np.int64)
    for t in range(BLOCK):
        for n in range(dim):
            if which == 0:
                at = (((t // 16 * (dim // 64) + n // 64) * 4 + n // 16 % 4) * 16 + t % 16) * 16 + n % 16
            else:
                at = ((n // 16 * 4 + t // 4 % 4) * 16 + n % 16) * 16 + t // 16 * 4 + t % 4
            token[at], number[at] = t, n
    return token, number


def tokens_of(cache, table_row, slot, length, head, which):
    """[length, dim] of one sequence and head from a cache's buffers (numpy)."""
    dim = cache["pages"].shape[-1] // BLOCK
    token, number = codes(which, dim)
    out = np.zeros((length, dim))
    for b in range((length + BLOCK - 1) // BLOCK):
        x = np.zeros((BLOCK, dim))
        if (b + 1) * BLOCK <= length:
            page = table_row[b]
            x[token, number] = cache["pages"][page, head, which].astype(np.float64) * float(cache["scales"][page, head, which])
        else:
            o = cache["open"][slot, b % 2, head].astype(np.float64)
            x[token, number] = 256 * o[2 * which] + o[2 * which + 1]
            x = x * cache["open_scales"][slot, b % 2, head, which].astype(np.float64)[:, None]
        n = min(BLOCK, length - b * BLOCK)
        out[b * BLOCK:b * BLOCK + n] = x[:n]
    return out


def attend(q, keys, values, positions, scale, window):
    """q [rows, dim] at `positions` over keys and values [length, dim]:
    (out, lse, largest |score|)."""
    out, lse, most = np.zeros(q.shape), np.zeros(q.shape[0]), 0.0
    for r, p in enumerate(positions):
        lo = max(0, p - window + 1) if window else 0
        s = scale * (keys[lo:p + 1] @ q[r])
        most = max(most, float(np.abs(s).max()))
        e = np.exp(s - s.max())
        out[r] = e @ values[lo:p + 1] / e.sum()
        lse[r] = s.max() + np.log(e.sum())
    return out, lse, most
