"""kv_append and kv_read against their definitions in 64 bits."""
import itertools

import numpy as np
import pytest
import torch

import layer_reference as R

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROUND = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a last place, relative


def make_cache(kv_heads, dim, pages, slots, seed=0):
    """A cache whose buffers hold another use's leftovers, NaN scales among them."""
    from q4rdna import api
    g = torch.Generator().manual_seed(seed)
    size = 64 * dim
    return api.KVCache(torch.randint(-127, 128, (pages, kv_heads, 2, size), generator=g, dtype=torch.int8).cuda(),
                       torch.full((pages, kv_heads, 2), float("nan")).cuda(),
                       torch.randint(-127, 128, (slots, 2, kv_heads, 4, size), generator=g, dtype=torch.int8).cuda(),
                       torch.full((slots, 2, kv_heads, 2, 64), float("nan")).cuda())


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def step(past, counts, table, slots=None):
    from q4rdna import api
    if all(c == 1 for c in counts):
        return api.KVBatch(ints(past), table, slots=None if slots is None else ints(slots))
    return api.KVBatch(ints(past), table, cu_tokens=ints([0] + list(itertools.accumulate(counts))),
                       slots=None if slots is None else ints(slots), max_tokens=max(1, max(counts)))


def rotary_table(positions, rotary, seed=1):
    angle = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(rotary // 2) / max(1, rotary // 2))
    return (torch.tensor(np.cos(angle), dtype=torch.float32, device="cuda"),
            torch.tensor(np.sin(angle), dtype=torch.float32, device="cuda"))


def snapshot(c):
    return {"pages": c.pages.cpu().numpy(), "scales": c.scales.cpu().numpy(), "open": c.open.cpu().numpy(),
            "open_scales": c.open_scales.cpu().numpy()}


def normal(shape, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * spread).to(DTYPES[dtype]).cuda()


def f64(t):
    return t.detach().cpu().double().numpy()


def check_values(cache, table_row, slot, length, k, v, first=0):
    """The sequence's stored numbers against the given ones (float64, from token
    `first`): each is off by half a 16-bit step and, in a full block, half an
    8-bit step, the steps being the stored scales; 2^-20 more for the fp32
    arithmetic before the rounding (a few roundings of 2^-24)."""
    snap = snapshot(cache)
    for head in range(k.shape[1]):
        for which, want in ((0, k), (1, v)):
            got = R.tokens_of(snap, table_row, slot, length, head, which)
            for t in range(first, length):
                x = want[t - first, head]
                top = np.abs(x).max()
                step16 = top / R.CODE16
                b = t // 64
                step8 = float(snap["scales"][table_row[b], head, which]) if (b + 1) * 64 <= length else 0.0
                bound = 0.5 * step16 + 0.5 * step8 + 2.0 ** -20 * top
                assert np.abs(got[t] - x).max() <= bound, (head, which, t, np.abs(got[t] - x).max(), bound)
            for b in range(length // 64):  # the block's scale is that of its largest token
                lo, hi = max(first, b * 64), (b + 1) * 64
                if lo == b * 64:
                    top = np.abs(want[lo - first:hi - first, head]).max()
                    s = float(snap["scales"][table_row[b], head, which])
                    assert abs(s - 256 * top / R.CODE16) <= 2.0 ** -20 * s


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,kv_heads", [(64, 3), (128, 2)])
@pytest.mark.parametrize("length", [1, 15, 16, 63, 64, 65, 127, 128, 193, 320])
def test_append_stores_the_numbers(cuda, dtype, dim, kv_heads, length):
    cache = make_cache(kv_heads, dim, 9, 3)
    row = [7, 2, 5, 0, 8, 3]
    k, v = normal((length, kv_heads, dim), dtype, 1, 2.0), normal((length, kv_heads, dim), dtype, 2)
    cache.append(step([0], [length], ints([row]), [1]), k, v)
    check_values(cache, row, 1, length, f64(k), f64(v))
    assert cache.faults() == 0
    got = cache.read(step([0], [length], ints([row]), [1]), length)
    snap = snapshot(cache)
    for which in (0, 1):
        for head in range(kv_heads):
            want = R.tokens_of(snap, row, 1, length, head, which)
            # one fp32 product per number
            assert np.abs(f64(got[which])[:, head] - want).max() <= 2.0 ** -23 * np.abs(want).max()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("chunks", [[1] * 130, [64, 66], [63, 1, 1, 65], [5, 190, 5], [70, 130, 130], [17, 400, 3],
                                    [127, 2, 63, 128, 1], [100, 28, 64, 64]])
def test_bytes_do_not_depend_on_the_chunks(cuda, dim, chunks):
    kv_heads, total = 2, sum(chunks)
    row = list(range(8))
    k, v = normal((total, kv_heads, dim), "f32", 3), normal((total, kv_heads, dim), "f32", 4)
    cos, sin = rotary_table(total, dim)
    whole, parts = make_cache(kv_heads, dim, 8, 1), make_cache(kv_heads, dim, 8, 1)
    whole.append(step([0], [total], ints([row])), k, v, cos=cos, sin=sin)
    at = 0
    for c in chunks:
        parts.append(step([at], [c], ints([row])), k[at:at + c], v[at:at + c], cos=cos, sin=sin)
        at += c
    a, b = snapshot(whole), snapshot(parts)
    full = total // 64
    assert np.array_equal(a["pages"][:full], b["pages"][:full])
    assert np.array_equal(a["scales"][:full], b["scales"][:full])
    # the open block, and the last full one (kept for cutting back)
    for block in range(max(0, full - 1), (total + 63) // 64):
        n = min(64, total - block * 64)
        for which in (0, 1):
            token, _ = R.codes(which, dim)
            live = token < n
            planes = slice(2 * which, 2 * which + 2)
            assert np.array_equal(a["open"][0, block % 2, :, planes][:, :, live], b["open"][0, block % 2, :, planes][:, :, live])
            assert np.array_equal(a["open_scales"][0, block % 2, :, which, :n], b["open_scales"][0, block % 2, :, which, :n])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (64, 16), (128, 128), (128, 64), (128, 8), (128, 0)])
@pytest.mark.parametrize("norm", [False, True])
def test_rotation_and_norm(cuda, dtype, interleaved, dim, rotary, norm):
    kv_heads, group, past, counts = 2, 3, [3, 60], [2, 7]
    cache = make_cache(kv_heads, dim, 4, 2)
    table = ints([[0, 1], [2, 3]])
    tokens = sum(counts)
    q, k = normal((tokens, kv_heads * group, dim), dtype, 5), normal((tokens, kv_heads, dim), dtype, 6, 3.0)
    v = normal((tokens, kv_heads, dim), dtype, 7)
    cos, sin = rotary_table(80, rotary) if rotary else (None, None)
    wq, wk = (1 + 0.3 * normal((dim,), "f32", 8), 1 + 0.3 * normal((dim,), "f32", 9)) if norm else (None, None)
    q_out = cache.append(step(past, counts, table), k, v, q=q, cos=cos, sin=sin, interleaved=interleaved,
                         q_norm=wq, k_norm=wk, eps=1e-5)
    want_q, want_k = f64(q), f64(k)
    if norm:
        want_q, want_k = R.rms(want_q, f64(wq), 1e-5), R.rms(want_k, f64(wk), 1e-5)
    position = [3, 4] + list(range(60, 67))
    if rotary:
        c, s = f64(cos), f64(sin)
        want_q = np.stack([R.rotate(want_q[n], p, c, s, interleaved) for n, p in enumerate(position)])
        want_k = np.stack([R.rotate(want_k[n], p, c, s, interleaved) for n, p in enumerate(position)])
    # The norm's sum of squares and product chain: under 16 roundings; the rotation: three.
    near = 2.0 ** -20 * np.abs(want_q).max()
    assert (np.abs(f64(q_out) - want_q) <= ROUND[dtype] * np.abs(want_q) + near).all()
    check_values(cache, [0, 1], 0, 5, want_k[:2], f64(v)[:2], first=3)
    snap = snapshot(cache)
    for head in range(kv_heads):  # the second sequence's block closed over unknown tokens: its open part is checked
        got = R.tokens_of(snap, [2, 3], 1, 67, head, 0)[64:]
        top = np.abs(want_k[6:, head]).max(axis=-1, keepdims=True)
        assert (np.abs(got - want_k[6:, head]) <= (0.5 / R.CODE16 + 2.0 ** -20) * top).all()


@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_and_misaligned_rows(cuda, offset, dtype):
    """q, k and v as slices of one buffer that starts anywhere."""
    kv_heads, group, dim, tokens = 2, 2, 64, 5
    heads = kv_heads * group
    width = (heads + 2 * kv_heads) * dim + 1
    flat = normal((offset + tokens * width,), dtype, 11)
    qkv = flat[offset:].view(tokens, width)[:, :-1].unflatten(1, (heads + 2 * kv_heads, dim))
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    cos, sin = rotary_table(64, dim)
    a, b = make_cache(kv_heads, dim, 1, 1), make_cache(kv_heads, dim, 1, 1)
    batch = step([0], [tokens], ints([[0]]))
    got = a.append(batch, k, v, q=q, cos=cos, sin=sin)
    want = b.append(batch, k.contiguous(), v.contiguous(), q=q.contiguous(), cos=cos, sin=sin)
    assert torch.equal(got, want)
    x, y = a.read(batch, tokens), b.read(batch, tokens)
    assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])
    # in place over the strided q, and read into strided rows
    before = qkv[:, heads:].clone()
    assert a.append(batch, k, v, q=q, q_out=q, cos=cos, sin=sin) is q
    assert torch.equal(q, want) and torch.equal(qkv[:, heads:], before)
    a.read(batch, tokens, dtype=DTYPES[dtype], k=qkv[:, heads:heads + kv_heads], v=qkv[:, heads + kv_heads:])
    assert torch.equal(qkv[:, heads:heads + kv_heads], y[0].to(DTYPES[dtype])) and torch.equal(q, want)


def test_numbers_that_are_not_finite(cuda):
    """Such a token reads as NaN, in its head alone, and so does its block once
    full; zeros and tiny tokens read as zero; huge ones are kept."""
    kv_heads, dim = 2, 64
    cache = make_cache(kv_heads, dim, 4, 1)
    table = ints([[0, 1, 2, 3]])
    k, v = normal((130, kv_heads, dim), "f32", 12), normal((130, kv_heads, dim), "f32", 13)
    k[3, 0, 5] = float("nan")
    v[70, 1, 0] = float("inf")
    k[129, 1] = 0.0
    v[128, 0] *= 1e-33
    k[128, 0] *= 1e37
    cache.append(step([0], [50], table), k[:50], v[:50])
    got = cache.read(step([0], [50], table), 50)
    assert torch.isnan(got[0][3, 0]).all() and torch.isfinite(got[0][3, 1]).all()
    assert torch.isfinite(got[0][:3]).all() and torch.isfinite(got[0][4:]).all() and torch.isfinite(got[1]).all()
    cache.append(step([50], [80], table), k[50:], v[50:])
    got = cache.read(step([0], [130], table), 130)
    assert torch.isnan(got[0][:64, 0]).all() and torch.isfinite(got[0][:64, 1]).all()
    assert torch.isnan(got[1][64:128, 1]).all() and torch.isfinite(got[1][64:128, 0]).all()
    assert torch.isfinite(got[0][64:]).all()
    assert (got[0][129, 1] == 0).all() and (got[1][128, 0] == 0).all()
    big = k[128, 0]
    assert (got[0][128, 0] - big).abs().max() <= big.abs().max() * (0.5 / R.CODE16 + 2.0 ** -20)


def test_cut_back_and_appended_again(cuda):
    """A sequence cut back into its last full block goes on as if the tokens
    had never been there."""
    kv_heads, dim, row = 1, 128, [0, 1, 2, 3]
    k, v = normal((200, kv_heads, dim), "f32", 14), normal((200, kv_heads, dim), "f32", 15)
    k2, v2 = normal((60, kv_heads, dim), "f32", 16), normal((60, kv_heads, dim), "f32", 17)
    for total, back in ((130, 64), (130, 100), (128, 70), (70, 3), (129, 127)):
        a, b = make_cache(kv_heads, dim, 4, 1), make_cache(kv_heads, dim, 4, 1)
        a.append(step([0], [total], ints([row])), k[:total], v[:total])
        a.append(step([back], [60], ints([row])), k2, v2)
        b.append(step([0], [back], ints([row])), k[:back], v[:back])
        b.append(step([back], [60], ints([row])), k2, v2)
        whole = step([0], [back + 60], ints([row]))
        for x, y in zip(a.read(whole, back + 60), b.read(whole, back + 60)):
            assert torch.equal(x, y), (total, back)


def test_refused_entries_are_counted_and_harmless(cuda):
    """Out-of-range entries touch nothing, are counted, and leave the batch's
    other sequences alone."""
    kv_heads, dim = 2, 64
    k, v = normal((5, kv_heads, dim), "f32", 18), normal((5, kv_heads, dim), "f32", 19)
    from q4rdna import api
    good_past = [10, 63, 5, 0, 7]
    cases = [("past", 0, -1), ("past", 2, 128), ("past", 4, 2 ** 31 - 1), ("slots", 1, 9), ("slots", 3, -4), ("table", 1, 77),
             ("table", 1, -1)]
    for what, at, value in cases:
        cache = make_cache(kv_heads, dim, 10, 5)
        past, slots = list(good_past), [4, 3, 2, 1, 0]
        table = [[2 * i, 2 * i + 1] for i in range(5)]
        if what == "past":
            past[at] = value
        elif what == "slots":
            slots[at] = value
        else:
            table[at][0] = value
        before = snapshot(cache)
        cache.append(api.KVBatch(ints(past), ints(table), slots=ints(slots)), k, v)
        assert cache.faults() == (kv_heads if what == "table" else 1), (what, at, value)
        after = snapshot(cache)
        for i in range(5):
            held = np.array_equal(after["open"][4 - i], before["open"][4 - i])
            assert held == (i == at and what != "table"), (what, at, value, i)
        closes = what == "table" or at == 1
        assert np.array_equal(after["pages"], before["pages"]) == closes


def test_tokens_outside_the_step_are_refused(cuda):
    from q4rdna import api
    cache = make_cache(1, 64, 4, 2)
    k, v = normal((6, 1, 64), "f32", 20), normal((6, 1, 64), "f32", 21)
    before = snapshot(cache)
    table = ints([[0, 1], [2, 3]])
    for cu, most in (([0, 3, 7], 4), ([0, 3, 2], 4), ([-2, 3, 2], 6), ([0, 6, 6], 3)):
        cache.append(api.KVBatch(ints([0, 0]), table, cu_tokens=ints(cu), max_tokens=most), k, v)
        assert cache.faults() > 0
    after = snapshot(cache)
    # only the first sequence of the first two steps was in range
    assert np.array_equal(before["open"][1], after["open"][1]) and np.array_equal(before["pages"], after["pages"])


def test_sequences_without_tokens_and_empty_steps(cuda):
    from q4rdna import api
    cache = make_cache(1, 64, 4, 3)
    k, v = normal((4, 1, 64), "f32", 22), normal((4, 1, 64), "f32", 23)
    table = ints([[0], [1], [2]])
    cache.append(step([0, 5, 9], [0, 4, 0], table), k, v)
    got = cache.read(step([5, 5, 9], [0, 4, 0], table), 4)
    assert (got[0] - k).abs().max() <= k.abs().max() * (0.5 / R.CODE16 + 2.0 ** -20) and cache.faults() == 0
    cache.append(api.KVBatch(ints([0, 5, 9]), table, cu_tokens=ints([0, 0, 0, 0])), k[:0], v[:0])
    empty = torch.empty((0, 1), dtype=torch.int32, device="cuda")
    cache.append(api.KVBatch(ints([]), empty), k[:0], v[:0])


def test_pages_past_four_gigabytes(cuda):
    """A page whose bytes lie past 2^32."""
    kv_heads, dim, pages = 16, 128, 17000
    from q4rdna import api
    cache = api.KVCache(torch.empty((pages, kv_heads, 2, 64 * dim), dtype=torch.int8, device="cuda"),
                        torch.zeros((pages, kv_heads, 2), device="cuda"),
                        torch.zeros((1, 2, kv_heads, 4, 64 * dim), dtype=torch.int8, device="cuda"),
                        torch.zeros((1, 2, kv_heads, 2, 64), device="cuda"))
    assert (pages - 1) * kv_heads * 2 * 64 * dim > 2 ** 32
    k, v = normal((64, kv_heads, dim), "bf16", 24), normal((64, kv_heads, dim), "bf16", 25)
    batch = step([0], [64], ints([[pages - 1]]))
    cache.append(batch, k, v)
    got = cache.read(batch, 64)
    assert (got[0] - k.float()).abs().max() <= cache.scales[pages - 1].max() * 0.51
    q = normal((64, kv_heads, dim), "bf16", 26)
    out = cache.attend(batch, q)
    for head in (0, 15):
        want, _, _ = R.attend(f64(q)[:, head], f64(got[0])[:, head], f64(got[1])[:, head], range(64), dim ** -0.5, 0)
        assert np.abs(f64(out)[:, head] - want).max() <= 2.0 ** -8 * np.abs(want).max() + 2.0 ** -10 * np.abs(f64(got[1])).max()


@pytest.mark.parametrize("sequences", [100, 4300])
def test_ragged_steps_of_many_sequences(cuda, sequences):
    """Places are found among more sequences than one trip of the search sees:
    appended raggedly and read back."""
    kv_heads, dim = 1, 64
    r = np.random.RandomState(sequences)
    counts = [int(c) for c in r.randint(0, 4, sequences)]
    counts[7] = 150
    past = [0] * sequences
    rows = [[i, sequences + i, 2 * sequences + i] for i in range(sequences)]
    cache = make_cache(kv_heads, dim, 3 * sequences, sequences)
    table = ints(rows)
    total = sum(counts)
    q, k, v = normal((total, 3, dim), "f32", 50), normal((total, kv_heads, dim), "f32", 51), normal((total, kv_heads, dim), "f32", 52)
    cos, sin = rotary_table(160, dim)
    batch = step(past, counts, table)
    q_out = cache.append(batch, k, v, q=q, cos=cos, sin=sin)
    got = cache.read(batch, total)
    assert cache.faults() == 0
    position = np.concatenate([np.arange(c) for c in counts])
    c, s = f64(cos), f64(sin)
    want_q = np.stack([R.rotate(f64(q[n]), p, c, s, False) for n, p in enumerate(position)])
    want_k = np.stack([R.rotate(f64(k[n]), p, c, s, False) for n, p in enumerate(position)])
    assert np.abs(f64(q_out) - want_q).max() <= 2.0 ** -20 * np.abs(want_q).max()
    # 8-bit steps in the one sequence's full blocks, 16-bit steps elsewhere
    first = sum(counts[:7])
    full = np.zeros(total, dtype=bool)
    full[first:first + 128] = True
    for x, want in ((got[0], want_k), (got[1], f64(v))):
        err, top = np.abs(f64(x) - want).max(axis=(1, 2)), np.abs(want).max()
        assert (err[full] <= top * (0.5 / 127 + 0.5 / R.CODE16 + 2.0 ** -20)).all()
        assert (err[~full] <= top * (0.5 / R.CODE16 + 2.0 ** -20)).all()
