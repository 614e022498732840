"""kv_attend against attention in 64 bits over the numbers that the cache holds."""
import numpy as np
import pytest
import torch

import layer_reference as R
from test_gpu_kv_cache import DTYPES, f64, ints, make_cache, normal, snapshot, step

pytestmark = pytest.mark.gpu

# Half a last place of the output's type, and what the weights' rounding adds
# relative to the largest |v|: none in fp32 (30-bit fixed point, or two 11-bit
# halves), 2^-11 where a prompt's weights are fp16.
OUT_ROUND = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
WEIGHT_ROUND = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -11}


def filled(kv_heads, dim, lengths, seed=0, spread=1.0, kv_dtype="f32"):
    """A cache with sequences of these lengths in scattered pages and slots:
    (cache, table, slots)."""
    blocks = [(n + 63) // 64 for n in lengths]
    width = max(1, max(blocks))
    order = np.random.RandomState(seed).permutation(sum(blocks) + 2)
    rows, at = [], 0
    for b in blocks:
        rows.append(list(order[at:at + b]) + [0] * (width - b))
        at += b
    slots = [len(lengths) - i for i in range(len(lengths))]  # slot 0 stays unused
    cache = make_cache(kv_heads, dim, len(order), len(lengths) + 1, seed)
    total = sum(lengths)
    k = normal((total, kv_heads, dim), kv_dtype, 100 + seed, spread)
    v = normal((total, kv_heads, dim), kv_dtype, 200 + seed)
    table = ints(rows)
    if total:
        cache.append(step([0] * len(lengths), lengths, table, slots), k, v)
    assert cache.faults() == 0
    return cache, table, slots


def check(cache, table, slots, past, counts, q, out, dtype, lse=None, scale=None, window=0):
    """Every row: |error| <= half a last place, the weights' rounding times
    max |v|, and the scores' fp32 roundings: a score is a chain of under 16
    roundings of 2^-24 relative to the largest score, which enter the weights
    as absolute errors, and so does exp2's own error (2^-22)."""
    snap, rows = snapshot(cache), table.cpu().numpy()
    kv_heads, dim = cache.kv_heads, cache.head_dim
    group = q.shape[1] // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    q64, got = f64(q), f64(out)
    at = 0
    for i, (p, c) in enumerate(zip(past, counts)):
        for head in range(kv_heads if c else 0):
            keys = R.tokens_of(snap, rows[i], slots[i], p + c, head, 0)
            values = R.tokens_of(snap, rows[i], slots[i], p + c, head, 1)
            heads = slice(head * group, (head + 1) * group)
            x = q64[at:at + c, heads].reshape(-1, dim)
            positions = np.repeat(p + np.arange(c), group)
            want, want_lse, most = R.attend(x, keys, values, positions, scale, window)
            # products of |q| |k| that cancel leave larger roundings than the score itself
            reach = scale * (np.abs(x) @ np.abs(np.nan_to_num(keys)).T).max()
            noise = 2.0 ** -24 * (16 * reach + 16)
            top = np.nanmax(np.abs(values))
            bound = OUT_ROUND[dtype] * np.abs(want) + (WEIGHT_ROUND[dtype] + 2 * noise) * top
            err = np.abs(got[at:at + c, heads].reshape(-1, dim) - want)
            assert (err <= bound).all(), (i, head, err.max(), bound.max(), most)
            if lse is not None:
                e = np.abs(f64(lse)[at:at + c, heads].reshape(-1) - want_lse)
                assert (e <= noise + 2.0 ** -22 * (1 + np.abs(want_lse))).all(), (i, head, e.max())
        at += c


SHAPES = [(1, 1, 64), (2, 4, 128), (3, 5, 64), (1, 8, 128), (2, 12, 64), (1, 33, 128)]


@pytest.mark.parametrize("kv_heads,group,dim", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_single_tokens(cuda, kv_heads, group, dim, dtype):
    lengths = [1, 2, 63, 64, 65, 128, 129, 400]
    cache, table, slots = filled(kv_heads, dim, lengths)
    past = [n - 1 for n in lengths]
    q = normal((len(lengths), kv_heads * group, dim), dtype, 1, 2.0)
    out, lse = cache.attend(step(past, [1] * len(lengths), table, slots), q, lse=True)
    check(cache, table, slots, past, [1] * len(lengths), q, out, dtype, lse)
    assert cache.faults() == 0


@pytest.mark.parametrize("kv_heads,group,dim", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window", [0, 1, 40, 64, 130])
def test_several_tokens_ragged(cuda, kv_heads, group, dim, dtype, window):
    past, counts = [0, 5, 60, 64, 190, 127, 300], [1, 3, 9, 0, 2, 1, 6]
    lengths = [p + c for p, c in zip(past, counts)]
    cache, table, slots = filled(kv_heads, dim, lengths, 1)
    q = normal((sum(counts), kv_heads * group, dim), dtype, 2, 1.5)
    out, lse = cache.attend(step(past, counts, table, slots), q, lse=True, window=window)
    check(cache, table, slots, past, counts, q, out, dtype, lse, window=window)


@pytest.mark.parametrize("kv_heads,group,dim,dtype", [(2, 4, 128, "f32"), (2, 4, 128, "bf16"), (1, 3, 64, "f16"),
                                                      (1, 7, 64, "f32"), (1, 1, 128, "f16"), (1, 1, 64, "bf16")])
@pytest.mark.parametrize("past,counts,window", [([0], [200], 0), ([70], [131], 0), ([0, 33], [90, 64], 0),
                                                ([64], [128], 50), ([100, 0, 3], [100, 1, 140], 64), ([250], [33], 0),
                                                ([5, 0], [96, 300], 7)])
def test_prompts(cuda, kv_heads, group, dim, dtype, past, counts, window):
    lengths = [p + c for p, c in zip(past, counts)]
    cache, table, slots = filled(kv_heads, dim, lengths, 2)
    q = normal((sum(counts), kv_heads * group, dim), dtype, 3, 1.5)
    out, lse = cache.attend(step(past, counts, table, slots), q, lse=True, window=window)
    check(cache, table, slots, past, counts, q, out, dtype, lse, window=window)
    again = cache.attend(step(past, counts, table, slots), q, window=window)
    assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [1, 3, 40])
def test_long_sequences_are_split_and_joined_alike(cuda, dtype, tokens):
    """One long sequence over many workgroups; two calls give the same bits."""
    length = 9000
    cache, table, slots = filled(1, 64, [length], 3)
    past = [length - tokens]
    q = normal((tokens, 3, 64), dtype, 4, 2.0)
    batch = step(past, [tokens], table, slots)
    out, lse = cache.attend(batch, q, lse=True)
    check(cache, table, slots, past, [tokens], q, out, dtype, lse)
    for _ in range(3):
        assert torch.equal(cache.attend(batch, q), out)


@pytest.mark.parametrize("tokens", [1, 50])
def test_peaked_and_shifted_scores(cuda, tokens):
    """Scores in the hundreds, a maximum that grows along the sequence, blocks
    whose numbers are a million times smaller than their neighbours'."""
    kv_heads, dim, length = 1, 128, 330
    cache, table, slots = make_cache(kv_heads, dim, 8, 1), ints([[0, 1, 2, 3, 4, 5]]), [0]
    k, v = normal((length, 1, dim), "f32", 5, 4.0), normal((length, 1, dim), "f32", 6)
    k *= torch.linspace(0.1, 3.0, length, device="cuda")[:, None, None]
    v[64:128] *= 1e-6
    k[128:192] *= 1e-6
    v[200:210] *= 100.0
    cache.append(step([0], [length], table), k, v)
    q = normal((tokens, 4, dim), "f32", 7, 3.0)
    past = [length - tokens]
    out, lse = cache.attend(step(past, [tokens], table), q, lse=True)
    check(cache, table, slots, past, [tokens], q, out, "f32", lse)


@pytest.mark.parametrize("tokens", [1, 4, 60])
def test_nan_stays_where_it_is_seen(cuda, tokens):
    """A NaN in a query row, in a full block outside the window, and in one
    head's open block: only rows that read it are NaN."""
    kv_heads, group, dim, length = 2, 2, 64, 200
    cache, table, slots = filled(kv_heads, dim, [length], 8)
    past = [length - tokens]
    q = normal((tokens, kv_heads * group, dim), "f32", 9)
    page = int(table[0, 0])
    saved = cache.scales[page].clone()
    cache.scales[page] = float("nan")
    window = length - 64 - tokens + 1  # the first row's window begins at token 64
    batch = step(past, [tokens], table, slots)
    out = cache.attend(batch, q, window=window)
    check(cache, table, slots, past, [tokens], q, out, "f32", window=window)
    assert torch.isnan(cache.attend(batch, q)).all()
    cache.scales[page] = saved
    for which in (0, 1):
        saved_open = cache.open_scales.clone()
        cache.open_scales[slots[0], 1, 1, which, 5] = float("nan")  # token 197 of kv head 1
        out = cache.attend(batch, q)
        seen = torch.arange(past[0], length, device="cuda") >= 197
        assert torch.equal(torch.isnan(out).any(-1), seen[:, None] & (torch.arange(4, device="cuda") >= 2)[None])
        assert torch.equal(torch.isnan(out).all(-1), torch.isnan(out).any(-1))
        cache.open_scales.copy_(saved_open)
    q[0, 1, 3] = float("nan")
    q[0, 2, 0] = float("inf")
    out = cache.attend(batch, q)
    bad = torch.zeros((tokens, 4), dtype=torch.bool, device="cuda")
    bad[0, 1:3] = True
    assert torch.equal(torch.isnan(out).any(-1), bad) and torch.equal(torch.isnan(out).all(-1), bad)


def test_zero_queries_scale_and_blocks(cuda):
    """All scores equal: the mean of the visible values; zero values give zero."""
    cache, table, slots = filled(1, 64, [150], 10)
    batch = step([149], [1], table, slots)
    q = torch.zeros((1, 2, 64), device="cuda")
    q[0, 1] = normal((64,), "f32", 11)
    out = cache.attend(batch, q, scale=0.0)
    check(cache, table, slots, [149], [1], q, out, "f32", scale=0.0)
    out = cache.attend(batch, q)
    check(cache, table, slots, [149], [1], q, out, "f32")
    zero = make_cache(1, 64, 3, 1)
    t = ints([[0, 1, 2]])
    k = torch.zeros((150, 1, 64), device="cuda")
    zero.append(step([0], [150], t), k, k)
    for tokens in (1, 70):
        q = normal((tokens, 2, 64), "f32", 12)
        assert (zero.attend(step([150 - tokens], [tokens], t), q) == 0).all()


@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("dtype,offset", [("f32", 1), ("bf16", 0), ("bf16", 3), ("f16", 8)])
def test_strided_rows(cuda, tokens, dtype, offset):
    kv_heads, group, dim = 2, 3, 64
    cache, table, slots = filled(kv_heads, dim, [170], 13)
    heads = kv_heads * group
    wide = normal((offset + tokens * (heads + 2) * dim,), dtype, 14)[offset:].view(tokens, heads + 2, dim)
    q = wide[:, 1:1 + heads]
    batch = step([170 - tokens], [tokens], table, slots)
    want = cache.attend(batch, q.contiguous())
    assert torch.equal(cache.attend(batch, q), want)
    into = torch.zeros((heads, tokens, dim + 1), dtype=DTYPES[dtype], device="cuda")
    out = into.transpose(0, 1)[:, :, :dim]
    assert cache.attend(batch, q, out=out) is out
    assert torch.equal(out, want) and (into[:, :, dim:] == 0).all()
    cache.attend(batch, q, out=q)
    assert torch.equal(q, want)


@pytest.mark.parametrize("tokens", [1, 48])
def test_bad_pages_give_nan_and_bad_sequences_are_skipped(cuda, tokens):
    cache, table, slots = filled(2, 64, [200, 100], 15)
    q = normal((2 * tokens, 4, 64), "f32", 16)
    past = [200 - tokens, 100 - tokens]
    want = cache.attend(step(past, [tokens] * 2, table, slots), q)
    broken = table.clone()
    broken[0, 1] = 10 ** 6
    out = cache.attend(step(past, [tokens] * 2, broken, slots), q)
    assert torch.isnan(out[:tokens]).all() and torch.equal(out[tokens:], want[tokens:]) and cache.faults() > 0
    for bad_past, bad_slot in ((-5, slots[0]), (10 ** 9, slots[0]), (past[0], 99)):
        before = cache.faults()
        out = torch.full_like(q, 7.0)
        cache.attend(step([bad_past, past[1]], [tokens] * 2, table, [bad_slot, slots[1]]), q, out=out)
        assert (out[:tokens] == 7.0).all() and torch.equal(out[tokens:], want[tokens:]) and cache.faults() > before


def test_graph_replays_with_other_lengths(cuda):
    """Append and attend captured once; replays read the lengths that are in
    the tensors then, and agree with eager calls, eager work in between."""
    from q4rdna import api
    kv_heads, dim, n = 2, 128, 3
    table = ints(np.arange(3 * 20).reshape(3, 20).tolist())
    graphed, eager = (make_cache(kv_heads, dim, 60, n) for _ in range(2))
    starts = [700, 63, 0]
    for c in (graphed, eager):
        total = sum(starts)
        c.append(step([0] * 3, starts, table), normal((total, kv_heads, dim), "f32", 20), normal((total, kv_heads, dim), "f32", 21))
    past = ints(starts)
    batch = api.KVBatch(past, table)
    k, v, q = (torch.zeros((n, h, dim), device="cuda") for h in (kv_heads, kv_heads, 8))
    out = torch.zeros_like(q)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graphed.append(batch, k, v)  # the shapes once on this stream, before the capture
        graphed.attend(batch, q, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        graphed.append(batch, k, v)
        graphed.attend(batch, q, out=out)
    for i in range(5):
        k.copy_(normal(k.shape, "f32", 30 + i))
        v.copy_(normal(v.shape, "f32", 40 + i))
        q.copy_(normal(q.shape, "f32", 50 + i))
        graph.replay()
        torch.cuda.synchronize()
        other = api.KVBatch(past.clone(), table)
        eager.append(other, k, v)
        assert torch.equal(eager.attend(other, q), out), i
        past += 1


def test_calls_on_two_streams(cuda):
    """The scratch belongs to the stream: overlapping calls do not disturb each other."""
    cache, table, slots = filled(1, 128, [4000], 22)
    batch = step([3999], [1], table, slots)
    qs = [normal((1, 4, 128), "f32", 60 + i) for i in range(2)]
    want = [cache.attend(batch, q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(cache.attend(batch, qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_a_prompt_s_row_equals_the_single_token(cuda):
    """Token 64 alone and as the last of its prompt, the same cache behind both."""
    kv_heads, dim, n = 2, 64, 65
    k, v, q = normal((n, kv_heads, dim), "f32", 70), normal((n, kv_heads, dim), "f32", 71), normal((n, 6, dim), "f32", 72)
    table = ints([[0, 1]])
    cache = make_cache(kv_heads, dim, 2, 1)
    cache.append(step([0], [n], table), k, v)
    whole = cache.attend(step([0], [n], table), q)
    single = cache.attend(step([n - 1], [1], table), q[n - 1:])
    # two results within the bound of `check`, sum |q k| / 8 under 16
    assert (single[0] - whole[n - 1]).abs().max() <= 4 * 2.0 ** -24 * (16 * 16 + 16) * v.abs().max()


@pytest.mark.parametrize("sequences,cu", [(70, False), (70, True), (130, True), (1100, False), (4200, True)])
def test_many_sequences(cuda, sequences, cu):
    """More sequences than a wave has lanes, than are dealt by length, and than
    two steps of the search over them reach; some long ones among them."""
    kv_heads, dim, group = 1, 64, 2
    r = np.random.RandomState(sequences)
    counts = [int(c) for c in r.randint(0, 3, sequences)] if cu else [1] * sequences
    counts[-1] = 1
    past = [int(p) for p in r.randint(0, 90, sequences)]
    past[sequences // 2], past[3] = 1500, 700
    lengths = [p + c for p, c in zip(past, counts)]
    cache, table, slots = filled(kv_heads, dim, lengths, 30)
    q = normal((sum(counts), kv_heads * group, dim), "f32", 31)
    batch = step(past, counts, table, slots)
    out = cache.attend(batch, q)
    every = list(range(sequences)) if sequences < 200 else sorted({0, 1, 3, sequences // 2, sequences - 1, *r.randint(0, sequences, 40)})
    at = np.concatenate([[0], np.cumsum(counts)])
    for i in every:
        if counts[i]:
            rows = slice(int(at[i]), int(at[i + 1]))
            check(cache, table[i:i + 1], slots[i:i + 1], past[i:i + 1], counts[i:i + 1], q[rows], out[rows], "f32")
    assert cache.faults() == 0


def test_a_prompt_among_single_tokens(cuda):
    """Both kernels in one call: long and short sequences take their own."""
    past, counts = [300, 0, 20, 511, 64], [1, 150, 1, 2, 70]
    cache, table, slots = filled(2, 128, [p + c for p, c in zip(past, counts)], 32)
    q = normal((sum(counts), 8, 128), "bf16", 33)
    batch = step(past, counts, table, slots)
    out, lse = cache.attend(batch, q, lse=True)
    check(cache, table, slots, past, counts, q, out, "bf16", lse)
    assert torch.equal(cache.attend(batch, q), out) and cache.faults() == 0


def test_the_batch_s_limit_may_be_generous(cuda):
    """max_tokens far above what the sequences have."""
    from q4rdna import api
    past, counts = [100, 3], [2, 1]
    cache, table, slots = filled(1, 64, [102, 4], 34)
    q = normal((3, 2, 64), "f32", 35)
    batch = api.KVBatch(ints(past), table, cu_tokens=ints([0, 2, 3]), slots=ints(slots), max_tokens=4000)
    check(cache, table, slots, past, counts, q, cache.attend(batch, q), "f32")


def test_refusals_of_the_python_calls(cuda):
    from q4rdna import api
    cache, table, slots = filled(2, 64, [70], 36)
    batch = step([69], [1], table, slots)
    q = normal((1, 4, 64), "f32", 37)
    for bad in (q[0], q.double(), q.cpu(), q[:, :, :32], q.transpose(1, 2), normal((2, 4, 64), "f32", 38)):
        with pytest.raises(ValueError):
            cache.attend(batch, bad)
    with pytest.raises(ValueError):
        cache.attend(batch, q, window=-1)
    with pytest.raises(ValueError):
        cache.attend(batch, q, out=torch.empty((1, 1, 64), device="cuda").expand(1, 4, 64))
    with pytest.raises(ValueError):
        cache.attend(batch, q, lse=torch.empty((4, 1), device="cuda"))
    with pytest.raises(api.Q4RdnaError):
        cache.attend(batch, normal((1, 3, 64), "f32", 39))
    with pytest.raises(ValueError):
        api.KVBatch(ints([0]).long(), table)
    with pytest.raises(ValueError):
        api.KVBatch(ints([0, 1]), table)
    with pytest.raises(ValueError):
        api.KVBatch(ints([0]), table, max_tokens=4)
    with pytest.raises(ValueError):
        api.KVCache(cache.pages, cache.scales[:-1], cache.open, cache.open_scales)
    k = normal((1, 2, 64), "f32", 40)
    with pytest.raises(ValueError):
        cache.append(batch, k, k.half())
    with pytest.raises(ValueError):
        cache.append(batch, k, k, q_out=q)
    with pytest.raises(ValueError):
        cache.append(batch, k, k, sin=k[0])
    with pytest.raises(ValueError):
        cache.read(batch, 2)
    with pytest.raises(ValueError):
        api.add_norm(k[0], k[0].half(), None)
    with pytest.raises(ValueError):
        api.add_norm(k[0], None, None, gate=k[0])
    with pytest.raises(ValueError):
        api.add_norm(k[0], k[0], torch.ones(63, device="cuda"))
    assert cache.faults() == 0
