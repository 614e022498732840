"""tree and attend_tree against their definitions in 64 bits."""
import itertools

import numpy as np
import pytest
import torch

import branch_reference as B
import layer_reference as R
from test_gpu_kv_attend import OUT_ROUND, WEIGHT_ROUND, filled
from test_gpu_kv_cache import f64, ints, make_cache, normal, snapshot, step

pytestmark = pytest.mark.gpu


def drafted(past, counts, table, slots=None):
    """A step whose sequences may have one token each or several."""
    from q4rdna import api
    return api.KVBatch(ints(past), table, cu_tokens=ints([0] + list(itertools.accumulate(counts))),
                       slots=None if slots is None else ints(slots), max_tokens=max(1, max(counts)))


def bits(values):
    return torch.tensor([v - (1 << 64) if v >> 63 else v for v in values], dtype=torch.int64, device="cuda")


def unsigned(t):
    return [int(v) & ((1 << 64) - 1) for v in t.cpu()]


def chains(counts, seed=0):
    """Parents of random trees, several roots among them."""
    r = np.random.RandomState(seed)
    return [int(r.randint(max(-1, j - 5), j)) if j else -1 for c in counts for j in range(c)]


def check(cache, table, slots, past, counts, q, k, v, seen, out, dtype, lse=None, scale=None, window=0):
    """Every row: |error| <= half a last place of the output, the weights'
    rounding times the largest |v| that the row sees, and the scores' roundings
    as weights': a chain of under 16 of 2^-24 of the largest products' sum,
    exp2's own, and numbers of q and k that two fp16 parts hold to 2^-23 of
    their row's largest, which counts once for each of the other's numbers.  (v
    is held like k: 2^-23 of the largest again, and the parts' products.)"""
    snap, rows = snapshot(cache), table.cpu().numpy()
    kv_heads, dim = cache.kv_heads, cache.head_dim
    group = q.shape[1] // kv_heads
    scale = dim ** -0.5 if scale is None else scale
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
            mine = got[at:at + c, heads].reshape(-1, dim)
            for r in range(len(x)):
                ks, vs = keys[sees[r]], values[sees[r]]
                if not len(ks):
                    assert (mine[r] == 0).all()
                    continue
                reach = scale * (np.abs(ks) @ np.abs(x[r])).max()
                parts = scale * (np.abs(ks).max() * np.abs(x[r]).sum() + np.abs(ks).sum(-1).max() * np.abs(x[r]).max())
                noise = 2.0 ** -24 * (16 * reach + 16) + 2.0 ** -23 * parts
                top = np.abs(vs).max()
                bound = OUT_ROUND[dtype] * np.abs(want[r]) + (WEIGHT_ROUND[dtype] + 2.0 ** -21 + 2 * noise) * top
                err = np.abs(mine[r] - want[r])
                assert (err <= bound).all(), (i, head, r, err.max(), bound.max())
                if lse is not None:
                    e = abs(f64(lse)[at:at + c, heads].reshape(-1)[r] - want_lse[r])
                    assert e <= noise + 2.0 ** -22 * (1 + abs(want_lse[r])), (i, head, r, e)
            if lse is not None:
                assert (np.isneginf(f64(lse)[at:at + c, heads].reshape(-1)) == np.isneginf(want_lse)).all()
        at += c


@pytest.mark.parametrize("counts", [[1], [1, 1, 1], [64], [5, 0, 63, 1, 64, 17]])
def test_positions_and_ancestors(cuda, counts):
    from q4rdna import api
    past = [(37 * i * i) % 500 for i in range(len(counts))]
    parents = chains(counts, len(counts))
    if counts == [64]:
        parents = list(range(-1, 63))  # a chain of the largest depth
    batch = drafted(past, counts, ints([[0]] * len(counts)))
    positions, seen = api.tree(batch, ints(parents))
    want = B.tree(past, counts, parents)
    assert positions.tolist() == want[0] and unsigned(seen) == want[1]
    assert positions.dtype == torch.int32 and seen.dtype == torch.int64


def test_bad_parents_and_sequences(cuda):
    """A parent that comes later, is itself, or does not exist: it and what is
    below it.  A sequence out of range: all its tokens.  Nothing behind the last."""
    from q4rdna import api
    table = ints([[0]] * 4)
    counts, past = [6, 2, 3, 2], [10, -1, 5, 2 ** 30 + 1]
    parents = [-1, 0, 3, 1, 2, -2, -1, 0, 0, 5, -1, -1, 0]
    cu = ints([0, 6, 8, 11, 13])
    batch = api.KVBatch(ints(past), table, cu_tokens=cu, max_tokens=6)
    positions, seen = torch.full((15,), 77, dtype=torch.int32, device="cuda"), torch.full((15,), 99, device="cuda")
    api.tree(batch, ints(parents + [0, 0]), positions=positions, seen=seen)
    want = B.tree(past, counts, parents)
    for i in (6, 7, 11, 12):
        want[0][i], want[1][i] = -1, 0
    assert want[0][2] == want[0][4] == want[0][5] == want[0][8] == -1
    assert positions.tolist() == want[0] + [77, 77] and unsigned(seen) == want[1] + [99, 99]
    # more tokens than max_tokens
    batch = api.KVBatch(ints([3]), table[:1].contiguous(), cu_tokens=ints([0, 5]), max_tokens=4)
    positions, seen = api.tree(batch, ints([-1] * 5))
    assert positions.tolist() == [-1] * 5 and seen.tolist() == [0] * 5


SHAPES = [(1, 1, 64), (2, 4, 128), (3, 5, 64), (1, 8, 128), (2, 12, 64), (1, 33, 128)]


@pytest.mark.parametrize("kv_heads,group,dim", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window", [0, 1, 3, 40, 130])
def test_trees_ragged(cuda, kv_heads, group, dim, dtype, window):
    from q4rdna import api
    past, counts = [0, 5, 60, 64, 190, 127, 300, 65], [1, 3, 9, 0, 2, 1, 6, 20]
    cache, table, slots = filled(kv_heads, dim, past, 1)
    n = sum(counts)
    q, k, v = (normal((n, h, dim), dtype, s, 1.5) for s, h in ((2, kv_heads * group), (3, kv_heads), (4, kv_heads)))
    batch = drafted(past, counts, table, slots)
    _, seen = api.tree(batch, ints(chains(counts)))
    before = snapshot(cache)
    out, lse = cache.attend_tree(batch, q, k, v, seen, lse=True, window=window)
    check(cache, table, slots, past, counts, q, k, v, seen, out, dtype, lse, window=window)
    assert torch.equal(cache.attend_tree(batch, q, k, v, seen, window=window), out)
    after = snapshot(cache)
    assert cache.faults() == 0 and all(np.array_equal(before[x], after[x], equal_nan=before[x].dtype != np.int8) for x in before)


@pytest.mark.parametrize("dtype,kv_heads,group,dim,past,count,window",
                         [("f32", 1, 3, 64, 9000, 1, 0), ("bf16", 1, 4, 128, 9000, 16, 0), ("f32", 2, 4, 128, 3000, 64, 0),
                          ("f16", 2, 7, 64, 4097, 63, 1000), ("bf16", 2, 2, 128, 2048, 33, 64), ("f32", 1, 1, 128, 6000, 64, 0)])
def test_long_sequences_are_split_and_joined_alike(cuda, dtype, kv_heads, group, dim, past, count, window):
    """One long sequence over many workgroups; calls give the same bits."""
    from q4rdna import api
    cache, table, slots = filled(kv_heads, dim, [past], 3)
    q, k, v = (normal((count, h, dim), dtype, s, 1.5) for s, h in ((5, kv_heads * group), (6, kv_heads), (7, kv_heads)))
    batch = drafted([past], [count], table, slots)
    _, seen = api.tree(batch, ints(chains([count], 5)))
    out, lse = cache.attend_tree(batch, q, k, v, seen, lse=True, window=window)
    check(cache, table, slots, [past], [count], q, k, v, seen, out, dtype, lse, window=window)
    for _ in range(3):
        assert torch.equal(cache.attend_tree(batch, q, k, v, seen, window=window), out)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_any_mask(cuda, dtype):
    """Masks that are no trees: later tokens, none, all, bits beyond the sequence."""
    past, counts = [0, 70, 0], [7, 12, 64]
    cache, table, slots = filled(2, 64, past, 4)
    n = sum(counts)
    r = np.random.RandomState(3)
    masks = [int(r.randint(0, 2 ** 31)) | int(r.randint(0, 2 ** 31)) << 33 for _ in range(n)]
    masks[0] = masks[9] = masks[40] = 0
    masks[3] = masks[10] = 2 ** 64 - 1
    seen = bits(masks)
    q, k, v = (normal((n, h, 64), dtype, s) for s, h in ((8, 6), (9, 2), (10, 2)))
    batch = drafted(past, counts, table, slots)
    for window in (0, 5, 66):
        out, lse = cache.attend_tree(batch, q, k, v, seen, lse=True, window=window)
        check(cache, table, slots, past, counts, q, k, v, seen, out, dtype, lse, window=window)
    assert (cache.attend_tree(batch, q, k, v, seen)[[0, 40]] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("past", [0, 130])
def test_what_is_not_a_number_stays_where_it_is_seen(cuda, dtype, past):
    """A NaN, an infinity, the type's largest and lowest numbers in drafts that
    some rows do not see."""
    from q4rdna import api
    kv_heads, group, dim, count = 2, 2, 64, 12
    cache, table, slots = filled(kv_heads, dim, [past], 8)
    q, k, v = (normal((count, h, dim), dtype, s) for s, h in ((11, 4), (12, 2), (13, 2)))
    batch = drafted([past], [count], table, slots)
    parents = chains([count], 2)
    _, seen = api.tree(batch, ints(parents))
    sees = (seen[:, None] >> torch.arange(count, device="cuda")) & 1 > 0
    want = cache.attend_tree(batch, q, k, v, seen)
    for at, which, value in ((4, k, float("nan")), (7, v, float("inf")), (2, v, float("nan")), (5, k, -float("inf"))):
        saved = which[at, 1, 3].clone()
        which[at, 1, 3] = value
        out, lse = cache.attend_tree(batch, q, k, v, seen, lse=True)
        which[at, 1, 3] = saved
        bad = sees[:, at][:, None] & (torch.arange(4, device="cuda") >= 2)[None]
        assert torch.equal(torch.isnan(out).any(-1), bad) and torch.equal(torch.isnan(out).all(-1), bad)
        assert torch.equal(out[~bad], want[~bad])
        assert (torch.isnan(lse) == (bad if which is k else torch.zeros_like(bad))).all()
    # a loud draft beside quiet ones: rows that do not see it keep their own last places
    loud = torch.finfo(v.dtype).max
    v[6, 0] = loud
    k[6, 0, :] = torch.finfo(v.dtype).min / 2 ** 10 if dtype == "f16" else -1e4
    out = cache.attend_tree(batch, q, k, v, seen)
    blind = ~sees[:, 6]
    assert torch.equal(out[blind], want[blind]) and torch.equal(out[:, 2:], want[:, 2:])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_loud_and_quiet_drafts_and_blocks(cuda, dtype):
    """Keys and values of drafts a factor of 10^20 apart from each other and from
    the cache's: each row by its own sum of p |v|."""
    from q4rdna import api
    dim, past, count = 64, 200, 16
    cache, table, slots = make_cache(1, dim, 6, 1), ints([[0, 1, 2, 3, 4]]), [0]
    k0, v0 = normal((past, 1, dim), "f32", 14), normal((past, 1, dim), "f32", 15)
    v0[64:128] *= 1e-20
    cache.append(step([0], [past], table), k0, v0)
    for spread in (1e-25, 1e-12, 1e12, 1e25):
        q, k, v = (normal((count, h, dim), dtype, s) for s, h in ((16, 2), (17, 1), (18, 1)))
        v[::2] *= spread
        batch = drafted([past], [count], table)
        _, seen = api.tree(batch, ints(chains([count], 6)))
        for window in (0, 8):
            out = f64(cache.attend_tree(batch, q, k, v, seen, window=window))
            snap = snapshot(cache)
            keys = np.concatenate((R.tokens_of(snap, [0, 1, 2, 3], 0, past, 0, 0), f64(k)[:, 0]))
            values = np.concatenate((R.tokens_of(snap, [0, 1, 2, 3], 0, past, 0, 1), f64(v)[:, 0]))
            sees = np.repeat(B.visible(past, count, unsigned(seen), window), 2, axis=0)
            x = f64(q).reshape(-1, dim)
            want = B.attend(x, keys, values, sees, dim ** -0.5)[0].reshape(out.shape)
            size = B.attend(x, keys, np.abs(values), sees, dim ** -0.5)[0].reshape(out.shape)
            # a token's own largest |v| scales its 2^-23 roundings: up to 4 times its rms here, per number
            size = np.broadcast_to(size.max(-1, keepdims=True), out.shape)
            noise = 2.0 ** -24 * (16 * 8 + 16) * 4
            assert (np.abs(out - want) <= OUT_ROUND[dtype] * np.abs(want) + (WEIGHT_ROUND[dtype] + 2.0 ** -21 + noise) * size).all(), spread


@pytest.mark.parametrize("dtype,offset", [("f32", 1), ("bf16", 0), ("bf16", 3), ("f16", 8)])
def test_strides_and_alignment(cuda, dtype, offset):
    """Rows in a larger tensor, at odd places, heads and tokens in other orders."""
    from q4rdna import api
    past, counts, dim = [70, 3], [5, 9], 64
    cache, table, slots = filled(2, dim, past, 5)
    batch = drafted(past, counts, table, slots)
    _, seen = api.tree(batch, ints(chains(counts)))
    n = sum(counts)
    q, k, v = (normal((n, h, dim), dtype, s) for s, h in ((19, 6), (20, 2), (21, 2)))
    want = cache.attend_tree(batch, q, k, v, seen)

    def moved(x, turned):
        big = torch.zeros((x.shape[0] * x.shape[1] * (dim + 24) + offset,), dtype=x.dtype, device="cuda")
        shape = (x.shape[1], x.shape[0]) if turned else (x.shape[0], x.shape[1])
        y = big[offset:].view(*shape, dim + 24)[..., :dim]
        y = y.transpose(0, 1) if turned else y
        y.copy_(x)
        return y

    for turned in (False, True):
        out = moved(torch.zeros_like(q), turned)
        got = cache.attend_tree(batch, moved(q, turned), moved(k, turned), moved(v, not turned), seen, out=out)
        assert got is out and torch.equal(out, want)
    with pytest.raises(ValueError):
        cache.attend_tree(batch, q, k, v, seen, out=want[:, :1].expand(-1, 6, -1))


def test_refused_entries_and_rows_behind(cuda):
    """Bad lengths, slots and pages: counted, their rows not written or NaN."""
    from q4rdna import api
    dim = 64
    cache, table, slots = filled(1, dim, [100, 100, 100], 6)
    counts = [2, 3, 2]
    n = sum(counts) + 2
    q, k, v = (normal((n, 1, dim), "f32", s) for s in (22, 23, 24))
    seen = torch.ones(n, dtype=torch.int64, device="cuda")

    def call(past=(100, 100, 100), slots=slots, table=table, cu=(0, 2, 5, 7), most=3):
        out = torch.full_like(q, 55.0)
        before = cache.faults()
        cache.attend_tree(api.KVBatch(ints(list(past)), table, cu_tokens=ints(list(cu)), slots=ints(list(slots)), max_tokens=most),
                          q, k, v, seen, out=out)
        return out, cache.faults() - before

    want, faults = call()
    assert faults == 0 and (want[7:] == 55.0).all() and not (want[:7] == 55.0).any()
    for change in (dict(past=(100, -1, 100)), dict(past=(100, 129, 100)), dict(slots=(slots[0], 4, slots[2])),
                   dict(slots=(slots[0], -1, slots[2])), dict(most=2)):
        out, faults = call(**change)
        assert faults == 1 and (out[2:5] == 55.0).all() and (out[7:] == 55.0).all()
        assert torch.equal(out[:2], want[:2]) and torch.equal(out[5:7], want[5:7]), change
    out, faults = call(cu=(0, 2, 10, 12))
    assert faults == 2 and torch.equal(out[:2], want[:2]) and (out[2:] == 55.0).all()
    bad = table.clone()
    bad[1, 0] = 1000
    out, faults = call(table=bad)
    assert faults >= 1 and torch.isnan(out[2:5]).all() and torch.equal(out[5:7], want[5:7])


def test_many_sequences(cuda):
    """More than one scan's sequences, and more than are dealt by length."""
    from q4rdna import api
    for n, count in ((70, 3), (300, 2)):
        past = [(i * 37) % 300 for i in range(n)]
        counts = [1 + (i % count) for i in range(n)]
        cache, table, slots = filled(1, 64, past, 7)
        total = sum(counts)
        q, k, v = (normal((total, h, 64), "bf16", s) for s, h in ((25, 2), (26, 1), (27, 1)))
        batch = drafted(past, counts, table, slots)
        _, seen = api.tree(batch, ints(chains(counts, 9)))
        out = cache.attend_tree(batch, q, k, v, seen)
        check(cache, table, slots, past, counts, q, k, v, seen, out, "bf16")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_chain_is_what_appended_tokens_see(cuda, dtype):
    """A chain of drafts gives what attend gives after the same tokens were
    appended, but for their rounding to 16-bit codes (2^-16 of a token's largest
    in k and in v) while they lie in the open block."""
    from q4rdna import api
    kv_heads, group, dim, past, count = 2, 4, 128, 65, 20
    cache, table, slots = filled(kv_heads, dim, [past], 9)
    table = torch.cat((table, ints([[0]])), 1).contiguous()
    q, k, v = (normal((count, h, dim), dtype, s) for s, h in ((28, 8), (29, 2), (30, 2)))
    batch = drafted([past], [count], table, slots)
    _, seen = api.tree(batch, ints(list(range(-1, count - 1))))
    got = cache.attend_tree(batch, q, k, v, seen)
    cache.append(batch, k, v)
    want = cache.attend(batch, q)
    # a score moves by scale * sum |q| * 2^-16 max |k|, 2^-16 * 128 * 0.8 * 4 / 11.3 = 36 * 2^-16, as the weights do
    top = float(v.float().abs().max())
    assert (got.float() - want.float()).abs().max() <= (2 * 36 * 2.0 ** -16 + 2.0 ** -16 + 2 * OUT_ROUND[dtype]) * top


def test_captured_and_replayed(cuda):
    """Replays with other lengths, masks and trees in the same tensors."""
    from q4rdna import api
    dim, lengths = 64, [3000, 900]
    cache, table, slots = filled(2, dim, lengths, 10)
    past, cu, parents = ints(lengths), ints([0, 9, 20]), ints(chains([9, 11], 3))
    q, k, v = (normal((20, h, dim), "f32", s) for s, h in ((31, 6), (32, 2), (33, 2)))
    batch = api.KVBatch(past, table, cu_tokens=cu, slots=ints(slots), max_tokens=16)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def call():
        positions, seen = api.tree(batch, parents)
        return positions, seen, cache.attend_tree(batch, q, k, v, seen)

    with torch.cuda.stream(stream):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = call()
    torch.cuda.synchronize()
    for lengths, counts, seed in (([3000, 900], [9, 11], 3), ([70, 2900], [4, 16], 5), ([0, 64], [16, 4], 6), ([3000, 0], [10, 10], 7)):
        if lengths[1] > 900:  # (its table has that many pages)
            lengths[1] = 900
        past.copy_(ints(lengths))
        cu.copy_(ints([0, counts[0], 20]))
        parents.copy_(ints(chains(counts, seed)))
        q.copy_(normal(tuple(q.shape), "f32", 40 + seed))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in got]
        eager = call()
        assert all(torch.equal(a, b) for a, b in zip(replayed, eager))


def test_gradients_and_shapes_are_refused(cuda):
    from q4rdna import api
    cache, table, slots = filled(1, 64, [10], 11)
    batch = drafted([10], [3], table, slots)
    q, k, v = (normal((3, h, 64), "f32", s) for s, h in ((34, 2), (35, 1), (36, 1)))
    seen = torch.ones(3, dtype=torch.int64, device="cuda")
    ok = dict(q=q, k=k, v=v, seen=seen)
    for change in (dict(q=q[0]), dict(k=k[:2]), dict(v=v.half()), dict(seen=seen.int()), dict(seen=seen[:2]), dict(q=q[:, :, :32]),
                   dict(k=k.cpu()), dict(q=q.clone().requires_grad_()), dict(v=v.clone().requires_grad_())):
        with pytest.raises(ValueError):
            cache.attend_tree(batch, **{**ok, **change})
    with pytest.raises(ValueError):
        cache.attend_tree(batch, **ok, window=-1)
    wide = api.KVBatch(ints([10]), table, cu_tokens=ints([0, 3]), slots=ints(slots))  # max_tokens not given
    for call in (lambda: cache.attend_tree(wide, **ok), lambda: api.tree(wide, ints([-1, 0, 1]))):
        with pytest.raises(api.Q4RdnaError, match="max_tokens"):
            call()
    with pytest.raises(ValueError):
        api.tree(batch, ints([[-1, 0, 1]]))


def test_streams(cuda):
    """stream=: outputs come from that stream's memory, and wait for its work."""
    from q4rdna import api
    cache, table, slots = filled(1, 64, [500], 12)
    batch = drafted([500], [30], table, slots)
    q, k, v = (normal((30, h, 64), "bf16", s) for s, h in ((37, 4), (38, 1), (39, 1)))
    parents = ints(chains([30], 8))
    positions, seen = api.tree(batch, parents)
    want = cache.attend_tree(batch, q, k, v, seen, lse=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = api.tree(batch, parents, stream=side.cuda_stream) + cache.attend_tree(batch, q, k, v, seen, lse=True, stream=side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, (positions, seen) + want))


@pytest.mark.parametrize("group", [8191, 9001, 32767, 32768])
def test_many_query_heads_of_a_kv_head(cuda, group):
    """Rows are counted off right however many share a kv head: with one value
    per token and head a row's result tells its token, its query its head."""
    from q4rdna import api
    dim, n = 64, 3
    cache = api.KVCache.empty(1, 1, 1, dim)
    step = api.KVBatch(torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros((1, 1), dtype=torch.int32, device="cuda"),
                       cu_tokens=torch.tensor([0, n], dtype=torch.int32, device="cuda"), max_tokens=n)
    k = torch.zeros(n, 1, dim, device="cuda", dtype=torch.float16)
    k[:, 0, 0] = 1.0
    v = torch.arange(1, n + 1, device="cuda").half()[:, None, None].expand(n, 1, dim).contiguous()
    head = (torch.arange(group, device="cuda") % 2039 - 1019).half()
    q = torch.zeros(n, group, dim, device="cuda", dtype=torch.float16)
    q[:, :, 0] = head
    seen = torch.tensor([1, 2, 4], dtype=torch.int64, device="cuda")  # each itself alone
    out, lse = cache.attend_tree(step, q, k, v, seen, scale=1.0, lse=True)
    assert torch.equal(out, v.expand(n, group, dim))
    assert ((lse - head.float()).abs() <= 2.0 ** -20 * head.float().abs() + 2.0 ** -20).all()


@pytest.mark.parametrize("dtype,n,kv_heads,dim", [("f32", 40, 2, 128), ("bf16", 70, 2, 128), ("f16", 100, 1, 64), ("f32", 9, 8, 64)])
def test_long_and_short_sequences_together(cuda, dtype, n, kv_heads, dim):
    """Lengths of every size and tables as wide as the longest: each sequence
    alone gives what the batch gives, up to the order of its parts (fp32
    accumulators, two fp16 parts: 2^-18 of the largest; 16-bit outputs a rounding
    apart)."""
    from q4rdna import api
    r = np.random.RandomState(n)
    past = [int(x) for x in np.exp(r.uniform(0, np.log(9000), n))]
    count = [int(x) for x in r.randint(0, 20, n)]
    width = max(past) // 64 + 1
    pages = sum(p // 64 + 1 for p in past)
    cache = api.KVCache.empty(pages, n, kv_heads, dim)
    order, rows, at = r.permutation(pages), np.full((n, width), -1), 0
    for i, p in enumerate(past):
        rows[i, :p // 64 + 1] = order[at:at + p // 64 + 1]
        at += p // 64 + 1
    ints = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
    table, slots, starts = ints(rows), ints(r.permutation(n)), lambda c: ints(np.concatenate([[0], np.cumsum(c)]))  # noqa: E731
    torch.manual_seed(n)
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    k, v = torch.randn(2, sum(past), kv_heads, dim, device="cuda", dtype=t)
    cache.append(api.KVBatch(ints([0] * n), table, starts(past), slots, max_tokens=max(past)), k, v)
    total = sum(count)
    q, dk, dv = (torch.randn(total, h, dim, device="cuda", dtype=t) for h in (4 * kv_heads, kv_heads, kv_heads))
    step = api.KVBatch(ints(past), table, starts(count), slots, max_tokens=20)
    up = [j - 1 if r.rand() < 0.7 else max(j - 3, -1) for c in count for j in range(c)]
    _, seen = api.tree(step, ints(up))
    out, lse = cache.attend_tree(step, q, dk, dv, seen, lse=True)
    assert cache.faults() == 0
    at = 0
    for i in range(n):
        rows = slice(at, at + count[i])
        at += count[i]
        if count[i]:
            one = api.KVBatch(ints(past[i:i + 1]), table[i:i + 1], starts(count[i:i + 1]), slots[i:i + 1], max_tokens=20)
            a, b = cache.attend_tree(one, q[rows], dk[rows], dv[rows], seen[rows], lse=True)
            step_of = 2.0 ** -18 if dtype == "f32" else torch.finfo(t).eps
            assert ((a.float() - out[rows].float()).abs() <= step_of * a.float().abs().amax(-1, keepdim=True)).all()
            assert ((b - lse[rows]).abs() <= 2.0 ** -18 * (1 + b.abs())).all()
