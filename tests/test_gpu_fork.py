"""KVBatch.fork against its definition."""
import numpy as np
import pytest
import torch

import branch_reference as B
from test_gpu_kv_cache import f64, ints, make_cache, normal, step

pytestmark = pytest.mark.gpu


def state(past, width, pages, slot_count, layers=2, kv_heads=2, dim=64, seed=0):
    """(caches, batch, past, table, slots): rows of full blocks in distinct random pages."""
    from q4rdna import api
    r = np.random.RandomState(seed)
    n = len(past)
    order = list(r.permutation(pages))
    rows = [[order.pop() if b < p // 64 and order else -1 for b in range(width)] for p in past]
    slots = [int(x) for x in r.permutation(slot_count)[:n]]
    caches = [make_cache(kv_heads, dim, pages, slot_count, seed + i) for i in range(layers)]
    for c in caches:
        c.open_scales.copy_(torch.rand(c.open_scales.shape, generator=torch.Generator().manual_seed(seed)))
    p, t, s = ints(past), ints(rows), ints(slots)
    return caches, api.KVBatch(p, t, slots=s), p, t, s


def run(caches, batch, past, table, slots, parents, room=1, kept=None):
    """One fork, its tensors and every byte of the caches against the definition."""
    before = [[x.cpu().numpy().copy() for x in (c.open, c.open_scales, c.pages)] for c in caches]
    pages, slot_count, faults = caches[0].pages.shape[0], caches[0].open.shape[0], caches[0].faults()
    marked = () if kept is None else set(kept.cpu().nonzero().flatten().tolist())
    want = B.fork(past.tolist(), table.tolist(), slots.tolist(), list(parents), pages, room, slot_count, marked)
    batch.fork(ints(list(parents)), caches, room=room, kept=kept)
    assert past.tolist() == want[0]
    assert table.tolist() == want[1]
    assert slots.tolist() == want[2]
    assert caches[0].faults() - faults == want[4]
    for c, (planes, scales, codes) in zip(caches, before):
        for src, dst, block in want[3]:
            planes[dst, block % 2], scales[dst, block % 2] = planes[src, block % 2].copy(), scales[src, block % 2].copy()
        assert np.array_equal(c.open.cpu().numpy(), planes) and np.array_equal(c.open_scales.cpu().numpy(), scales)
        assert np.array_equal(c.pages.cpu().numpy(), codes)


@pytest.mark.parametrize("past,parents", [
    ([70], [0]), ([70, 0], [0, 0]), ([0, 0], [1, 1]), ([64, 200], [1, 1]), ([63, 130, 128, 5], [1, 1, 2, 1]),
    ([300, 300, 300, 300, 300], [4, 3, 2, 1, 0]), ([10, 700, 64, 65], [3, 2, 1, 0]), ([5, 6, 7], [-1, 0, -1]), ([5, 6, 7], [-1, -1, -1]),
    ([500, 400, 300, 200], [3, 3, 3, 3])])
@pytest.mark.parametrize("room", [0, 1, 64, 300])
@pytest.mark.parametrize("dim,kv_heads", [(64, 2), (128, 3)])
def test_against_the_definition(cuda, past, parents, room, dim, kv_heads):
    width = (max(past) + room + 63) // 64 + 1
    s = state(past, width, len(past) * width + 3, len(past) + 2, dim=dim, kv_heads=kv_heads, seed=len(past) + room)
    run(*s, parents, room)
    run(*s, [0] * len(past), room)


@pytest.mark.parametrize("n,layers,pages", [(33, 1, 700), (64, 3, 2000), (1500, 1, 20000)])
def test_random_forks_one_after_the_other(cuda, n, layers, pages):
    """Renamed, shared, dropped and given out again, also on the rows that forks left."""
    r = np.random.RandomState(n)
    past = [int(x) for x in r.randint(0, 64 * min(12, pages // n), n)]
    s = state(past, 14, pages, n, layers=layers, kv_heads=1, seed=n)
    for room in (1, 100, 5):
        run(*s, [int(x) for x in r.randint(-1, n, n)], room)
        s[2].copy_(torch.clamp(s[2] + room, max=14 * 64) * (s[2] > 0))


def test_pages_run_out_and_kept_ones_stay(cuda):
    s = state([130, 130, 70], 5, 8, 3, seed=3)  # five pages held, three free
    kept = torch.zeros(8, dtype=torch.bool, device="cuda")
    kept[:3] = True
    run(*s, [0, 1, 2], 130, kept=kept.to(torch.uint8))
    s = state([130, 130, 70], 5, 8, 3, seed=3)
    run(*s, [0, 0, 0], 200, kept=kept)
    s = state([0, 0, 0], 2, 1, 3, seed=4)
    run(*s, [0, 1, 2], 1)
    s = state([0], 4, 40, 1, seed=5)  # the last word of the pages' bits
    run(*s, [0], 256, kept=torch.ones(40, dtype=torch.bool, device="cuda"))


def test_refused_entries(cuda):
    """Parents, lengths and slots out of range: counted, the sequence dropped."""
    for change in (dict(parents=[3, 0, 1]), dict(parents=[-2, 0, 1]), dict(parents=[2 ** 31 - 1, -2 ** 31, 1]), dict(past=[-1, 70, 10]),
                   dict(past=[64 * 4 + 1, 70, 10]), dict(slots=[7, 1, 2]), dict(slots=[-1, 1, 2]), dict(slots=[0, 1, 9], parents=[0, 0, 1])):
        caches, batch, past, table, slots = state([130, 70, 10], 4, 12, 3, seed=6)
        if "past" in change:
            past.copy_(ints(change["past"]))
        if "slots" in change:
            slots.copy_(ints(change["slots"]))
        run(caches, batch, past, table, slots, change.get("parents", [0, 0, 2]), 1)


def test_bad_pages_pass_through(cuda):
    """Entries outside the cache are neither held nor a fault here."""
    caches, batch, past, table, slots = state([130, 200], 4, 12, 2, seed=7)
    table[0, 0], table[1, 2] = 10000, -7
    run(caches, batch, past, table, slots, [1, 1], 1)


def test_forked_sequences_read_and_grow_alike(cuda):
    """Tokens appended to forks: each reads its parent's tokens and then its own,
    pages are never written twice, tokens can be taken back into the block before."""
    from q4rdna import api
    n, kv, dim = 4, 2, 64
    cache = api.KVCache.empty(40, n, kv, dim)
    past, table, slots = ints([0] * n), torch.full((n, 8), -1, dtype=torch.int32, device="cuda"), ints([2, 0, 3, 1])
    batch = api.KVBatch(past, table, slots=slots)
    tokens = [[] for _ in range(n)]
    r = np.random.RandomState(5)
    for at in range(300):
        parents = [int(x) for x in r.randint(0, n, n)] if at % 3 == 0 else list(range(n))
        batch.fork(ints(parents), [cache], room=1)
        tokens = [list(tokens[p]) for p in parents]
        k, v = normal((n, kv, dim), "f32", 2 * at), normal((n, kv, dim), "f32", 2 * at + 1)
        cache.append(batch, k, v)
        past += 1
        for i in range(n):
            tokens[i].append((at, i))
        if at in (5, 62, 63, 64, 100, 200, 299):
            length = at + 1
            whole = api.KVBatch(ints([0] * n), table, cu_tokens=ints([length * i for i in range(n + 1)]), slots=slots, max_tokens=length)
            got = [f64(x).reshape(n, length, kv, dim) for x in cache.read(whole, n * length)]
            for which in (0, 1):
                made = np.stack([f64(normal((n, kv, dim), "f32", 2 * t + which)) for t in range(length)])
                for i in range(n):
                    want = np.stack([made[t, j] for t, j in tokens[i]])
                    # half a step of 8 bits of a full block's largest number, 16 bits in the open one
                    for b in range(0, length, 64):
                        top = np.abs(want[b:b + 64]).max(axis=(0, 2), keepdims=True)
                        step_ = top / 254 if b + 64 <= length else top / 65024
                        assert (np.abs(got[which][i, b:b + 64] - want[b:b + 64]) <= step_ * 1.001 + top / 65024).all(), (at, i, b)
    assert cache.faults() == 0
    # taken back to the block before the last
    batch.fork(ints([1, 1, 1, 2]), [cache], room=1)
    back = api.KVBatch(ints([0] * n), table, cu_tokens=ints([250 * i for i in range(n + 1)]), slots=slots, max_tokens=250)
    got = cache.read(back, n * 250)
    assert all(torch.equal(x.view(n, 250, kv, dim)[0], x.view(n, 250, kv, dim)[i]) for x in got for i in (1, 2))


def test_more_layers_than_a_launch_takes(cuda):
    caches, batch, past, table, slots = state([70, 10, 64], 3, 12, 3, layers=70, kv_heads=1, seed=8)
    run(caches, batch, past, table, slots, [0, 0, 0], 1)


def test_captured_and_replayed(cuda):
    from q4rdna import api
    caches, batch, past, table, slots = state([130, 70, 10, 300], 8, 40, 4, seed=9)
    parents = ints([0, 0, 1, 1])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    keep = [t.clone() for t in (past, table, slots)]
    with torch.cuda.stream(stream):
        batch.fork(parents, caches)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            batch.fork(parents, caches)
    torch.cuda.synchronize()
    for t, k in zip((past, table, slots), keep):
        t.copy_(k)
    for p in ([0, 0, 1, 1], [3, 2, 1, 0], [-1, 2, 2, 2], [1, 1, 1, 1]):
        before = [x.clone() for c in caches for x in (c.open, c.open_scales)]
        want = B.fork(past.tolist(), table.tolist(), slots.tolist(), p, 40, 1, 4)
        parents.copy_(ints(p))
        graph.replay()
        torch.cuda.synchronize()
        assert past.tolist() == want[0] and table.tolist() == want[1] and slots.tolist() == want[2]
        for x in before:
            for src, dst, block in want[3]:
                x[dst, block % 2] = x[src, block % 2].clone()
        assert all(torch.equal(a, b) for a, b in zip(before, [x for c in caches for x in (c.open, c.open_scales)]))
        past += 30


def test_refusals(cuda):
    from q4rdna import api
    caches, batch, past, table, slots = state([5, 6], 2, 4, 2)
    ok = ints([0, 1])
    with pytest.raises(ValueError, match="slots"):
        api.KVBatch(past, table).fork(ok, caches)
    for call in (lambda: batch.fork(ok, []), lambda: batch.fork(ok[:1], caches), lambda: batch.fork(ok.long(), caches),
                 lambda: batch.fork(ok.cpu(), caches), lambda: batch.fork(ok, caches, room=-1),
                 lambda: batch.fork(ok, caches, kept=torch.zeros(3, dtype=torch.bool, device="cuda")),
                 lambda: batch.fork(ok, caches, kept=ints([0, 0, 0, 0]))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(api.Q4RdnaError, match="geometry"):
        batch.fork(ok, caches + [make_cache(2, 64, 5, 2)])
    with pytest.raises(api.Q4RdnaError, match="share"):
        batch.fork(ok, caches + caches[:1])
    assert past.tolist() == [5, 6]


@pytest.mark.parametrize("width", [1, 2, 3, 4, 5, 6, 7, 9])
def test_rows_of_few_columns(cuda, width):
    """Full to the last entry, or short of it; the last row ends where the table does."""
    past = [64 * width, 64 * width - 1, 64 * (width - 1), 3, 64 * width]
    for parents in ([0, 1, 2, 3, 4], [4, 4, 0, 1, 2], [4, 4, 4, 4, 4], [3, -1, 1, 0, 0]):
        s = state(past, width, 6 * width + 1, 5, seed=width)
        run(*s, parents, 64)
        run(*s, [1, 0, 2, 4, 4], 64 * width)


def test_kept_pages_of_a_large_cache(cuda):
    """More marks than the workgroup reads at a time, the last one's included."""
    pages = 20011
    s = state([700, 64, 6400, 1], 200, pages, 4, seed=8)
    kept = torch.rand(pages, generator=torch.Generator().manual_seed(9)).lt(0.9)
    kept[-3:] = torch.tensor([False, True, True])
    run(*s, [2, 2, 0, 1], 6000, kept=kept.cuda())
    run(*s, [0, 1, 2, 3], 64, kept=kept.cuda())


@pytest.mark.parametrize("n,width,pages,layers", [
    (256, 16, 2000, 1), (257, 16, 2000, 1), (256, 17, 2000, 1), (16, 256, 3000, 2), (15, 300, 3000, 2), (3, 64, 65536, 1), (3, 64, 65537, 1),
    (1, 4096, 5000, 1), (1, 5000, 5000, 1), (256, 128, 20000, 1), (256, 129, 20000, 1), (200, 100, 20000, 3), (7, 4000, 20000, 1)])
def test_either_side_of_one_launch(cuda, n, width, pages, layers):
    """Small tables take one launch, others two: the same results."""
    r = np.random.RandomState(n + width)
    past = [int(x) for x in r.randint(0, 64 * min(width, pages // n) - 100, n)]
    s = state(past, width, pages, n + 1, layers=layers, kv_heads=1, seed=n)
    for room in (1, 70, 0):
        run(*s, [int(x) for x in r.randint(-1, n, n)], room)
    run(*s, list(range(n)), 10000)


@pytest.mark.parametrize("n", [60, 200])
def test_more_entries_than_pages(cuda, n):
    """Pages for 16 columns of every sequence are wanted, few are there."""
    s = state([5] * n, 16, 100, n, layers=1, kv_heads=1, seed=n)
    run(*s, [0] * n, 1024)
    run(*s, [n - 1] * n, 1024)
