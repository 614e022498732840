"""Several threads that call on one stream: each call's results are those that it
has alone, bit for bit."""
import threading

import numpy as np
import pytest
import torch

from test_gpu_attend_tree import chains, drafted
from test_gpu_fork import state
from test_gpu_kv_attend import filled
from test_gpu_kv_cache import ints, normal, step

pytestmark = pytest.mark.gpu


def tree_of(dtype, past, count, seed):
    """attend_tree of a long sequence, whose parts are joined by a second launch."""
    from q4rdna import api
    cache, table, slots = filled(2, 128, [past], seed)
    q, k, v = (normal((count, h, 128), dtype, seed + i) for i, h in ((1, 8), (2, 2), (3, 2)))
    batch = drafted([past], [count], table, slots)
    _, seen = api.tree(batch, ints(chains([count], seed)))
    return lambda: cache.attend_tree(batch, q, k, v, seen, lse=True)


def one_token(past, seed):
    cache, table, slots = filled(2, 128, [past], seed)
    q = normal((1, 8, 128), "f32", seed + 1)
    batch = step([past - 1], [1], table, slots)
    return lambda: (cache.attend(batch, q),)


def beams(groups, count, seed):
    from q4rdna import api
    logits, scores = normal((groups, 4, 30000), "f32", seed), normal((groups, 4), "f32", seed + 1)
    return lambda: api.beam_select(logits, scores, count)


def forks(n, seed):
    """A fork of a table of more than 2^15 entries, a launch for the plan and one
    for each 64 layers, from the same state every time."""
    r = np.random.RandomState(seed)
    width = 2 ** 15 // n + 2
    caches, batch, past, table, slots = state([int(x) for x in r.randint(0, 400, n)], width, 8 * n, n, layers=66, kv_heads=1, seed=seed)
    parents = ints([int(x) for x in r.randint(-1, n, n)])
    saved = [t.clone() for t in (past, table, slots)]
    opened = [(c.open.clone(), c.open_scales.clone()) for c in caches[::13]]

    def call():
        for t, s in zip((past, table, slots), saved):
            t.copy_(s)
        for c, (codes, scales) in zip(caches[::13], opened):
            c.open.copy_(codes)
            c.open_scales.copy_(scales)
        batch.fork(parents, caches, room=70)
        return [t.clone() for t in (past, table, slots)] + [x.clone() for c in caches[::13] for x in (c.open, c.open_scales)]

    return call


def test_threads_on_one_stream(cuda):
    calls = [tree_of("f32", 4000, 16, 80), tree_of("bf16", 2500, 40, 84), beams(3, 20, 88), forks(520, 90), one_token(3000, 92)]
    want = [[t.clone() for t in call()] for call in calls]
    torch.cuda.synchronize()
    wrong, ready = [], threading.Barrier(len(calls))

    def work(i):
        try:
            torch.cuda.set_device(cuda)
            ready.wait()
            for n in range(40):
                got = calls[i]()
                if n % 4 == 3 and not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append((i, n))
        except Exception as e:  # a thread's failure is the test's
            wrong.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong
