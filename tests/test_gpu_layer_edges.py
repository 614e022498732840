"""Small things at the edges of the decoder-layer calls."""
import pytest
import torch

from test_gpu_kv_attend import check, filled
from test_gpu_kv_cache import ints, normal, step

pytestmark = pytest.mark.gpu


def test_a_refused_sequence_counts_once(cuda):
    """In a step that both attention kernels take part in, and in each of them alone."""
    for past, counts in (([300, 0, 20], [1, 150, 1]), ([300, 60], [1, 1]), ([0, 10], [150, 90]), ([5], [150])):
        cache, table, slots = filled(1, 64, [p + c for p, c in zip(past, counts)], 70)
        q = normal((sum(counts), 4, 64), "bf16", 71)
        for bad in range(len(past)):
            for other, at in (([-5 if i == bad else p for i, p in enumerate(past)], slots),
                              (past, [99 if i == bad else s for i, s in enumerate(slots)])):
                before = cache.faults()
                cache.attend(step(other, counts, table, at), q)
                assert cache.faults() == before + 1


def test_one_row_in_place_under_another_stride(cuda):
    """A single row has no stride to agree on."""
    from q4rdna import api
    base, y, w = normal((4, 300), "f32", 72), normal((1, 100), "f32", 73), torch.ones(100, device="cuda")
    x = base[1:2, :100]
    want = api.add_norm(x, y, w)
    h = base[1, :100].unsqueeze(0)
    assert h.data_ptr() == x.data_ptr() and h.stride() != x.stride()
    got = api.add_norm(x, y, w, h=h)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(x, want[0])


@pytest.mark.parametrize("shape", [(3, 0), (0, 0), (0, 64)])
def test_rows_without_numbers(cuda, shape):
    from q4rdna import api
    x, one = torch.empty(shape, device="cuda"), torch.ones(shape[1], device="cuda")
    for y, gate in ((None, None), (torch.empty(shape, device="cuda"), None), (torch.empty(shape, device="cuda"), one)):
        h, n = api.add_norm(x, y, one, gate=gate)
        assert h.shape == n.shape == shape


@pytest.mark.parametrize("tokens,window", [(16, 100), (32, 7), (9, 1000)])
def test_a_window_bounds_the_blocks_without_max_tokens(cuda, tokens, window):
    """One sequence under a table far wider than it is long: the step's tokens
    bound its own as max_tokens does, and both calls take the same path."""
    from q4rdna import api
    length = 1300
    cache, table, slots = filled(8, 64, [length], 74)
    wide = torch.full((1, 5000), -7, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    past, cu = ints([length - tokens]), ints([0, tokens])
    q = normal((tokens, 32, 64), "f32", 75)
    want = cache.attend(api.KVBatch(past, wide, cu, ints(slots), max_tokens=tokens), q, window=window)
    got = cache.attend(api.KVBatch(past, wide, cu, ints(slots)), q, window=window)
    check(cache, wide, slots, [length - tokens], [tokens], q, got, "f32", window=window)
    assert torch.equal(got, want)


def test_more_rows_than_one_launch_holds(cuda):
    """2^26 and a few rows of 64 threads are over 2^32 threads."""
    from q4rdna import api
    rows = 2 ** 26 + 70
    x = torch.randint(-3, 4, (rows, 1), device="cuda", generator=torch.Generator("cuda").manual_seed(80)).half()
    y = torch.ones_like(x)
    h, n = api.add_norm(x, y, torch.ones(1, device="cuda"), scale=0.5, eps=0.25)
    assert torch.equal(h, x + 0.5)
    # n = h / sqrt(h^2 + 1/4): one rounding to fp16, and fp32's before it
    at = torch.cat([torch.arange(1000), torch.arange(rows - 1000, rows), torch.arange(2 ** 26 - 500, 2 ** 26 + 70)]).cuda()
    want = h[at].double() / (h[at].double() ** 2 + 0.25).sqrt()
    assert ((n[at].double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -20).all()
    assert (n.float() - h.float() / (h.float() ** 2 + 0.25).sqrt()).abs().max() <= 2.0 ** -10


def test_inputs_that_require_gradients_are_refused(cuda):
    """The calls have no backward: where torch would record one they say so."""
    from q4rdna import api
    cache, table, slots = filled(2, 64, [70], 76)
    batch = step([69], [1], table, slots)
    q, k = normal((1, 4, 64), "f32", 77), normal((1, 2, 64), "f32", 78)
    w, x = torch.ones(64, device="cuda"), normal((3, 64), "f32", 79)
    wants = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = [lambda: cache.attend(batch, wants(q)), lambda: cache.append(batch, wants(k), k), lambda: cache.append(batch, k, wants(k)),
             lambda: cache.append(batch, k, k, q=wants(q)), lambda: cache.append(batch, k, k, q=q, q_norm=wants(w)),
             lambda: cache.append(batch, k, k, k_norm=wants(w)),
             lambda: api.add_norm(wants(x), x, w), lambda: api.add_norm(x, wants(x), w), lambda: api.add_norm(x, x, wants(w)),
             lambda: api.add_norm(x, x, w, post_weight=wants(w)), lambda: api.add_norm(x, x, w, gate=wants(w))]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            call()
        with torch.inference_mode():
            call()
