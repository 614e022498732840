"""kv_attend with tables far wider than the sequences are long.  The width is
what bounds the lengths when a call is made, so the same prompts go to the other
of the two kernels here, and many sequences are dealt as if they could be long.
The columns behind a sequence hold numbers that are no pages."""
import os
import subprocess
import sys

import pytest
import torch

import test_gpu_kv_attend as narrow
from test_gpu_kv_cache import normal, step

pytestmark = pytest.mark.gpu

WIDTH = 5000


def widen(table):
    wide = torch.full((table.shape[0], WIDTH), -7, dtype=torch.int32, device=table.device)
    wide[:, :table.shape[1]] = table
    return wide


@pytest.fixture
def wide_tables(monkeypatch):
    def wide_step(past, counts, table, *args, **kwargs):
        return step(past, counts, widen(table), *args, **kwargs)
    monkeypatch.setattr(narrow, "step", wide_step)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [1, 40])
def test_long_sequences_are_split_and_joined_alike(cuda, wide_tables, dtype, tokens):
    narrow.test_long_sequences_are_split_and_joined_alike(cuda, dtype, tokens)


@pytest.mark.parametrize("tokens", [1, 50])
def test_peaked_and_shifted_scores(cuda, wide_tables, tokens):
    narrow.test_peaked_and_shifted_scores(cuda, tokens)


@pytest.mark.parametrize("tokens", [1, 60])
def test_nan_stays_where_it_is_seen(cuda, wide_tables, tokens):
    narrow.test_nan_stays_where_it_is_seen(cuda, tokens)


@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("dtype,offset", [("f32", 1), ("bf16", 3), ("f16", 8)])
def test_strided_rows(cuda, wide_tables, tokens, dtype, offset):
    narrow.test_strided_rows(cuda, tokens, dtype, offset)


@pytest.mark.parametrize("tokens", [1, 48])
def test_bad_pages_give_nan_and_bad_sequences_are_skipped(cuda, wide_tables, tokens):
    narrow.test_bad_pages_give_nan_and_bad_sequences_are_skipped(cuda, tokens)


@pytest.mark.parametrize("kv_heads,group,dim,dtype", [(2, 4, 128, "f32"), (1, 3, 64, "f16"), (1, 1, 128, "bf16")])
@pytest.mark.parametrize("past,counts,window", [([0], [200], 0), ([100, 0, 3], [100, 1, 140], 64), ([250], [33], 0),
                                                ([5, 0], [96, 40], 7)])
def test_prompts(cuda, wide_tables, kv_heads, group, dim, dtype, past, counts, window):
    narrow.test_prompts(cuda, kv_heads, group, dim, dtype, past, counts, window)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [[8], [9], [16], [17], [32], [33], [8, 9, 1], [16, 0, 17, 2], [33, 32, 5, 1]])
@pytest.mark.parametrize("wide", [False, True])
def test_rows_around_the_kernels_limits(cuda, dtype, tokens, wide):
    """32, 64 and 128 rows a kv head and four more, alone and next to others."""
    past = [130 + 61 * i for i in range(len(tokens))]
    lengths = [p + t for p, t in zip(past, tokens)]
    cache, table, slots = narrow.filled(2, 64, lengths, 31)
    q = normal((sum(tokens), 8, 64), dtype, 32, 2.0)
    out, lse = cache.attend(step(past, tokens, widen(table) if wide else table, slots), q, lse=True)
    narrow.check(cache, table, slots, past, tokens, q, out, dtype, lse)
    assert cache.faults() == 0


@pytest.mark.parametrize("length", [256, 250])
@pytest.mark.parametrize("group", [4, 8])
def test_no_weight_loses_a_digit(cuda, length, group):
    """256 single tokens with their own queries behind one sequence's blocks, a
    million and more weights: a carry between the digits of one that gets lost
    is an error of 2^-6 or 2^-14 of it, far above the bound."""
    sequences = 256
    cache, table, slots = narrow.filled(1, 64, [length], 35)
    past = [length - 1] * sequences
    q = normal((sequences, group, 64), "f32", 36, 2.0)
    same = table.expand(sequences, -1).contiguous()
    out, lse = cache.attend(step(past, [1] * sequences, same, slots * sequences), q, lse=True)
    narrow.check(cache, same, slots * sequences, past, [1] * sequences, q, out, "f32", lse)


@pytest.mark.parametrize("sequences", [255, 256, 257, 300])
def test_sequences_around_the_deal_s_limit(cuda, sequences):
    """Ragged single tokens, one of them behind a long sequence."""
    lengths = [1 + 37 * i % 150 for i in range(sequences)]
    lengths[sequences // 2] = 3000
    cache, table, slots = narrow.filled(1, 64, lengths, 33)
    past = [n - 1 for n in lengths]
    q = normal((sequences, 2, 64), "f32", 34)
    out, lse = cache.attend(step(past, [1] * sequences, table, slots), q, lse=True)
    narrow.check(cache, table, slots, past, [1] * sequences, q, out, "f32", lse)


@pytest.mark.parametrize("kv_heads,sequences", [(1, 3), (32, 150)])
def test_without_a_bound_on_the_tokens(cuda, kv_heads, sequences):
    """max_tokens left out: the step's tokens bound every sequence's.  With 150
    sequences of 32 kv heads the row groups are too many to be split."""
    from q4rdna import api
    past, counts = [1100, 0] + [1 + 5 * i % 70 for i in range(sequences - 2)], [5, 90] + [1] * (sequences - 2)
    cache, table, slots = narrow.filled(kv_heads, 64, [p + c for p, c in zip(past, counts)], 37)
    q = normal((sum(counts), kv_heads, 64), "f32", 38)
    ends = torch.tensor([0] + counts, device="cuda").cumsum(0).int()
    past_d, slots_d = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (past, slots))
    out, lse = cache.attend(api.KVBatch(past_d, table, ends, slots_d), q, lse=True)
    assert cache.faults() == 0
    narrow.check(cache, table, slots, past, counts, q, out, "f32", lse)


FIRST_CALL_CAPTURED = """
import sys
sys.path[:0] = sys.argv[1:3]
import pytest, torch
import test_gpu_kv_attend as narrow
from q4rdna._lib import Q4RdnaError
cache, table, slots = narrow.filled(1, 64, [3000], 39)
batch = narrow.step([2999], [1], table, slots)
q = narrow.normal((1, 2, 64), "f32", 40)
out, count = torch.zeros_like(q), torch.zeros(1, device="cuda")
stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=stream):
    count += 1
    with pytest.raises(Q4RdnaError, match="captured"):
        cache.attend(batch, q, out=out)
graph.replay()
torch.cuda.synchronize()
assert count.item() == 1 and (out == 0).all()
want = cache.attend(batch, q)
with torch.cuda.stream(stream):
    cache.attend(batch, q, out=out)
torch.cuda.synchronize()
assert torch.equal(out, want)
out.zero_()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=stream):
    cache.attend(batch, q, out=out)
for _ in range(3):
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    out.zero_()
print("captured")
"""


def test_a_first_call_under_capture_is_refused(cuda):
    """In a fresh process, where no stream has scratch: the call that needs some
    is refused under capture, the capture stays whole, and after one call outside
    it the same call is captured."""
    tests = os.path.dirname(os.path.abspath(__file__))
    run = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED, tests, os.path.dirname(tests)], capture_output=True,
                         text=True, timeout=100)
    assert run.returncode == 0 and "captured" in run.stdout, run.stderr[-2000:]
