"""beam_select against its definition in 64 bits."""
import numpy as np
import pytest
import torch

import branch_reference as B
from test_gpu_kv_cache import DTYPES, f64, normal

pytestmark = pytest.mark.gpu


def check(logits, scores, count, got=None):
    """Rows and tokens are equal, scores off by the rounding to fp32, 2^-24, and
    by the log-sum-exp: of its fp32 exponentials each is off by 2^-23 (the
    instruction) and 2^-24 of its argument, weighted by itself (x e^-x <= 0.37),
    and up to 32 of them are added in fp32: under 2^-20 in all."""
    from q4rdna import api
    scores_out, rows, tokens = api.beam_select(logits, scores, count) if got is None else got
    want, want_rows, want_tokens = B.beam_select(f64(logits), None if scores is None else f64(scores), count)
    assert rows.dtype == tokens.dtype == torch.int32 and scores_out.dtype == torch.float32
    assert np.array_equal(rows.cpu().numpy(), want_rows) and np.array_equal(tokens.cpu().numpy(), want_tokens)
    s = f64(scores_out)
    assert np.array_equal(np.isneginf(s), np.isneginf(want))
    finite = np.isfinite(want)
    assert (np.abs(s - want)[finite] <= 2.0 ** -24 * np.abs(want[finite]) + 2.0 ** -20).all()
    return scores_out, rows, tokens


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("groups,beams,vocab,count", [
    (1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 4, 12), (1, 1, 1023, 1), (3, 1, 1025, 7), (1, 4, 50257, 8), (2, 5, 32003, 10), (1, 2, 151936, 128),
    (7, 2, 777, 64), (1, 3, 2049, 65), (1, 32, 4001, 64), (40, 4, 999, 9), (1, 1, 200001, 100)])
def test_against_the_definition(cuda, dtype, groups, beams, vocab, count):
    logits = normal((groups, beams, vocab), dtype, vocab + count, 3.0)
    scores = -20 * torch.rand((groups, beams), generator=torch.Generator().manual_seed(count)).cuda()
    first = check(logits, scores, count)
    from q4rdna import api
    assert all(torch.equal(a, b) for a, b in zip(first, api.beam_select(logits, scores, count)))
    check(logits, None, count) if groups * beams == 1 else None


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [40, 2047, 40000])
@pytest.mark.parametrize("count", [1, 6, 70])
def test_equal_logits_go_by_token(cuda, dtype, vocab, count):
    """All equal, few values, rows that are sorted either way, both zeros, one
    value at many places."""
    x = torch.zeros((5, 3, vocab))
    g = torch.Generator().manual_seed(vocab)
    x[1] = torch.randint(0, 3, (3, vocab), generator=g).float()
    x[2] = (torch.arange(vocab) // 7 - vocab // 14).float() / 64
    x[3] = -x[2]
    x[4] = torch.where(torch.rand((3, vocab), generator=g) < 0.5, 0.0, -0.0)
    scores = torch.tensor([[0.0, -1.0, -2.5]]).expand(5, 3).contiguous().cuda()
    check(x.to(DTYPES[dtype]).cuda(), scores, count)


@pytest.mark.parametrize("vocab", [10, 9000])
def test_equal_beams_go_by_row(cuda, vocab):
    """Beams that are copies of each other, as in a first step: all candidates
    are tied in pairs, also where a row's chunks lie at other addresses."""
    row = normal((vocab,), "f32", 1)
    logits = torch.stack([row, row, row])[None]
    check(logits, torch.zeros((1, 3), device="cuda"), 9)
    big = torch.zeros((1, 3, vocab + 3), device="cuda")
    big[:, :, 1:vocab + 1] = logits
    check(big[:, :, 1:vocab + 1], torch.zeros((1, 3), device="cuda"), 9)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_beams_without_a_continuation(cuda, dtype):
    """Scores that are not finite, rows of -inf, with NaN, with +inf; tokens at
    -inf; too few continuations, so that the dead ones come in, lowest first."""
    inf, nan = float("inf"), float("nan")
    for vocab, count in ((6, 30), (3000, 12), (3000, 128), (6, 1)):
        logits = normal((6, 5, vocab), dtype, 7, 2.0)
        scores = -torch.rand((6, 5), generator=torch.Generator().manual_seed(8)).cuda()
        scores[0, 1:] = -inf
        scores[1, 0], scores[1, 2], scores[1, 3] = nan, inf, -inf
        logits[2, 1] = -inf
        logits[2, 0, vocab // 2] = nan
        logits[2, 2, 1] = inf
        logits[3] = -inf
        logits[4, :, 2:] = -inf
        logits[5, 1, 3:] = -inf
        scores[5, 2:] = -inf
        check(logits, scores, count)


def test_large_numbers(cuda):
    """Logits at the type's ends, and a row whose exponentials all but one vanish."""
    for dtype in DTYPES:
        top = torch.finfo(DTYPES[dtype]).max
        logits = normal((3, 2, 500), dtype, 9)
        logits[0, 0, 77], logits[0, 1, 3] = top, -top
        logits[1] *= 1000
        logits[2] += 60000 if dtype == "f16" else 1e6
        check(logits, torch.tensor([[-1.0, -3e38], [-5.0, -6.0], [0.0, 0.0]], device="cuda"), 4)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_strides(cuda, dtype):
    """Rows at odd places, beams before groups, one row for all beams."""
    big = normal((3, 4, 5007), dtype, 10)
    scores = torch.rand((3, 4), generator=torch.Generator().manual_seed(11)).cuda()
    check(big[:, :, 1:5006], scores, 5)
    check(big.transpose(0, 1)[..., 3:4000], scores.t().contiguous(), 5)
    check(big[:1, :1].expand(3, 4, 5007), scores, 5)


def test_given_outputs_streams_and_replays(cuda):
    """Several replays between other calls on the stream that share its scratch."""
    from q4rdna import api
    logits, scores = normal((2, 3, 30011), "bf16", 12, 3.0), torch.zeros((2, 3), device="cuda")
    out = (torch.empty((2, 6), device="cuda"), torch.empty((2, 6), dtype=torch.int32, device="cuda"),
           torch.empty((2, 6), dtype=torch.int32, device="cuda"))
    got = api.beam_select(logits, scores, 6, out=out)
    assert all(a is b for a, b in zip(got, out))
    check(logits, scores, 6, got)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        api.beam_select(logits, scores, 6)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = api.beam_select(logits, scores, 6)
    for seed in (13, 14, 15):
        logits.copy_(normal((2, 3, 30011), "bf16", seed, 3.0))
        scores.copy_(normal((2, 3), "f32", seed))
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            graph.replay()
            other = api.beam_select(normal((1, 8, 5000), "f32", seed), None, 16)
        stream.synchronize()
        check(logits, scores, 6, got)
        check(normal((1, 8, 5000), "f32", seed), None, 16, other)
    side = api.beam_select(logits, scores, 6, stream=stream.cuda_stream)
    stream.synchronize()
    check(logits, scores, 6, side)
    fresh = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    big = normal((8, 8, 30011), "f32", 16)
    with torch.cuda.graph(graph, stream=fresh):  # a first call under capture is refused, the capture whole
        with pytest.raises(api.Q4RdnaError, match="captured"):
            api.beam_select(big, None, 16, out=(torch.empty((8, 16), device="cuda"), torch.empty((8, 16), dtype=torch.int32, device="cuda"),
                                                torch.empty((8, 16), dtype=torch.int32, device="cuda")))
        scores.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert (scores == 0).all()


def test_refusals(cuda):
    from q4rdna import api
    x, s = normal((2, 3, 50), "f32", 17), torch.zeros((2, 3), device="cuda")
    for call in (lambda: api.beam_select(x[0], s, 1), lambda: api.beam_select(x, s[0], 1), lambda: api.beam_select(x, s.half(), 1),
                 lambda: api.beam_select(x, s, 0), lambda: api.beam_select(x, s, 129), lambda: api.beam_select(x[..., :2], s, 7),
                 lambda: api.beam_select(x[..., ::2], s, 1), lambda: api.beam_select(x.double(), s, 1),
                 lambda: api.beam_select(x.clone().requires_grad_(), s, 1), lambda: api.beam_select(x, s.cpu(), 1),
                 lambda: api.beam_select(x, s, 2, out=(s, s, s)), lambda: api.beam_select(x, s, 2, out=(s[:, :2].contiguous(),))):
        with pytest.raises(ValueError):
            call()
    empty = api.beam_select(x[:0], s[:0], 2)
    assert [t.shape for t in empty] == [(0, 2)] * 3


@pytest.mark.parametrize("beams", [1, 5, 64])
def test_scores_in_place(cuda, beams):
    """A search's step: the new scores where the old ones were."""
    from q4rdna import api
    logits, scores = normal((7, beams, 9001), "f32", 18, 2.0), normal((7, beams), "f32", 19)
    scores[3, 0] = float("-inf")
    want = api.beam_select(logits, scores, beams)
    got = api.beam_select(logits, scores, beams, out=(scores, torch.empty_like(want[1]), torch.empty_like(want[2])))
    assert got[0] is scores and all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("beams,vocab,count", [(32, 392, 64), (256, 150, 128), (200, 300, 33), (17, 5000, 128), (256, 4097, 16)])
@pytest.mark.parametrize("spread", [0.0, 0.5, 30.0])
def test_beams_far_apart(cuda, beams, vocab, count, spread):
    """One beam's best are all before the next one's, rising and falling, and
    all beams alike: more candidates than are ordered at a time reach any first
    bound."""
    logits = normal((3, beams, vocab), "f32", beams + count, 2.0)
    logits[2] = logits[2, :1]
    scores = spread * torch.arange(beams, dtype=torch.float32).expand(3, beams).clone()
    scores[1] = -scores[1]
    scores[2] = spread * torch.randn(beams, generator=torch.Generator().manual_seed(count))
    check(logits, scores.cuda(), count)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("count", [1, 33, 128])
def test_masked_vocabularies(cuda, dtype, count):
    """Few tokens allowed, the others -inf: those come behind, by token."""
    logits = normal((4, 5, 30011), dtype, count, 2.0)
    g = torch.Generator().manual_seed(count)
    for i, share in enumerate((0.001, 0.00004, 0.2, 0.0)):
        allowed = torch.rand((5, 30011), generator=g) < share
        allowed[0, 12345] = True
        logits[i].masked_fill_(~allowed.cuda(), float("-inf"))
    check(logits, normal((4, 5), "f32", count + 1), count)
