"""rotate: the norm of heads and the rotation by given positions."""
import numpy as np
import pytest
import torch

import layer_reference as R
from test_gpu_kv_attend import filled
from test_gpu_kv_cache import DTYPES, ROUND, f64, ints, normal, rotary_table, step

pytestmark = pytest.mark.gpu


def reference(x, positions, cos, sin, interleaved, weight, eps):
    x = x if weight is None else R.rms(x, weight, eps)
    return np.stack([R.rotate(x[n], p, cos, sin, interleaved) for n, p in enumerate(positions)])


@pytest.mark.parametrize("dim,rotary", [(64, 64), (64, 24), (128, 128), (128, 64), (128, 8)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("tokens,q_heads,k_heads", [(1, 8, 2), (7, 5, 5), (300, 12, 4), (3, 0, 3), (33, 7, 0)])
def test_against_the_definition(cuda, dim, rotary, interleaved, dtype, tokens, q_heads, k_heads):
    """Half a last place of the output, and four roundings of 2^-24 of the
    pair's numbers: the norm's factor and its product, the weight's, the turn's
    two products and their sum."""
    from q4rdna import api
    cos, sin = rotary_table(500, rotary)
    positions = np.random.RandomState(tokens).randint(0, 500, tokens)
    positions[0] = 499
    q = normal((tokens, q_heads, dim), dtype, 1, 2.0) if q_heads else None
    k = normal((tokens, k_heads, dim), dtype, 2) if k_heads else None
    qw, kw = (1 + 0.2 * normal((dim,), "f32", s) for s in (3, 4))
    for norm in (False, True):
        got = api.rotate(q, k, ints(positions.tolist()), cos, sin, interleaved=interleaved, q_norm=qw if norm and q_heads else None,
                         k_norm=kw if norm and k_heads else None, eps=1e-5)
        for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
            if x is None:
                assert y is None
                continue
            want = reference(f64(x), positions, f64(cos), f64(sin), interleaved, f64(w) if norm else None, 1e-5)
            size = np.abs(want) + np.abs(R.rms(f64(x), f64(w), 1e-5) if norm else f64(x)).max(-1, keepdims=True)
            assert y.dtype == x.dtype and (np.abs(f64(y) - want) <= ROUND[dtype] * np.abs(want) + 6 * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("interleaved", [False, True])
def test_the_bits_of_append(cuda, dtype, interleaved):
    """q as append returns it, and k as the cache holds it: its codes are the same."""
    from q4rdna import api
    past, count, dim = 37, 90, 128
    cache, table, slots = filled(2, dim, [past + count], 1)
    other, _, _ = filled(2, dim, [past + count], 1)
    q, k, v = (normal((count, h, dim), dtype, s) for s, h in ((5, 6), (6, 2), (7, 2)))
    qw, kw = (1 + 0.2 * normal((dim,), "f32", s) for s in (8, 9))
    cos, sin = rotary_table(200, 96)
    batch = step([past], [count], table, slots)
    want = cache.append(batch, k, v, q=q, cos=cos, sin=sin, interleaved=interleaved, q_norm=qw, k_norm=kw)
    got, turned = api.rotate(q, k, ints(list(range(past, past + count))), cos, sin, interleaved=interleaved, q_norm=qw, k_norm=kw)
    assert torch.equal(got, want)
    if dtype == "f32":  # (a 16-bit k is rounded before it is coded)
        other.append(batch, turned, v)
        assert torch.equal(cache.pages, other.pages)  # (an open block's bytes behind its last token are not defined)
        assert all(torch.equal(a, b) for a, b in zip(cache.read(step([0], [past + count], table, slots), past + count),
                                                     other.read(step([0], [past + count], table, slots), past + count)))


def test_positions_outside_the_tables(cuda):
    from q4rdna import api
    cos, sin = rotary_table(10, 32)
    q, k = normal((6, 3, 64), "f32", 10), normal((6, 1, 64), "f32", 11)
    at = [0, 9, 10, -1, 2 ** 31 - 1, 5]
    out = api.rotate(q, k, ints(at), cos, sin)
    good = api.rotate(q[[0, 1, 5]], k[[0, 1, 5]], ints([0, 9, 5]), cos, sin)
    for x, y in zip(out, good):
        assert torch.equal(x[[0, 1, 5]], y) and torch.isnan(x[2:5]).all()


def test_in_place_strides_and_no_rotation(cuda):
    from q4rdna import api
    cos, sin = rotary_table(50, 64)
    at = ints([3, 49, 0, 7, 7])
    for dtype, offset in (("f32", 1), ("bf16", 3), ("f16", 4)):
        q, k = normal((5, 4, 64), dtype, 12), normal((5, 2, 64), dtype, 13)
        want = api.rotate(q, k, at, cos, sin)
        both = torch.zeros(5 * 6 * 72 + offset, dtype=q.dtype, device="cuda")[offset:].view(6, 5, 72)[..., :64].transpose(0, 1)
        both[:, :4].copy_(q)
        both[:, 4:].copy_(k)
        got = api.rotate(both[:, :4], both[:, 4:], at, cos, sin, q_out=both[:, :4], k_out=both[:, 4:])
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0].data_ptr() == both.data_ptr()
    w = torch.ones(64, device="cuda")
    plain = api.rotate(q, None, None, q_norm=w)[0]
    assert torch.equal(plain, api.rotate(q, None, ints([0] * 5), torch.ones((1, 4), device="cuda"), torch.zeros((1, 4), device="cuda"), q_norm=w)[0])
    base = normal((2000,), "f32", 14)
    slide = base.as_strided((5, 4, 64), (1, 64, 1))
    assert torch.equal(api.rotate(slide, None, at, cos, sin)[0], api.rotate(slide.contiguous(), None, at, cos, sin)[0])
    with pytest.raises(ValueError):
        api.rotate(q, None, at, cos, sin, q_out=q[:1].expand(5, 4, 64))
    empty = api.rotate(q[:0], k[:0], at[:0].contiguous(), cos, sin)
    assert empty[0].shape == (0, 4, 64) and empty[1].shape == (0, 2, 64)


def test_refusals(cuda):
    from q4rdna import api
    cos, sin = rotary_table(10, 32)
    q, at = normal((3, 2, 64), "f32", 15), ints([0, 1, 2])
    for call in (lambda: api.rotate(q, q.half(), at, cos, sin), lambda: api.rotate(q, q[:2], at, cos, sin),
                 lambda: api.rotate(q, None, at.long(), cos, sin), lambda: api.rotate(q, None, at[:2], cos, sin),
                 lambda: api.rotate(q, None, at, cos), lambda: api.rotate(q, None, at, None, sin), lambda: api.rotate(q, None, None, cos, sin),
                 lambda: api.rotate(q, None, at, cos, sin, k_norm=cos[0]), lambda: api.rotate(q, None, at, cos, sin, q_norm=cos[0]),
                 lambda: api.rotate(q.clone().requires_grad_(), None, at, cos, sin), lambda: api.rotate(q.double(), None, at, cos, sin)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(api.Q4RdnaError, match="head_dim"):
        api.rotate(normal((3, 2, 96), "f32", 16), None, at, cos, sin)
    with pytest.raises(api.Q4RdnaError, match="cos"):
        api.rotate(q, None, at, cos[:0], sin[:0])


def test_streams_and_replays(cuda):
    from q4rdna import api
    cos, sin = rotary_table(300, 128)
    q, k, at = normal((40, 8, 128), "bf16", 17), normal((40, 2, 128), "bf16", 18), ints(list(range(40)))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = api.rotate(q, k, at, cos, sin, stream=stream.cuda_stream)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, api.rotate(q, k, at, cos, sin)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = api.rotate(q, k, at, cos, sin)
    for shift in (0, 100, 260):
        at.copy_(ints([(7 * i + shift) % 300 for i in range(40)]))
        q.copy_(normal((40, 8, 128), "bf16", 19 + shift))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, api.rotate(q, k, at, cos, sin)))
