"""`stream=`: outputs that a call allocates come from that stream's memory, so
they overwrite nothing that the current stream still reads."""
import pytest
import torch

from test_gpu_kv_attend import filled
from test_gpu_kv_cache import normal, step

pytestmark = pytest.mark.gpu

TOKENS = 4096  # outputs of a megabyte and more, which the allocator keeps apart


def freed(shape, dtype):
    """The address that the current stream's next allocation of this size gets."""
    x = torch.empty(shape, dtype=dtype, device="cuda")
    y = torch.empty(shape, dtype=dtype, device="cuda")
    at = {x.data_ptr(), y.data_ptr()}
    del x, y
    return at


@pytest.mark.parametrize("current", [False, True])
def test_outputs_on_a_stream_of_their_own(cuda, current):
    from q4rdna import api
    cache, table, slots = filled(1, 64, [TOKENS], 60)
    batch = step([0], [TOKENS], table, slots)
    q, k = normal((TOKENS, 4, 64), "f32", 61), normal((TOKENS, 1, 64), "f32", 62)
    x, one = q.view(TOKENS, 256), torch.ones(256, device="cuda")
    weight = torch.randn((256, 256), device="cuda")
    side = torch.cuda.Stream()
    handle = torch.cuda.current_stream().cuda_stream if current else side.cuda_stream
    calls = [lambda **s: cache.attend(batch, q, **s), lambda **s: cache.append(batch, k, k, q=q, **s),
             lambda **s: cache.read(batch, TOKENS, dtype=torch.float32, **s), lambda **s: api.add_norm(x, x, one, **s),
             lambda **s: api.pack(weight, **s)]
    tiles = api.pack(weight)
    w = api.QWeight.from_tiles(tiles, 256, 256)
    calls += [lambda **s: api.dequantize(w, **s)]
    for i, call in enumerate(calls):
        want = call()
        torch.cuda.synchronize()
        want = [t.clone() for t in (want if isinstance(want, tuple) else (want,))]
        taken = set().union(*(freed(t.shape, t.dtype) for t in want))
        side.wait_stream(torch.cuda.current_stream())
        got = call(stream=handle)
        got = got if isinstance(got, tuple) else (got,)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        mine = {t.data_ptr() for t in got}
        assert bool(mine & taken) == current, i
        assert torch.cuda.current_stream().cuda_stream != side.cuda_stream


def test_vectors_on_a_stream_of_their_own(cuda):
    from q4rdna import api
    w = api.QWeight.from_tiles(api.pack(torch.randn((2048, 256), device="cuda")), 2048, 256)
    x, add = torch.randn(256, device="cuda"), torch.randn(2048, device="cuda")
    side = torch.cuda.Stream()
    for call in (lambda **s: api.mul_mat(w, x, **s), lambda **s: api.mul_mat_add(w, x, add, **s), lambda **s: api.mul_mat_glu(w, w, x, **s)):
        want = call().clone()
        with torch.cuda.stream(side):
            call()  # the stream's scratch
        torch.cuda.synchronize()
        taken = freed(want.shape, want.dtype)
        got = call(stream=side.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and got.data_ptr() not in taken
