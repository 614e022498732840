"""The norms' reciprocal root, to the last place: rows of small whole numbers,
with a one in them that shows the factor."""
import numpy as np
import pytest
import torch

from test_gpu_kv_cache import f64, ints, make_cache, step

pytestmark = pytest.mark.gpu


def rows(count, width):
    """Whole numbers under 64, a one in the first place."""
    x = torch.randint(-63, 64, (count, width), generator=torch.Generator().manual_seed(width)).float().cuda()
    x[:, 0] = 1.0
    return x


def check(got, x):
    """Half a last place of fp32, and 1/64 of one for the steps before the last
    rounding (a refined root is off by some 2^-40)."""
    want = 1 / np.sqrt(np.mean(f64(x) ** 2, axis=-1))
    place = 2.0 ** (np.floor(np.log2(want)) - 23)
    assert (np.abs(f64(got) - want) <= (0.5 + 1 / 64) * place).all()


@pytest.mark.parametrize("width", [4, 64, 256, 1024, 4096, 16384])
def test_add_norm(cuda, width):
    from q4rdna import api
    x = rows(500, width)
    one = torch.ones(width, device="cuda")
    _, n = api.add_norm(x, None, one, eps=0.0)
    check(n[:, 0], x)
    # the norm of y, added to zeros
    h, _ = api.add_norm(torch.zeros_like(x), x, None, post_weight=one, eps=0.0)
    check(h[:, 0], x)


@pytest.mark.parametrize("dim", [64, 128])
def test_the_norm_of_heads(cuda, dim):
    x = rows(600, dim).view(100, 6, dim)
    cache = make_cache(2, dim, 2, 1)
    k = torch.zeros((100, 2, dim), device="cuda")
    q = cache.append(step([0], [100], ints([[0, 1]])), k, k, q=x, q_norm=torch.ones(dim, device="cuda"), eps=0.0)
    check(q[:, :, 0], x)


def test_rows_whose_squares_pass_fp32_s_range(cuda):
    """Squares that overflow give zeros and rows of zeros NaN without eps, as the
    formula in fp32 does; small rows are normalised."""
    from q4rdna import api
    x = torch.ones((4, 64), device="cuda")
    x[0] *= 1e25
    x[1] *= 0
    x[2] *= 2.0 ** -60
    x[3] *= 2.0 ** 60
    one = torch.ones(64, device="cuda")
    cache, k = make_cache(1, 64, 1, 1), torch.zeros((4, 1, 64), device="cuda")
    for n in (api.add_norm(x, None, one, eps=0.0)[1],
              cache.append(step([0], [4], ints([[0]])), k, k, q=x[:, None], q_norm=one, eps=0.0)[:, 0]):
        assert (n[0] == 0).all() and torch.isnan(n[1]).all() and (n[2:] == 1).all()
    for n in (api.add_norm(x, None, one, eps=1e-6)[1],
              cache.append(step([0], [4], ints([[0]])), k, k, q=x[:, None], q_norm=one, eps=1e-6)[:, 0]):
        assert (n[0] == 0).all() and (n[1] == 0).all() and (n[3] == 1).all()


def test_rows_whose_squares_are_subnormal(cuda):
    from q4rdna import api
    x = torch.full((3, 64), 2.0 ** -70, device="cuda")
    x[1] *= -0.5
    x[2, 1:] = 0
    one = torch.ones(64, device="cuda")
    want = f64(x) / np.sqrt(np.mean(f64(x) ** 2, axis=-1, keepdims=True))  # powers of two
    cache, k = make_cache(1, 64, 1, 1), torch.zeros((3, 1, 64), device="cuda")
    for n in (api.add_norm(x, None, one, eps=0.0)[1], api.add_norm(torch.zeros_like(x), x, None, post_weight=one, eps=0.0)[0],
              cache.append(step([0], [3], ints([[0]])), k, k, q=x[:, None], q_norm=one, eps=0.0)[:, 0]):
        assert np.array_equal(f64(n), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,width", [(9, 64), (50, 264), (600, 1032), (40, 3000), (700, 5000), (5, 8192), (3, 16384)])
def test_aligned_and_unaligned_rows_give_the_same_bits(cuda, dtype, rows, width):
    """A row's factor does not depend on how many numbers a thread takes."""
    from q4rdna import api
    x, y = (torch.randn((rows, width), device="cuda").to(dtype) for _ in range(2))
    one = torch.ones(width, device="cuda")
    shifted = [torch.empty(rows * width + 1, dtype=dtype, device="cuda")[1:].view(rows, width).copy_(t) for t in (x, y)]
    assert shifted[0].data_ptr() % 16 != 0
    for a, b in zip(api.add_norm(x, y, one, post_weight=one), api.add_norm(*shifted, one, post_weight=one)):
        assert torch.equal(a, b)
