"""The open block's tokens have scales of their own: a loud one takes nothing
from the rows that do not see it, nor from those that hardly weigh it."""
import math

import pytest

from test_gpu_kv_cache import ints, step
from test_gpu_kv_spread import check_rows, spread_cache, toward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("spread", [2.0 ** 20, 2.0 ** 33, 1e24])
@pytest.mark.parametrize("loud", [186, 150])
@pytest.mark.parametrize("tokens", [4, 60, 100])
@pytest.mark.parametrize("hidden", [False, True])
def test_a_loud_token_of_the_open_block(cuda, dim, dtype, spread, loud, tokens, hidden):
    """Token 150 of 187 or the last one, for few rows and for many."""
    length = 187
    cache, row, side = spread_cache(dim, length, slice(loud, loud + 1), spread, math.log(spread) + (35 if hidden else 0), 3)
    past = length - tokens
    q = toward(side, tokens, 2, dtype, 9)
    out = cache.attend(step([past], [tokens], ints([row]), [1]), q)
    check_rows(cache, row, 1, past, q, out, dtype)


@pytest.mark.parametrize("tokens", [4, 60, 100])
def test_loud_tokens_outside_the_window(cuda, tokens):
    length, window = 250, 9
    cache, row, side = spread_cache(64, length, slice(192, 200), 1e12, 5.0, 4)
    past = length - tokens
    q = toward(side, tokens, 2, "f32", 10)
    out = cache.attend(step([past], [tokens], ints([row]), [1]), q, window=window)
    check_rows(cache, row, 1, past, q, out, "f32", window)
