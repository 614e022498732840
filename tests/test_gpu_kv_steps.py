"""The cache after many steps of any size, with norm, rotation and tokens taken
back, holds the bytes of one step with the tokens that are left."""
import random

import pytest
import torch

from test_gpu_kv_cache import ints, make_cache, normal, rotary_table, step

pytestmark = pytest.mark.gpu

WIDTH = 9  # blocks a sequence may have


def same_bytes(a, b, table, lengths):
    whole = step([0] * len(lengths), lengths, table)
    for x, y in zip(a.read(whole, sum(lengths)), b.read(whole, sum(lengths))):
        assert torch.equal(x, y)
    for i, n in enumerate(lengths):
        full = table[i, :n // 64].long()
        assert torch.equal(a.pages[full], b.pages[full]) and torch.equal(a.scales[full], b.scales[full])


@pytest.mark.parametrize("dim,kv_heads,rotary", [(64, 5, 32), (128, 2, 128), (128, 5, 0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("back", [False, True])
def test_any_steps_leave_the_same_bytes(cuda, dim, kv_heads, rotary, dtype, interleaved, back):
    """`back`: now and then tokens are taken back, to no less than the block
    before the last that the sequence ever reached."""
    rng = random.Random(dim + rotary + interleaved)
    extra = {"k_norm": torch.rand(dim, device="cuda") + 0.5, "interleaved": interleaved}
    if rotary:
        extra["cos"], extra["sin"] = rotary_table(WIDTH * 64, rotary)
    for seed in range(8):
        sequences = 3
        table = torch.randperm(sequences * WIDTH, generator=torch.Generator().manual_seed(seed)).int().view(sequences, WIDTH).cuda()
        cache, once = (make_cache(kv_heads, dim, sequences * WIDTH, sequences, seed) for _ in range(2))
        kept = [[normal((0, kv_heads, dim), dtype, 1) for _ in range(2)] for _ in range(sequences)]
        reached = [0] * sequences
        for turn in range(10):
            past, counts = [], []
            for i in range(sequences):
                n = kept[i][0].shape[0]
                if back and rng.random() < 0.4:
                    n = rng.randint(min(n, max(0, 64 * (reached[i] // 64 - 1))), n)
                    kept[i] = [x[:n] for x in kept[i]]
                past.append(n)
                counts.append(min(rng.choice([0, 1, 1, 2, 5, 17, 63, 64, 65, 130, 200]), WIDTH * 64 - n))
                reached[i] = max(reached[i], n + counts[i])
            if sum(counts) == 0:
                continue
            k, v = (normal((sum(counts), kv_heads, dim), dtype, 100 * seed + 2 * turn + which) for which in (0, 1))
            cache.append(step(past, counts, table), k, v, **extra)
            for i, (a, b) in enumerate(zip(k.split(counts), v.split(counts))):
                kept[i] = [torch.cat([kept[i][0], a]), torch.cat([kept[i][1], b])]
        lengths = [x[0].shape[0] for x in kept]
        once.append(step([0] * sequences, lengths, table), torch.cat([x[0] for x in kept]), torch.cat([x[1] for x in kept]), **extra)
        assert cache.faults() == 0 and once.faults() == 0
        same_bytes(cache, once, table, lengths)


def test_a_token_s_place_in_its_step_does_not_matter_to_q(cuda):
    """q's norm and rotation, in one step and token by token."""
    tokens, heads, dim = 70, 6, 128
    q = normal((tokens, heads, dim), "f32", 3)
    k, v = normal((tokens, 2, dim), "f32", 4), normal((tokens, 2, dim), "f32", 5)
    cos, sin = rotary_table(128, dim)
    extra = {"q_norm": torch.rand(dim, device="cuda") + 0.5, "cos": cos, "sin": sin}
    table = ints([[0, 1]])
    whole = make_cache(2, dim, 2, 1).append(step([0], [tokens], table), k, v, q=q, **extra)
    cache = make_cache(2, dim, 2, 1)
    for t in range(tokens):
        one = cache.append(step([t], [1], table), k[t:t + 1], v[t:t + 1], q=q[t:t + 1], **extra)
        assert torch.equal(one[0], whole[t]), t
