"""examples/decoder.py: the caches of a prompt given eight tokens at a time and
one at a time."""
import pytest
import torch

from test_gpu_decoder_example import model_and_reference  # noqa: F401

pytestmark = pytest.mark.gpu


def test_full_blocks_hold_the_same_numbers(cuda, model_and_reference):  # noqa: F811
    """150 tokens, two full blocks and an open one.  The batched products add in
    another order than the single ones; a number that this moves across the
    middle between two codes changes by one step of 8 bits, in an open block of
    16.  Through the attention such a step moves later numbers by p / 127 of the
    values, spread over the output product's columns: under 1e-3 of a token's
    largest, which is 127e-3 of a step, so as many codes at most change."""
    decoder, shape = model_and_reference
    a, b = decoder.Decoder(shape, 192), decoder.Decoder(shape, 192)
    tokens = torch.randint(0, shape.vocab, (150,), generator=torch.Generator().manual_seed(5)).tolist()
    a.prompt(tokens)
    for t in tokens:
        b.prompt([t])
    from q4rdna import api
    whole = api.KVBatch(torch.zeros_like(a.past), a.table, cu_tokens=torch.tensor([0, 150], dtype=torch.int32, device="cuda"), max_tokens=150)
    for x, y in zip(a.caches, b.caches):
        assert x.faults() == 0 and y.faults() == 0
        scale = y.scales[:2]
        assert ((x.scales[:2] - scale).abs() <= 1e-3 * scale).all()
        off = (x.pages[:2].int() - y.pages[:2].int()).abs()
        assert off.max() <= 1 and (off > 0).float().mean() <= 0.127
        for u, v in zip(x.read(whole, 150), y.read(whole, 150)):
            top = v[128:].abs().amax(dim=-1, keepdim=True)
            assert ((u[128:] - v[128:]).abs() <= (1e-3 + 1 / 32512) * top).all()
