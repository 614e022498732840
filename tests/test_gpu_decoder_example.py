"""examples/decoder.py: the operators together, against the model in 64 bits."""
import os
import sys

import numpy as np
import pytest
import torch

import layer_reference as R

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model_and_reference():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import decoder
    shape = decoder.Shape(layers=2, hidden=256, heads=6, kv_heads=2, head_dim=64, ffn=512, vocab=320)
    return decoder, shape


def dense(w):
    from q4rdna import api
    return api.dequantize(w).cpu().double().numpy()


def reference_logits(model, shape, tokens):
    """The whole sequence's logits in 64 bits, with the weights as they are
    packed and keys and values unrounded."""
    g = lambda t: t.cpu().double().numpy()  # noqa: E731
    x, y = g(model.embedding)[tokens], 0.0
    n, d = len(tokens), shape.head_dim
    cos, sin = g(model.cos), g(model.sin)
    for layer in model.layers:
        x = x + y
        h = R.rms(x, g(layer["norm1"]), shape.eps)
        q, k, v = (h @ dense(layer[name]).T for name in "qkv")
        q = R.rms(q.reshape(n, shape.heads, d), g(layer["q_norm"]), shape.eps)
        k = R.rms(k.reshape(n, shape.kv_heads, d), g(layer["k_norm"]), shape.eps)
        v = v.reshape(n, shape.kv_heads, d)
        q = np.stack([R.rotate(q[t], t, cos, sin, False) for t in range(n)])
        k = np.stack([R.rotate(k[t], t, cos, sin, False) for t in range(n)])
        group = shape.heads // shape.kv_heads
        out = np.stack([R.attend(q[:, h_], k[:, h_ // group], v[:, h_ // group], range(n), d ** -0.5, 0)[0]
                        for h_ in range(shape.heads)], axis=1)
        x = x + out.reshape(n, -1) @ dense(layer["o"]).T
        h = R.rms(x, g(layer["norm2"]), shape.eps)
        gate, up = h @ dense(layer["gate"]).T, h @ dense(layer["up"]).T
        y = (up * gate / (1 + np.exp(-gate))) @ dense(layer["down"]).T
    return R.rms(x + y, g(model.norm), shape.eps) @ dense(model.head).T


def test_prompt_and_decoding_agree_with_the_model(model_and_reference):
    """Logits after a prompt of 77 tokens and the greedy tokens after it.  The
    cache rounds full blocks to 8 bits: a key or value is off by at most
    absmax / 254, rms absmax / 440, about 1% of an rms number (absmax 3.7 of
    64 x 64 normal numbers); through two layers, averaged over the tokens that
    a row attends to, the logits move by a few percent of their rms at most."""
    decoder, shape = model_and_reference
    model = decoder.Decoder(shape, 128)
    tokens = torch.randint(0, shape.vocab, (77,), generator=torch.Generator().manual_seed(3)).tolist()
    logits = model.prompt(tokens)
    want = reference_logits(model, shape, tokens)[-1]
    rms = np.sqrt(np.mean(want ** 2))
    got = logits.cpu().double().numpy()
    assert np.sqrt(np.mean((got - want) ** 2)) <= 0.03 * rms
    chosen, spent = model.decode(logits, 20)
    assert spent > 0 and sum(c.faults() for c in model.caches) == 0
    # each token is a best one in 64 bits, up to the logits' own error
    every = reference_logits(model, shape, tokens + chosen)
    for i, t in enumerate(chosen):
        row = every[len(tokens) - 1 + i]
        assert row[t] >= row.max() - 0.15 * np.sqrt(np.mean(row ** 2)), i


def test_steps_of_any_size_fill_the_cache_alike(model_and_reference):
    """The same tokens eight at a time and one at a time: full blocks hold the
    same codes up to what the two forms of the products differ by."""
    decoder, shape = model_and_reference
    a, b = decoder.Decoder(shape, 64), decoder.Decoder(shape, 64)
    tokens = torch.randint(0, shape.vocab, (40,), generator=torch.Generator().manual_seed(4)).tolist()
    x = a.prompt(tokens)
    for t in tokens:
        y = b.prompt([t])
    # fp32 sums in another order through two layers: under 1e-4 of the logits' rms
    assert (x - y).square().mean().sqrt() <= 1e-4 * x.square().mean().sqrt()
