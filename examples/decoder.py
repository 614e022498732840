"""A decoder on the library's operators: Q4 matrix products, cache append with
rotation, attention over the 8-bit paged cache, norms with the residual add.

Weights are random, in the shapes of Qwen3-8B by default.  A prompt goes
through in steps of up to eight tokens (the batched products' limit), then
tokens are decoded one by one, each step a replay of one captured HIP graph.

    python examples/decoder.py --layers 36 --prompt 100 --tokens 50
"""
from __future__ import annotations

import argparse
import os
import sys
import time
from dataclasses import dataclass

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rdna-gfx1201-v0.1_amd"))
from q4rdna import api  # noqa: E402


@dataclass
class Shape:
    layers: int = 36
    hidden: int = 4096
    heads: int = 32
    kv_heads: int = 8
    head_dim: int = 128
    ffn: int = 12288
    vocab: int = 151936
    rope_base: float = 1e6
    eps: float = 1e-6


class Decoder:
    """Random weights, one cache per layer, one sequence."""

    def __init__(self, shape: Shape, max_tokens: int, seed: int = 0, device: int = 0):
        self.shape, self.device = shape, torch.device("cuda", device)
        gen = torch.Generator(device=self.device).manual_seed(seed)

        def matrix(rows, cols):
            w = torch.randn((rows, cols), device=self.device, generator=gen) * cols ** -0.5
            return api.QWeight.from_tiles(api.pack(w), rows, cols)

        def weight(n):
            return 1 + 0.1 * torch.randn(n, device=self.device, generator=gen)

        s, q, kv = shape, shape.heads * shape.head_dim, shape.kv_heads * shape.head_dim
        self.embedding = torch.randn((s.vocab, s.hidden), device=self.device, generator=gen)
        self.layers = [dict(norm1=weight(s.hidden), norm2=weight(s.hidden), q_norm=weight(s.head_dim), k_norm=weight(s.head_dim),
                            q=matrix(q, s.hidden), k=matrix(kv, s.hidden), v=matrix(kv, s.hidden), o=matrix(s.hidden, q),
                            gate=matrix(s.ffn, s.hidden), up=matrix(s.ffn, s.hidden), down=matrix(s.hidden, s.ffn))
                       for _ in range(s.layers)]
        self.norm, self.head = weight(s.hidden), matrix(s.vocab, s.hidden)
        pages = (max_tokens + 63) // 64
        self.caches = [api.KVCache.empty(pages, 1, s.kv_heads, s.head_dim, device) for _ in range(s.layers)]
        self.table = torch.arange(pages, dtype=torch.int32, device=self.device)[None]
        self.past = torch.zeros(1, dtype=torch.int32, device=self.device)
        angle = torch.arange(max_tokens, device=self.device).double()[:, None] * s.rope_base ** (
            -torch.arange(s.head_dim // 2, device=self.device).double() / (s.head_dim // 2))
        self.cos, self.sin = angle.cos().float(), angle.sin().float()
        self.max_tokens, self.length = max_tokens, 0

    def _products(self, x, *weights):
        """One activation by several weights: a group launch for one token."""
        n = x.shape[0]
        ys = [torch.empty((n, w.rows), device=self.device) for w in weights]
        if n == 1:
            api.mul_mat_group([(w, y[0]) for w, y in zip(weights, ys)], x[0])
        else:
            for w, y in zip(weights, ys):
                api.mul_mat_batch(w, x, y)
        return ys

    def forward(self, x: torch.Tensor, batch: api.KVBatch) -> torch.Tensor:
        """Logits [n, vocab] of the step's n <= 8 embedded tokens [n, hidden]."""
        s, n = self.shape, x.shape[0]
        h, y = x, None
        for layer, cache in zip(self.layers, self.caches):
            h, normed = api.add_norm(h, y, layer["norm1"], eps=s.eps)
            q, k, v = self._products(normed, layer["q"], layer["k"], layer["v"])
            q = cache.append(batch, k.view(n, s.kv_heads, s.head_dim), v.view(n, s.kv_heads, s.head_dim),
                             q=q.view(n, s.heads, s.head_dim), cos=self.cos, sin=self.sin, q_norm=layer["q_norm"],
                             k_norm=layer["k_norm"], eps=s.eps)
            attended = cache.attend(batch, q)
            (y,) = self._products(attended.view(n, -1), layer["o"])
            h, normed = api.add_norm(h, y, layer["norm2"], eps=s.eps)
            inner = torch.empty((n, s.ffn), device=self.device)
            if n == 1:
                api.mul_mat_glu(layer["up"], layer["gate"], normed[0], inner[0])
            else:
                api.mul_mat_batch(layer["up"], normed, inner, gate=layer["gate"])
            (y,) = self._products(inner, layer["down"])
        _, normed = api.add_norm(h, y, self.norm, eps=s.eps)
        return self._products(normed, self.head)[0]

    def prompt(self, tokens: list[int]) -> torch.Tensor:
        """Append a prompt, up to eight tokens a step; the last token's logits."""
        if not tokens:
            raise ValueError("an empty prompt")
        for at in range(0, len(tokens), 8):
            ids = torch.tensor(tokens[at:at + 8], device=self.device)
            n = len(ids)
            if self.length + n > self.max_tokens:
                raise ValueError(f"more than {self.max_tokens} tokens")
            cu = torch.tensor([0, n], dtype=torch.int32, device=self.device)
            logits = self.forward(self.embedding[ids], api.KVBatch(self.past, self.table, cu_tokens=cu, max_tokens=n))
            self.past += n
            self.length += n
        return logits[-1]

    def decode(self, logits: torch.Tensor, count: int) -> tuple[list[int], float]:
        """Decode greedily from the given logits: (tokens, seconds a step).  The
        model's step is captured once; the sequence's length, the token and the
        logits live in tensors that the graph reads and writes."""
        if self.length + count > self.max_tokens:
            raise ValueError(f"more than {self.max_tokens} tokens")
        if count == 0:
            return [], 0.0
        batch = api.KVBatch(self.past, self.table)
        token = logits.argmax().reshape(1)

        def step():
            return self.forward(self.embedding[token], batch)[0]

        stream = torch.cuda.Stream(self.device)
        stream.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(stream):
            step()  # every shape once on this stream: scratch grows here, not in the capture
        torch.cuda.current_stream(self.device).wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            logits = step()
        chosen = []
        torch.cuda.synchronize(self.device)
        began = time.perf_counter()
        for _ in range(count):
            chosen.append(token.clone())
            graph.replay()
            # Outside the graph: torch's argmax over many logits sets memory
            # that it counts in, and such a node must not be replayed.
            token.copy_(logits.argmax())
            self.past += 1
        torch.cuda.synchronize(self.device)
        spent = (time.perf_counter() - began) / count
        self.length += count
        return [int(t) for t in chosen], spent


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=36)
    ap.add_argument("--prompt", type=int, default=100, help="tokens of the (random) prompt")
    ap.add_argument("--tokens", type=int, default=50, help="tokens to decode")
    a = ap.parse_args()
    model = Decoder(Shape(layers=a.layers), a.prompt + a.tokens + 1)
    ids = torch.randint(0, model.shape.vocab, (a.prompt,), generator=torch.Generator().manual_seed(1)).tolist()
    tokens, spent = model.decode(model.prompt(ids), a.tokens)
    print(f"{a.layers} layers, {a.prompt} + {a.tokens} tokens: {spent * 1e6:.1f} us a token ({1 / spent:.0f} tokens/s)")
    print("tokens", tokens[:10], "...", "cache faults", sum(c.faults() for c in model.caches))


if __name__ == "__main__":
    main()
