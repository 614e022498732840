"""The operators between a decoder layer's matrix products, as cases whose time can be measured.

A case is a dict of plain values.  `prepare` makes what a program holds before
the call (activations, the cache's buffers, the step's block tables), `run`
makes one pass through an operator, and `exact` gives the same outputs in 64
bits from the operator's definition.

Kinds of case:
  append  a step's keys and values, rotated by position, into the paged 8-bit
          cache, and the blocks they touch read back as numbers
  attend  attention of a step's query tokens over that cache
  norm    residual add with gate and scale, with the norms before and after it

The cache holds blocks of 64 tokens.  A full block is int8 codes with one
scale per head for K and one for V; the last, partly filled block of a
sequence is 16-bit codes, as two int8 planes (256 * hi + lo), with a scale per
token and head.  Codes lie in the order in which a 64-lane int8 matrix
instruction takes them (`_unlay_k`, `_unlay_v`).
"""
import math
import os
import random
import sys

import torch

own = False  # True: the library's kernels; False: the plain forms below

DEV = "cuda"
BLOCK = 64       # tokens of a cache block
CODE16 = 32512   # 127 * 256, the largest 16-bit code (its high byte fits int8)
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # The first answer token after a short prompt, one user: the smallest attention call.
        {"name": "attend_first_token", "kind": "attend", "dtype": "f32", "kv_heads": 8, "group": 4, "dim": 128,
         "seqs": 1, "min_past": 17, "max_past": 17, "tokens": 1, "ragged": False, "window": 0, "lse": False},
        # One user with a very long document behind every new token.
        {"name": "attend_long", "kind": "attend", "dtype": "f32", "kv_heads": 8, "group": 4, "dim": 128,
         "seqs": 1, "min_past": 130001, "max_past": 130001, "tokens": 1, "ragged": False, "window": 0, "lse": False},
        # A serving batch: 32 conversations of very different lengths, one token each.
        {"name": "attend_batch", "kind": "attend", "dtype": "bf16", "kv_heads": 8, "group": 4, "dim": 128,
         "seqs": 32, "min_past": 100, "max_past": 8000, "tokens": 1, "ragged": False, "window": 0, "lse": False},
        # Speculated tokens verified at once, sliding window, an odd number of query heads per kv head.
        {"name": "attend_verify", "kind": "attend", "dtype": "f16", "kv_heads": 4, "group": 7, "dim": 64,
         "seqs": 9, "min_past": 61, "max_past": 5000, "tokens": 5, "ragged": True, "window": 1000, "lse": True},
        # A whole prompt of one user, fp32 as the library's matrix products take and give it.
        {"name": "attend_prompt", "kind": "attend", "dtype": "f32", "kv_heads": 8, "group": 4, "dim": 128,
         "seqs": 1, "min_past": 0, "max_past": 0, "tokens": 2047, "ragged": False, "window": 0, "lse": False},
        # A further chunk of a long prompt.
        {"name": "attend_chunk", "kind": "attend", "dtype": "bf16", "kv_heads": 8, "group": 4, "dim": 128,
         "seqs": 1, "min_past": 6100, "max_past": 6100, "tokens": 2048, "ragged": False, "window": 0, "lse": False},
        # One token of one user into the cache, with the norm of each head's query and key.
        {"name": "append_token", "kind": "append", "dtype": "f32", "kv_heads": 8, "group": 4, "dim": 128,
         "seqs": 1, "min_past": 1000, "max_past": 1000, "tokens": 1, "ragged": False, "norm": True, "pairs": "halves"},
        # A serving batch: one token each, some of which fill their block.
        {"name": "append_batch", "kind": "append", "dtype": "bf16", "kv_heads": 8, "group": 4, "dim": 128,
         "seqs": 64, "min_past": 63, "max_past": 8000, "tokens": 1, "ragged": False, "norm": False, "pairs": "halves"},
        # Prompts of several users, ragged, neighbouring numbers rotated together.
        {"name": "append_prompts", "kind": "append", "dtype": "bf16", "kv_heads": 8, "group": 4, "dim": 128,
         "seqs": 6, "min_past": 0, "max_past": 700, "tokens": 2500, "ragged": True, "norm": True, "pairs": "neighbours"},
        # Between two matrix products of one decoded token.
        {"name": "norm_token", "kind": "norm", "dtype": "f32", "rows": 1, "width": 4096, "post": False, "gate": ""},
        # A small batch at an odd width.
        {"name": "norm_odd", "kind": "norm", "dtype": "f16", "rows": 77, "width": 1111, "post": True, "gate": "row"},
        # A prompt through a block with norms on both sides and a gate per channel.
        {"name": "norm_prompt", "kind": "norm", "dtype": "bf16", "rows": 8192, "width": 4096, "post": True,
         "gate": "channel"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "append", "norm"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind == "norm":
        width = _log(rng, 64, 16384)
        return {"kind": kind, "dtype": dtype, "rows": _log(rng, 1, max(1, min(16384, (1 << 25) // width))),
                "width": width, "post": rng.random() < 0.5, "gate": rng.choice(["", "channel", "row"])}
    dim, kv_heads, group = rng.choice([64, 128, 128]), rng.choice([1, 2, 3, 4, 8, 8, 16]), rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 12])
    base = {"kind": kind, "dtype": dtype, "kv_heads": kv_heads, "group": group, "dim": dim}
    if kind == "append":
        seqs = _log(rng, 1, 128)
        tokens = rng.choice([1, 1, _log(rng, 2, 12), _log(rng, 12, 4000)])
        tokens = max(1, min(tokens, (1 << 25) // (seqs * kv_heads * (group + 2) * dim)))
        lo = rng.randint(0, 200)
        return dict(base, seqs=seqs, min_past=lo, max_past=lo + _log(rng, 1, 8000), tokens=tokens,
                    ragged=rng.random() < 0.5, norm=rng.random() < 0.5, pairs=rng.choice(["halves", "neighbours"]))
    if rng.random() < 0.6:  # few query tokens over long caches
        tokens = rng.choice([1, 1, 1, _log(rng, 2, 16)])
        seqs = _log(rng, 1, 96)
        most = min(130000, (1 << 27) // (seqs * kv_heads * dim), (1 << 27) // (seqs * kv_heads * group * tokens))
        hi = _log(rng, 1, max(2, most))
        lo = _log(rng, 1, hi) if rng.random() < 0.7 else 0
    else:  # prompts and chunks of them
        tokens, seqs = _log(rng, 17, 2500), rng.choice([1, 1, 2, 3])
        most = max(0, min(20000, (1 << 28) // (seqs * kv_heads * group * tokens) - tokens))
        hi = rng.choice([0, rng.randint(0, most)])
        lo = rng.randint(0, hi)
        tokens = max(17, min(tokens, (1 << 28) // (seqs * kv_heads * group * (hi + tokens))))
    return dict(base, seqs=seqs, min_past=lo, max_past=hi, tokens=tokens, ragged=rng.random() < 0.5,
                window=rng.choice([0, 0, _log(rng, 16, 4096)]), lse=rng.random() < 0.3)


def _lengths(case):
    """(past, tokens) of each sequence: pasts spread over their range on a
    logarithmic scale, in a shuffled order; tokens from one to the most where
    they are ragged."""
    n, lo, hi, most = case["seqs"], case["min_past"], case["max_past"], case["tokens"]
    r = random.Random(n * 1000003 + hi * 31 + most)
    past = [int(round(math.exp(math.log(lo + 1) + (math.log(hi + 1) - math.log(lo + 1)) * i / max(1, n - 1)))) - 1
            for i in range(n)]
    r.shuffle(past)
    count = [r.randint(1, most) for _ in range(n)] if case["ragged"] else [most] * n
    if case["ragged"]:
        count[r.randrange(n)] = most
    return past, count


def _visible(case):
    """Sum over query tokens of the tokens that each sees, and the tokens that
    any query token of its sequence sees, summed over sequences."""
    pairs = read = 0
    w = case["window"]
    for p, t in zip(*_lengths(case)):
        if w:
            pairs += sum(min(w, p + j + 1) for j in range(t))
            read += min(p + t, w + t - 1)
        else:
            pairs += t * p + t * (t + 1) // 2
            read += p + t
    return pairs, read


def work(case):
    size = SIZE[case["dtype"]]
    if case["kind"] == "norm":
        n = case["rows"] * case["width"]
        rows = 4 * n + (n if case["gate"] == "row" else case["width"] if case["gate"] == "channel" else 0)
        return {"bytes": rows * size + case["width"] * 4 * (2 if case["post"] else 1),
                "flops": n * (10 if case["post"] else 6)}
    kv, heads, dim = case["kv_heads"], case["kv_heads"] * case["group"], case["dim"]
    past, count = _lengths(case)
    tokens = sum(count)
    if case["kind"] == "attend":
        pairs, read = _visible(case)
        # int8 codes, the open block's tokens with 16 bits, a scale per block
        opened = sum(min((p + t) % BLOCK, p + t) for p, t in zip(past, count))
        return {"bytes": 2 * kv * (dim * (read + opened) + 4 * read // BLOCK) + 2 * tokens * heads * dim * size
                + (tokens * heads * 4 if case["lse"] else 0), "flops": 4 * dim * heads * pairs}
    # q, k and v read, q written; new codes written (8 bits in full blocks, 16 in open ones), the touched
    # blocks' tokens given back as 16-bit numbers
    touched = sum(p % BLOCK + t for p, t in zip(past, count))
    opened = sum(min((p + t) % BLOCK, t) for p, t in zip(past, count))
    return {"bytes": tokens * (2 * heads + 2 * kv) * dim * size + 2 * kv * dim * (touched + opened)
            + 2 * kv * dim * 2 * touched + tokens * dim * 4, "flops": 10 * tokens * (heads + 2 * kv) * dim}


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _tables(case, gen, past, count):
    """Block table over physical pages in random order, and the pages there are."""
    need = [(p + t + BLOCK - 1) // BLOCK for p, t in zip(past, count)]
    pages = sum(need) + 3
    order = torch.randperm(pages, device=DEV, generator=gen).int()
    width = max(need)
    start = torch.tensor([sum(need[:i]) for i in range(len(need))], device=DEV)
    at = start[:, None] + torch.arange(width, device=DEV)[None, :]
    live = torch.arange(width, device=DEV)[None, :] < torch.tensor(need, device=DEV)[:, None]
    table = torch.where(live, order[at.clamp(max=pages - 1)], torch.zeros((), dtype=torch.int32, device=DEV))
    return table.contiguous(), pages


def _buffers(case, gen, pages, slots):
    """A cache in use: codes of normally distributed numbers with a scale of
    their own per block and head, some heads several times larger."""
    kv, dim = case["kv_heads"], case["dim"]

    def codes(shape, spread):
        x = torch.randn(shape, device=DEV, generator=gen)
        return x.mul_(spread).round_().clamp_(-127, 127).to(torch.int8)

    loud = 1 + 2 * (torch.rand((kv, 2), device=DEV, generator=gen) > 0.8).float()
    scales = (0.02 + 0.02 * torch.rand((pages, kv, 2), device=DEV, generator=gen)) * loud
    open_scales = (0.8 + 0.8 * torch.rand((slots, 2, kv, 2, BLOCK), device=DEV, generator=gen)) / 8192 * loud[:, :, None]
    return {"pages": codes((pages, kv, 2, BLOCK * dim), 35.0), "scales": scales.contiguous(),
            "open": codes((slots, 2, kv, 4, BLOCK * dim), 35.0), "open_scales": open_scales.contiguous()}


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, spread=1.0):
        return (torch.randn(shape, device=DEV, generator=gen) * spread).to(dtype)

    if case["kind"] == "norm":
        rows, width = case["rows"], case["width"]
        gate = {"": None, "channel": (width,), "row": (rows, width)}[case["gate"]]
        return {"case": case, "residual": normal(rows, width, spread=3.0), "y": normal(rows, width),
                "norm": 1 + 0.2 * torch.randn(width, device=DEV, generator=gen),
                "post": 1 + 0.2 * torch.randn(width, device=DEV, generator=gen) if case["post"] else None,
                "gate": None if gate is None else normal(*gate)}

    past, count = _lengths(case)
    n, tokens = case["seqs"], sum(count)
    heads, kv, dim = case["kv_heads"] * case["group"], case["kv_heads"], case["dim"]
    table, pages = _tables(case, gen, past, count)
    state = {"case": case, "table": table, "past": _ints(past),
             "cu": _ints([sum(count[:i]) for i in range(n + 1)]) if case["tokens"] > 1 else None}
    state.update(_buffers(case, gen, pages, n))
    seq = torch.repeat_interleave(torch.arange(n, device=DEV), torch.tensor(count, device=DEV))
    first = torch.tensor([sum(count[:i]) for i in range(n)], device=DEV)
    state["seq"] = seq
    state["place"] = torch.arange(tokens, device=DEV) - first[seq]  # of a token among its sequence's
    state["position"] = torch.tensor(past, device=DEV)[seq] + state["place"]
    state["most"] = max(count)
    if case["kind"] == "attend":
        state["q"] = normal(tokens, heads, dim, spread=1.7)
        state["longest"] = max(p + t for p, t in zip(past, count))
    else:
        state.update(q=normal(tokens, heads, dim), k=normal(tokens, kv, dim, spread=2.0), v=normal(tokens, kv, dim))
        limit = max(p + t for p, t in zip(past, count))
        angle = torch.arange(limit, device=DEV).double()[:, None] * 1e6 ** (
            -torch.arange(dim // 2, device=DEV).double() / (dim // 2))
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        for name in ("q_norm", "k_norm"):
            state[name] = 1 + 0.2 * torch.randn(dim, device=DEV, generator=gen) if case["norm"] else None
        # the blocks that the step touches, and the tokens in them
        blocks = [(i, b) for i in range(n) for b in range(past[i] // BLOCK, (past[i] + count[i] - 1) // BLOCK + 1)]
        base = {}
        for at, (i, b) in enumerate(blocks):
            base.setdefault(i, at - b)
        state["block_seq"] = torch.tensor([i for i, _ in blocks], device=DEV)
        state["block"] = torch.tensor([b for _, b in blocks], device=DEV)
        state["row"] = torch.tensor([base[i] for i in range(n)], device=DEV)[seq] + state["position"] // BLOCK
        length = torch.tensor([past[i] + count[i] for i, _ in blocks], device=DEV)
        state["full"] = (state["block"] + 1) * BLOCK <= length
        state["kept16"] = state["block"] >= length // BLOCK - 1
        state["live"] = state["block"][:, None] * BLOCK + torch.arange(BLOCK, device=DEV) < length[:, None]
        state["live_at"] = state["live"].reshape(-1).nonzero().squeeze(1)
        from_block = [p // BLOCK * BLOCK for p in past]
        span = [p + t - f for p, t, f in zip(past, count, from_block)]
        state["read_past"] = _ints(from_block)
        state["read_cu"] = _ints([sum(span[:i]) for i in range(n + 1)])
        state["read_most"], state["read_tokens"] = max(span), sum(span)
    if own:
        sys.path.insert(0, os.path.join(os.getcwd(), "rdna-gfx1201-v0.1_amd"))
        from q4rdna import api
        state["cache"] = api.KVCache(state["pages"], state["scales"], state["open"], state["open_scales"])
        state["step"] = api.KVBatch(state["past"], state["table"], cu_tokens=state["cu"], max_tokens=state["most"])
        if case["kind"] == "append":
            state["read_step"] = api.KVBatch(state["read_past"], state["table"], cu_tokens=state["read_cu"],
                                             max_tokens=state["read_most"])
    return state


# --- the plain forms ---------------------------------------------------------

def _unlay_k(codes, dim):
    """[..., 64 * dim] K codes -> [..., 64 tokens, dim]: 16-token tiles, 64-number steps, 4 lane groups of 16
    lanes (a token each) with 16 numbers."""
    lead = codes.shape[:-1]
    x = codes.reshape(*lead, 4, dim // 64, 4, 16, 16)
    k = len(lead)
    return x.permute(*range(k), k, k + 3, k + 1, k + 2, k + 4).reshape(*lead, BLOCK, dim)


def _lay_k(x):
    dim = x.shape[-1]
    lead = x.shape[:-2]
    k = len(lead)
    x = x.reshape(*lead, 4, 16, dim // 64, 4, 16)
    return x.permute(*range(k), k, k + 2, k + 3, k + 1, k + 4).reshape(*lead, BLOCK * dim)


def _unlay_v(codes, dim):
    """[..., 64 * dim] V codes -> [..., 64 tokens, dim]: 16-number tiles, 4 lane groups of 16 lanes (a number
    each) with 16 tokens: token 16 a + 4 group + b at byte 4 a + b."""
    lead = codes.shape[:-1]
    x = codes.reshape(*lead, dim // 16, 4, 16, 4, 4)
    k = len(lead)
    return x.permute(*range(k), k + 3, k + 1, k + 4, k, k + 2).reshape(*lead, BLOCK, dim)


def _lay_v(x):
    dim = x.shape[-1]
    lead = x.shape[:-2]
    k = len(lead)
    x = x.reshape(*lead, 4, 4, 4, dim // 16, 16)
    return x.permute(*range(k), k + 3, k + 1, k + 4, k, k + 2).reshape(*lead, BLOCK * dim)


def _plain_attend(s):
    case = s["case"]
    kv, group, dim, n = case["kv_heads"], case["group"], case["dim"], case["seqs"]
    t, nb = s["most"], s["table"].shape[1]
    slot = torch.arange(n, device=DEV)
    count = s["cu"].diff().long() if s["cu"] is not None else torch.ones(n, dtype=torch.long, device=DEV)
    length = s["past"].long() + count
    table = s["table"].long()
    last = length // BLOCK  # the open block, where there is one
    opened = ((length % BLOCK > 0)[:, None] & (torch.arange(nb, device=DEV) == last[:, None]))[:, :, None, None, None]
    both = []
    for which, unlay in ((0, _unlay_k), (1, _unlay_v)):
        x = unlay(s["pages"][:, :, which], dim)[table].float() * s["scales"][:, :, which][table][..., None, None]
        o, o_scale = s["open"][slot, last % 2], s["open_scales"][slot, last % 2, :, which]
        y = (unlay(o[:, :, 2 * which], dim).float() * 256 + unlay(o[:, :, 2 * which + 1], dim).float()) * o_scale[..., None]
        x = torch.where(opened, y[:, None], x)
        both.append(x.permute(0, 2, 1, 3, 4).reshape(n, kv, nb * BLOCK, dim))
    keys, values = both
    # query tokens of a sequence side by side, absent ones zero
    q = torch.zeros((n, t, kv, group, dim), dtype=torch.float32, device=DEV)
    q[s["seq"], s["place"]] = s["q"].float().reshape(-1, kv, group, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(n, kv, t * group, dim)
    scores = torch.matmul(q, keys.transpose(-1, -2).contiguous()) * dim ** -0.5
    position = s["past"].long()[:, None] + torch.arange(t, device=DEV)  # [n, t]
    key = torch.arange(nb * BLOCK, device=DEV)
    seen = key <= position[:, :, None]
    if case["window"]:
        seen &= key > position[:, :, None] - case["window"]
    scores = scores.reshape(n, kv, t, group, -1).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (top + total.log()).squeeze(-1)
    p = p.div_(total).reshape(n, kv, t * group, -1)
    out = torch.matmul(p, values).reshape(n, kv, t, group, dim).permute(0, 2, 1, 3, 4)
    out = out[s["seq"], s["place"]].reshape(-1, kv * group, dim).to(s["q"].dtype)
    if not case["lse"]:
        return {"out": out}
    return {"out": out, "lse": lse.permute(0, 2, 1, 3)[s["seq"], s["place"]].reshape(-1, kv * group)}


def _plain_rotate(s, x, weight):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight
    c, n = s["cos"][s["position"]][:, None], s["sin"][s["position"]][:, None]
    if s["case"]["pairs"] == "halves":
        a, b = x.chunk(2, -1)
        return torch.cat((a * c - b * n, b * c + a * n), -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * n, b * c + a * n), -1).flatten(-2)


def _plain_append(s):
    case = s["case"]
    dim = case["dim"]
    out = {"q": _plain_rotate(s, s["q"], s["q_norm"]).to(s["q"].dtype)}
    seq, block = s["block_seq"], s["block"]
    page = s["table"][seq, block].long()
    row, place = s["row"], s["position"] % BLOCK
    full, kept = s["full"], s["kept16"]
    for which, name, x, lay, unlay in ((0, "k", _plain_rotate(s, s["k"], s["k_norm"]), _lay_k, _unlay_k),
                                       (1, "v", s["v"].float(), _lay_v, _unlay_v)):
        top = x.abs().amax(-1, keepdim=True)
        code = torch.round(x * (CODE16 / top))
        # the touched blocks with 16 bits a number: [blocks, 64, heads, dim]
        o = s["open"][seq, block % 2]
        code16 = (unlay(o[:, :, 2 * which], dim).float() * 256 + unlay(o[:, :, 2 * which + 1], dim).float()).transpose(1, 2).contiguous()
        scale16 = s["open_scales"][seq, block % 2, :, which].transpose(1, 2).contiguous()
        code16[row, place] = code
        scale16[row, place] = top.squeeze(-1) / CODE16
        low = torch.remainder(code16 + 128, 256) - 128
        s["open"][seq[kept], block[kept] % 2, :, 2 * which] = lay(((code16 - low) / 256)[kept].transpose(1, 2)).to(torch.int8)
        s["open"][seq[kept], block[kept] % 2, :, 2 * which + 1] = lay(low[kept].transpose(1, 2)).to(torch.int8)
        s["open_scales"][seq[kept], block[kept] % 2, :, which] = scale16[kept].transpose(1, 2)
        scale8 = 256 * scale16.amax(1, keepdim=True)
        code8 = torch.round(code16 * (scale16 / scale8)[..., None])
        s["pages"][page[full], :, which] = lay(code8[full].transpose(1, 2)).to(torch.int8)
        s["scales"][page[full], :, which] = scale8.squeeze(1)[full]
        values = torch.where(full[:, None, None, None], code8 * scale8[..., None], code16 * scale16[..., None])
        out[name] = values.reshape(-1, case["kv_heads"], dim)[s["live_at"]].half()
    return out


def _plain_norm(s):
    y = s["y"].float()
    if s["post"] is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * s["post"]
    if s["gate"] is not None:
        y = y * s["gate"].float()
    h = s["residual"].float() + 0.5 * y
    n = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * s["norm"]
    return {"h": h.to(s["y"].dtype), "n": n.to(s["y"].dtype)}


def _own_attend(s):
    if s["case"]["lse"]:
        out, lse = s["cache"].attend(s["step"], s["q"], window=s["case"]["window"], lse=True)
        return {"out": out, "lse": lse}
    return {"out": s["cache"].attend(s["step"], s["q"], window=s["case"]["window"])}


def _own_append(s):
    q = s["cache"].append(s["step"], s["k"], s["v"], q=s["q"], cos=s["cos"], sin=s["sin"],
                          interleaved=s["case"]["pairs"] == "neighbours", q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6)
    k, v = s["cache"].read(s["read_step"], s["read_tokens"], dtype=torch.float16)
    return {"q": q, "k": k, "v": v}


def _own_norm(s):
    from q4rdna import api
    h, n = api.add_norm(s["residual"], s["y"], s["norm"], post_weight=s["post"], gate=s["gate"], scale=0.5, eps=1e-6)
    return {"h": h, "n": n}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attend": _own_attend, "append": _own_append, "norm": _own_norm}[kind](state)
    return {"attend": _plain_attend, "append": _plain_append, "norm": _plain_norm}[kind](state)


# --- the definitions in 64 bits ------------------------------------------------

def _code_places(dim):
    """For each code of a block, its token and its number within the head, for K and for V."""
    i = torch.arange(BLOCK * dim, device=DEV)
    byte, lane, tile = i % 16, i // 16 % 64, i // 1024
    steps = dim // 64
    k_token, k_number = tile // steps * 16 + lane % 16, tile % steps * 64 + lane // 16 * 16 + byte
    v_token, v_number = byte // 4 * 16 + lane // 16 * 4 + byte % 4, tile * 16 + lane % 16
    return (k_token, k_number), (v_token, v_number)


def _exact_tokens(s, i, head, which, past, count):
    """[length, dim] K or V of one sequence and head, 64 bits."""
    dim = s["case"]["dim"]
    token, number = _code_places(dim)[which]
    length = past + count
    blocks = (length + BLOCK - 1) // BLOCK
    x = torch.zeros((blocks, BLOCK, dim), dtype=torch.float64, device=DEV)
    pages = s["table"][i, :blocks].long()
    x[:, token, number] = s["pages"][pages, head, which].double() * s["scales"][pages, head, which].double()[:, None]
    if length % BLOCK:
        o = s["open"][i, (blocks - 1) % 2, head].double()
        x[blocks - 1, token, number] = 256 * o[2 * which] + o[2 * which + 1]
        x[blocks - 1] *= s["open_scales"][i, (blocks - 1) % 2, head, which].double()[:, None]
    return x.reshape(-1, dim)[:length]


def _exact_attend(s):
    case = s["case"]
    past, count = _lengths(case)
    kv, group, dim = case["kv_heads"], case["group"], case["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device=DEV)
    at = 0
    for i, (p, t) in enumerate(zip(past, count)):
        length = p + t
        for head in range(kv):
            keys, values = (_exact_tokens(s, i, head, which, p, t) for which in (0, 1))
            q = s["q"][at:at + t, head * group:(head + 1) * group].double()
            score = (q.reshape(-1, dim) @ keys.T.contiguous()).reshape(t, group, length) / math.sqrt(dim)
            ahead = torch.arange(length, device=DEV) - (p + torch.arange(t, device=DEV))[:, None]
            hidden = ahead > 0
            if case["window"]:
                hidden |= ahead <= -case["window"]
            score = score.masked_fill(hidden[:, None], -math.inf)
            lse[at:at + t, head * group:(head + 1) * group] = torch.logsumexp(score, -1)
            out[at:at + t, head * group:(head + 1) * group] = (
                torch.softmax(score, -1).reshape(-1, length) @ values).reshape(t, group, dim)
        at += t
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def _exact_append(s):
    case = s["case"]
    past, count = _lengths(case)
    dim, kv = case["dim"], case["kv_heads"]
    limit = max(p + t for p, t in zip(past, count))
    cos, sin = s["cos"][:limit].double(), s["sin"][:limit].double()

    def turned(x, weight):
        x = x.double()
        if weight is not None:
            x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
        z = (x.unflatten(-1, (2, dim // 2)).transpose(-1, -2) if case["pairs"] == "halves"
             else x.unflatten(-1, (dim // 2, 2)))
        z = torch.view_as_complex(z.contiguous()) * torch.complex(cos, sin)[s["position"]][:, None]
        z = torch.view_as_real(z)
        return z.transpose(-1, -2).flatten(-2) if case["pairs"] == "halves" else z.flatten(-2)

    got = {"q": turned(s["q"], s["q_norm"])}
    for which, name, x in ((0, "k", turned(s["k"], s["k_norm"])), (1, "v", s["v"].double())):
        token, number = _code_places(dim)[which]
        parts, at = [], 0
        for i, (p, t) in enumerate(zip(past, count)):
            first, length = p // BLOCK * BLOCK, p + t
            scale = torch.zeros((length - first, kv), dtype=torch.float64, device=DEV)
            code = torch.zeros((length - first, kv, dim), dtype=torch.float64, device=DEV)
            held = p - first
            if held:
                o = s["open"][i, p // BLOCK % 2].double()
                old = torch.zeros((BLOCK, kv, dim), dtype=torch.float64, device=DEV)
                old[token, :, number] = (256 * o[:, 2 * which] + o[:, 2 * which + 1]).T
                code[:held] = old[:held]
                scale[:held] = s["open_scales"][i, p // BLOCK % 2, :, which, :held].double().T
            new = x[at:at + t]
            scale[held:] = new.abs().amax(-1) / CODE16
            code[held:] = torch.round(new / scale[held:][..., None])
            value = code * scale[..., None]
            whole = (length - first) // BLOCK * BLOCK
            if whole:
                step = scale[:whole].reshape(-1, BLOCK, kv).amax(1).repeat_interleave(BLOCK, 0)[..., None] * 256
                value[:whole] = torch.round(value[:whole] / step) * step
            parts.append(value)
            at += t
        got[name] = torch.cat(parts)
    return got


def _exact_norm(s):
    def rms(x, weight):
        return x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()

    y = s["y"].double()
    if s["post"] is not None:
        y = rms(y, s["post"])
    if s["gate"] is not None:
        y = y * s["gate"].double()
    h = s["residual"].double() + y / 2
    return {"h": h, "n": rms(h, s["norm"])}


def exact(case, seed):
    state = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "norm": _exact_norm}[case["kind"]](state)
