"""The operators for several continuations of a sequence together: in
examples/decoder.py against the model in 64 bits, and in captured graphs that
share their stream's scratch."""
import numpy as np
import pytest
import torch

from test_gpu_decoder_example import model_and_reference, reference_logits  # noqa: F401

pytestmark = pytest.mark.gpu


def rms(x):
    return float(np.sqrt(np.mean(np.square(x))))


def ids(vocab, n, seed):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


PARENTS = [-1, 0, 0, 1, 1, 2, 5, -1]


def path_to(i, parents):
    path = []
    while i >= 0:
        path.insert(0, i)
        i = parents[i]
    return path


@pytest.mark.parametrize("past", [0, 5, 61, 64, 77])
def test_logits_of_drafts_are_the_model_s(cuda, model_and_reference, past):  # noqa: F811
    """A tree of eight drafts: each one's logits are those of a sequence that
    ends with its path, up to 3% of their rms where a full block is cached
    (8-bit codes; see test_prompt_and_decoding_agree_with_the_model)."""
    decoder, shape = model_and_reference
    model = decoder.Decoder(shape, 128)
    tokens, drafted = ids(shape.vocab, past, 11), ids(shape.vocab, 8, 12)
    if past:
        model.prompt(tokens)
    logits, drafts = model.verify(drafted, PARENTS)
    got = logits.cpu().double().numpy()
    for i in range(8):
        want = reference_logits(model, shape, tokens + [drafted[j] for j in path_to(i, PARENTS)])[-1]
        assert rms(got[i] - want) <= 0.03 * rms(want), i
    # A path of it appended, and decoding on.
    path = path_to(6, PARENTS)
    model.accept(drafts, path)
    tokens = tokens + [drafted[j] for j in path]
    assert model.length == int(model.past) == len(tokens)
    got = model.prompt([3]).cpu().double().numpy()
    want = reference_logits(model, shape, tokens + [3])[-1]
    assert rms(got - want) <= 0.03 * rms(want)
    assert sum(c.faults() for c in model.caches) == 0


def test_an_accepted_path_is_what_appending_it_gives(cuda, model_and_reference):  # noqa: F811
    """60 tokens, then four drafts of a tree accepted, or appended in a step:
    the open block becomes a full one.  The drafts see each other in fp32, the
    appended tokens as codes of 16 bits, 1 / 65024 of a token's largest off at
    most; that and the products' order move later layers' numbers by less than
    1e-3 of a token's largest, 127e-3 of a step between codes (see
    test_full_blocks_hold_the_same_numbers)."""
    decoder, shape = model_and_reference
    a, b = decoder.Decoder(shape, 128), decoder.Decoder(shape, 128)
    tokens, drafted = ids(shape.vocab, 60, 13), ids(shape.vocab, 8, 14)
    a.prompt(tokens), b.prompt(tokens)
    _, drafts = a.verify(drafted, PARENTS)
    path = path_to(6, PARENTS)
    a.accept(drafts, path)
    b.prompt([drafted[i] for i in path])
    for x, y in zip(a.caches, b.caches):
        assert x.faults() == 0 and y.faults() == 0
        scale = y.scales[:1]
        assert ((x.scales[:1] - scale).abs() <= 1e-3 * scale).all()
        off = (x.pages[:1].int() - y.pages[:1].int()).abs()
        assert off.max() <= 1 and (off > 0).float().mean() <= 0.127


def test_speculation_chooses_the_best_tokens(cuda, model_and_reference):  # noqa: F811
    """Guesses right and wrong: each token is a best one in 64 bits, up to the
    logits' own error, and every right guess saves a step."""
    decoder, shape = model_and_reference
    tokens = ids(shape.vocab, 50, 15)
    plain = decoder.Decoder(shape, 128)
    known, _ = plain.decode(plain.prompt(tokens), 30)

    def guess(history):
        at = len(history) - len(tokens)
        chain = known[at:at + 3]
        wrong = [(t + 1) % shape.vocab for t in chain]  # a sibling before each right one
        out, parents, up = [], [], 0
        for w, t in zip(wrong, chain):
            out += [w, t]
            parents += [up, up]
            up = len(out)
        return out, parents

    model = decoder.Decoder(shape, 128)
    chosen, steps = model.speculate(tokens, model.prompt(tokens), 30, guess)
    assert len(chosen) == 30 and model.length == int(model.past) == 80 and sum(c.faults() for c in model.caches) == 0
    every = reference_logits(model, shape, tokens + chosen)
    for i, t in enumerate(chosen):
        row = every[len(tokens) - 1 + i]
        assert row[t] >= row.max() - 0.15 * rms(row), i
    # The steps that these tokens take with these guesses.
    done = want = 0
    while done < 30:
        at = tokens + chosen[:done + 1]
        out, parents = guess(at)
        most, node, took = min(8, 30 - done), 0, 1
        while True:
            follow = [i + 1 for i, p in enumerate(parents) if p == node and i + 1 < most and done + took < 30
                      and out[i] == chosen[done + took]]
            if not follow:
                break
            node, took = follow[0], took + 1
        done, want = done + took, want + 1
    assert steps == want < 30
    # The program's own guesses.
    model = decoder.Decoder(shape, 128)
    again, steps = model.speculate(tokens, model.prompt(tokens), 30)
    assert len(again) == 30 and 1 <= steps <= 30
    every = reference_logits(model, shape, tokens + again)
    for i, t in enumerate(again):
        row = every[len(tokens) - 1 + i]
        assert row[t] >= row.max() - 0.15 * rms(row), i


def test_guesses_are_a_tree(model_and_reference):  # noqa: F811
    decoder, _ = model_and_reference
    assert decoder.lookup([1]) == ([], [])
    assert decoder.lookup([7, 1, 2, 7, 1, 3, 7]) == ([1, 3, 7, 2, 7], [0, 1, 2, 1, 4])
    tokens, parents = decoder.lookup([5, 1, 5, 2, 5, 3, 5], most=4)
    assert len(tokens) == 4 and all(0 <= p <= i for i, p in enumerate(parents))


@pytest.mark.parametrize("beams", [2, 4, 8])
def test_a_search_keeps_the_best_beams(cuda, model_and_reference, beams):  # noqa: F811
    """A prompt of 61 tokens and up to six more, over the end of a block, each
    length searched anew.  The beams of one length are the best continuations of
    those of the length before, by scores of plain prompts: the logits of the
    two forms differ by less than 1e-3 of their rms on average (see
    test_full_blocks_hold_the_same_numbers), by 5e-3 at most, and a
    log-probability by twice that."""
    decoder, shape = model_and_reference
    tokens = ids(shape.vocab, 61, 16)

    def plain(continuation):
        model = decoder.Decoder(shape, 128)
        row = model.prompt(tokens + continuation).cpu().double().numpy()
        return row - np.logaddexp.reduce(row), 0.01 * rms(row)

    last, last_scores = [[]], [0.0]
    for count in range(1, 7):
        model = decoder.Decoder(shape, 128, beams=beams)
        found, scores, logits = model.search(model.prompt(tokens), count)
        assert sum(c.faults() for c in model.caches) == 0 and len({tuple(f) for f in found}) == beams
        assert scores == sorted(scores, reverse=True) and all(len(f) == count for f in found)
        rows = [plain(f) for f in last]
        tol = sum(r[1] for r in rows) / len(rows) * count
        total = np.stack([s + r[0] for s, r in zip(last_scores, rows)])
        cut = np.sort(total.reshape(-1))[-beams]
        for f, s in zip(found, scores):
            at = total[last.index(f[:-1]), f[-1]]
            assert abs(s - at) <= tol and at >= cut - tol, (count, f)
        # The best one goes on as a sequence of its own.
        want, off = plain(found[0])
        got = logits.cpu().double().numpy()
        assert np.abs(got - np.logaddexp.reduce(got) - want).max() <= off
        assert model.length == int(model.past) == 61 + count
        last, last_scores = found, scores
    on, _ = model.decode(logits, 30)  # into pages that the search gave back
    assert sum(c.faults() for c in model.caches) == 0
    every = reference_logits(model, shape, tokens + last[0] + on)
    for i, t in enumerate(on):
        row = every[len(tokens) + 6 - 1 + i]
        assert row[t] >= row.max() - 0.15 * rms(row), i


def test_refusals(cuda, model_and_reference):  # noqa: F811
    decoder, shape = model_and_reference
    model = decoder.Decoder(shape, 64)
    logits = model.prompt([1, 2])
    with pytest.raises(ValueError):
        model.search(logits, 3)
    with pytest.raises(ValueError):
        model.speculate([1, 2], logits, 63)
    with pytest.raises(ValueError):
        decoder.Decoder(shape, 64, beams=2).search(logits, 65)


def test_graphs_that_share_scratch(cuda):
    """A tree's attention split over workgroups, a choice and a fork, captured
    on one stream in graphs of their own, replayed in turn with new inputs:
    each replay gives what the eager calls give, bit for bit."""
    from q4rdna import api
    torch.manual_seed(17)
    heads, group, dim, past0, most = 2, 4, 128, 1500, 12
    pages = 3 * 32
    caches = [api.KVCache.empty(pages, 3, heads, dim) for _ in range(2)]
    table = torch.arange(pages, dtype=torch.int32, device="cuda").view(3, 32).contiguous()
    past = torch.zeros(3, dtype=torch.int32, device="cuda")
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, past0, past0 + 70, past0 + 70], dtype=torch.int32, device="cuda")
    for c in caches:
        k, v = torch.randn(2, past0 + 70, heads, dim, device="cuda")
        c.append(api.KVBatch(past, table, cu_tokens=cu, slots=slots, max_tokens=past0), k, v)
    past += cu.diff()
    step_cu = torch.tensor([0, most, most + 4, most + 5], dtype=torch.int32, device="cuda")
    step = api.KVBatch(past, table, cu_tokens=step_cu, slots=slots, max_tokens=most)
    n = most + 5
    parents = torch.zeros(n, dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn(n, h, dim, device="cuda") for h in (heads * group, heads, heads))
    logits = torch.randn(1, 3, 30011, device="cuda")
    scores = torch.randn(1, 3, device="cuda")
    renamed = torch.zeros(3, dtype=torch.int32, device="cuda")

    def attend():
        positions, seen = api.tree(step, parents)
        return positions, seen, *caches[0].attend_tree(step, q, k, v, seen, lse=True)

    def choose():
        return api.beam_select(logits, scores, 6)

    def fork():
        step.fork(renamed, caches, room=3)

    state = [past, table, slots, *(t for c in caches for t in (c.open, c.open_scales))]

    def forked():
        """fork's results, and the state as it was."""
        before = [t.clone() for t in state]
        renamed_graph.replay()
        a = [t.clone() for t in state]
        for t, b in zip(state, before):
            t.copy_(b)
        fork()
        b = [t.clone() for t in state]
        for t, x in zip(state, before):
            t.copy_(x)
        return a, b

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    keep = [t.clone() for t in state]
    with torch.cuda.stream(stream):
        attend(), choose(), fork()
    torch.cuda.synchronize()
    for t, b in zip(state, keep):
        t.copy_(b)
    graphs, outs = [], []
    for f in (attend, choose, fork):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(f())
        graphs.append(g)
    renamed_graph = graphs[2]
    for turn in range(4):
        gen = torch.Generator().manual_seed(100 + turn)
        up = [torch.randint(-1, j, (1,), generator=gen).item() if j else -1 for c in (most, 4, 1) for j in range(c)]
        parents.copy_(torch.tensor(up, dtype=torch.int32))
        q.normal_(), k.normal_(), v.normal_(), logits.normal_(), scores.normal_()
        renamed.copy_(torch.tensor([[0, 0, 1], [1, 0, -1], [2, 1, 0], [1, 1, 1]][turn], dtype=torch.int32))
        for i in ((0, 1), (1, 0))[turn % 2]:
            graphs[i].replay()
        torch.cuda.synchronize()
        for a, b in zip(outs[0], attend()):
            assert torch.equal(a, b), turn
        for a, b in zip(outs[1], choose()):
            assert torch.equal(a, b), turn
        for a, b in zip(*forked()):
            assert torch.equal(a, b), turn
    assert sum(c.faults() for c in caches) == 0


def test_nothing_to_do(cuda):
    """No tokens, no sequences, a sequence without drafts: outputs of no rows, and
    rows of the others."""
    from q4rdna import api
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = api.KVCache.empty(4, 2, 2, 64)
    table, slots = ints([[0, 1], [2, 3]]), ints([0, 1])
    batch = api.KVBatch(ints([0, 0]), table, cu_tokens=ints([0, 0, 0]), slots=slots, max_tokens=4)
    positions, seen = api.tree(batch, ints([]))
    assert positions.shape == seen.shape == (0,)
    rows = lambda n, h: torch.randn(n, h, 64, device="cuda")  # noqa: E731
    out, lse = cache.attend_tree(batch, rows(0, 4), rows(0, 2), rows(0, 2), seen, lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    nobody = api.KVBatch(ints([]), torch.zeros((0, 2), dtype=torch.int32, device="cuda"), cu_tokens=ints([0]), slots=ints([]), max_tokens=4)
    nobody.fork(ints([]), [cache])
    assert api.tree(nobody, ints([]))[0].shape == (0,)
    # One draft of the second sequence, none of the first, nothing cached: it sees itself.
    one = api.KVBatch(ints([0, 0]), table, cu_tokens=ints([0, 0, 1]), slots=slots, max_tokens=4)
    v = rows(1, 2)
    positions, seen = api.tree(one, ints([-1]))
    out = cache.attend_tree(one, rows(1, 4), rows(1, 2), v, seen)
    assert positions.tolist() == [0] and seen.tolist() == [1]
    # Two fp16 parts of a number and fp32 products: 2^-21 of the row's largest at most.
    assert (out - v.repeat_interleave(2, dim=1)).abs().max() <= 2.0 ** -21 * v.abs().max()
    assert cache.faults() == 0


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device_than_the_current_one(cuda):
    from q4rdna import api
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda:1")  # noqa: E731
    torch.manual_seed(0)
    cache = api.KVCache.empty(8, 2, 2, 64, device=1)
    past, table, slots = ints([0, 0]), ints([[0, 1, 2], [3, 4, 5]]), ints([0, 1])
    k, q = torch.randn((140, 2, 64), device="cuda:1"), torch.randn((5, 4, 64), device="cuda:1")
    cache.append(api.KVBatch(past, table, ints([0, 70, 140]), slots, max_tokens=70), k, k)
    past += 70
    step = api.KVBatch(past, table, ints([0, 2, 5]), slots, max_tokens=3)
    parents, logits = ints([-1, 0, -1, 0, 0]), torch.randn((1, 2, 999), device="cuda:1")
    results = []
    for current in (1, 0):
        with torch.cuda.device(current):
            positions, seen = api.tree(step, parents)
            q1, k1 = api.rotate(q, k[:5], positions)
            results.append((positions, seen, q1, k1, cache.attend_tree(step, q1, k1, k[:5], seen), *api.beam_select(logits, None, 4)))
            assert torch.cuda.current_device() == current
    assert all(torch.equal(a, b) for a, b in zip(*results))
    step.fork(ints([1, 1]), [cache])
    assert torch.cuda.current_device() == 0 and past.tolist() == [70, 70]


def test_offsets_past_32_bits(cuda):
    """Pages and slots more than 4 GiB into a cache: the same bits as in a small
    one, from drafts and after a fork."""
    from q4rdna import api
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    torch.manual_seed(1)
    heads, dim, length = 8, 128, 200
    k, v = torch.randn(2, length, heads, dim, device="cuda")
    q, dk, dv = (torch.randn(3, h, dim, device="cuda") for h in (2 * heads, heads, heads))
    results = []
    for pages, slots in ((12, 2), (34000, 8300)):
        cache = api.KVCache.empty(pages, slots, heads, dim)
        if slots > 2:
            assert cache.pages.numel() > 2 ** 32 and cache.open.numel() > 2 ** 32
        table = ints([list(range(pages - 4, pages)), [-1] * 4])
        past, slot = ints([0, 0]), ints([slots - 1, 0])
        cache.append(api.KVBatch(past, table, ints([0, length, length]), slot, max_tokens=length), k, v)
        past[0] = length
        step = api.KVBatch(past, table, ints([0, 3, 3]), slot, max_tokens=3)
        _, seen = api.tree(step, ints([-1, 0, 0]))
        out = [cache.attend_tree(step, q, dk, dv, seen)]
        step.fork(ints([0, 0]), [cache])
        assert slot.tolist() == [slots - 1, 0] and past.tolist() == [length, length]
        # The second goes on from the copy of its open block.
        step = api.KVBatch(past, table, ints([0, 0, 3]), slot, max_tokens=3)
        out.append(cache.attend_tree(step, q, dk, dv, seen))
        assert torch.equal(out[0], out[1]) and cache.faults() == 0
        results.append(out)
        del cache
    assert all(torch.equal(a, b) for a, b in zip(*results))
