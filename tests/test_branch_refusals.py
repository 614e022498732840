"""What the entry points for several continuations refuse, before any device call."""
import ctypes

import pytest

import q4rdna
from q4rdna import _lib
from test_layer_refusals import BATCHES, CACHES, P, batch, cache, refused, rows


def rotate(**changes):
    d = _lib.RotateDesc()
    d.tokens, d.q_heads, d.k_heads, d.head_dim = 3, 4, 2, 64
    d.q = d.k = d.q_out = d.k_out = rows()
    d.position, d.cos, d.sin, d.positions, d.rotary = P, P, P, 8, 64
    for name, value in changes.items():
        setattr(d, name, value)
    return d


def tree(**changes):
    d = _lib.TreeDesc()
    d.q_heads, d.scale, d.seen = 4, 0.125, P
    d.q = d.k = d.v = d.out = rows()
    for name, value in changes.items():
        setattr(d, name, value)
    return d


def beam(**changes):
    d = _lib.BeamDesc()
    d.groups, d.beams, d.vocab, d.count = 2, 3, 50, 4
    d.group_stride, d.beam_stride = 150, 50
    d.logits = d.scores = d.out_scores = d.out_rows = d.out_tokens = P
    for name, value in changes.items():
        setattr(d, name, value)
    return d


def fork(**changes):
    d = _lib.ForkDesc()
    d.parents = d.past = d.table = d.slots = P
    d.sequences, d.table_width, d.room = 2, 4, 1
    for name, value in changes.items():
        setattr(d, name, value)
    return d


def caches(*changes):
    return (_lib.CacheDesc * len(changes))(*[cache(**dict(dict(open=P + 4096 * i, open_scales=P + 65536 + 4096 * i), **c))
                                             for i, c in enumerate(changes)])


def test_tree_arguments():
    L = q4rdna.load()
    go = lambda b, *at: L.q4rdna_kv_tree(ctypes.byref(b) if b else None, *at, None)  # noqa: E731
    refused(go(None, P, P, P), "null batch")
    for changes, word in BATCHES:
        refused(go(batch(**changes), P, P, P), word)
    refused(go(batch(cu_tokens=P, max_tokens=65), P, P, P), "max_tokens")
    for at in ((None, P, P), (P, None, P), (P, P, None)):
        refused(go(batch(), *at), "null parents")
    for at in ((P + 2, P, P), (P, P + 1, P), (P, P, P + 4)):
        refused(go(batch(), *at), "misaligned")
    assert go(batch(tokens=0, cu_tokens=P), None, None, None) == q4rdna.OK


def test_rotate_arguments():
    L = q4rdna.load()
    go = lambda **c: L.q4rdna_rotate(ctypes.byref(rotate(**c)), None)  # noqa: E731
    refused(L.q4rdna_rotate(None, None), "null descriptor")
    for changes, word in [(dict(dtype=3), "dtype"), (dict(head_dim=96), "head_dim"), (dict(reserved=1), "reserved"),
                          (dict(q_heads=32767), "heads"), (dict(tokens=2 ** 31), "tokens"), (dict(q=rows(None)), "null q"),
                          (dict(q_out=rows(P + 2)), "misaligned q_out"), (dict(k=rows(P + 1)), "misaligned k"),
                          (dict(k_out=rows(None)), "null k_out"), (dict(rotary=12), "rotary"), (dict(rotary=72), "rotary"),
                          (dict(cos=None), "cos"), (dict(sin=P + 8), "sin"), (dict(positions=0), "cos"),
                          (dict(position=None), "position"), (dict(position=P + 2), "position"), (dict(q_norm=P + 4), "norm"),
                          (dict(k_norm=P + 8), "norm")]:
        refused(go(**changes), word)
    assert go(tokens=0) == q4rdna.OK and go(q_heads=0, k_heads=0, q=rows(None)) == q4rdna.OK


def test_attend_tree_arguments():
    L = q4rdna.load()

    def go(c=cache(), b=batch(), **changes):
        return L.q4rdna_kv_attend_tree(ctypes.byref(c) if c else None, ctypes.byref(b) if b else None,
                                       ctypes.byref(tree(**changes)), None)

    refused(go(c=None), "null cache")
    refused(go(b=None), "null batch")
    for changes, word in CACHES:
        refused(go(c=cache(**changes)), word)
    for changes, word in BATCHES:
        refused(go(b=batch(**changes)), word)
    refused(go(b=batch(cu_tokens=P, max_tokens=65)), "max_tokens")
    refused(L.q4rdna_kv_attend_tree(ctypes.byref(cache()), ctypes.byref(batch()), None, None), "null descriptor")
    for changes, word in [(dict(dtype=7), "dtype"), (dict(q=rows(None)), "null q"), (dict(k=rows(None)), "null k"),
                          (dict(v=rows(P + 2)), "misaligned v"), (dict(out=rows(None)), "null out"), (dict(q_heads=0), "query heads"),
                          (dict(q_heads=5), "query heads"), (dict(scale=float("nan")), "scale"), (dict(scale=-1.0), "scale"),
                          (dict(seen=None), "seen"), (dict(seen=P + 4), "seen"), (dict(lse=P + 2), "lse")]:
        refused(go(**changes), word)
    assert go(b=batch(tokens=0, cu_tokens=P)) == q4rdna.OK
    many = batch(sequences=65535, tokens=65535)
    refused(go(c=cache(kv_heads=1024), b=many, q_heads=1024), "too many")


def test_beam_arguments():
    L = q4rdna.load()
    go = lambda **c: L.q4rdna_beam_select(ctypes.byref(beam(**c)), None)  # noqa: E731
    refused(L.q4rdna_beam_select(None, None), "null descriptor")
    for changes, word in [(dict(dtype=3), "dtype"), (dict(reserved=1), "reserved"), (dict(beams=0), "beams"),
                          (dict(beams=257), "beams"), (dict(vocab=0), "tokens"), (dict(vocab=2 ** 24 + 1), "tokens"),
                          (dict(groups=2 ** 31), "groups"), (dict(count=0), "count"), (dict(count=129), "count"),
                          (dict(vocab=1, beams=3, count=4), "count"), (dict(logits=None), "null"), (dict(out_scores=None), "null"),
                          (dict(out_rows=None), "null"), (dict(out_tokens=None), "null"), (dict(logits=P + 2), "misaligned"),
                          (dict(scores=P + 2), "misaligned"), (dict(out_tokens=P + 1), "misaligned")]:
        refused(go(**changes), word)
    assert go(groups=0) == q4rdna.OK


def test_fork_arguments():
    L = q4rdna.load()
    go = lambda c=caches({}, {}), n=2, **d: L.q4rdna_kv_fork(c, n, ctypes.byref(fork(**d)), None)  # noqa: E731
    refused(go(c=None), "no caches")
    refused(go(n=0), "no caches")
    refused(L.q4rdna_kv_fork(caches({}), 1, None, None), "null descriptor")
    for changes, word in CACHES:
        if "faults" not in changes:
            refused(go(c=caches({}, changes)), word)
    for changes in (dict(kv_heads=3), dict(head_dim=128), dict(page_count=5), dict(slot_count=3), dict(device=1)):
        refused(go(c=caches({}, changes)), "geometry")
    refused(go(c=caches({}, dict(open=P))), "share")
    refused(go(c=caches({}, dict(open_scales=P + 65536))), "share")
    refused(go(c=caches(dict(page_count=2 ** 18 + 1), dict(page_count=2 ** 18 + 1))), "pages")
    for changes, word in [(dict(reserved=1), "reserved"), (dict(sequences=4097), "sequences"), (dict(table_width=0), "columns"),
                          (dict(table_width=2 ** 24 + 1), "columns"), (dict(parents=None), "null"), (dict(past=None), "null"),
                          (dict(table=None), "null"), (dict(slots=None), "null"), (dict(parents=P + 1), "misaligned"),
                          (dict(slots=P + 2), "misaligned")]:
        refused(go(**changes), word)
    assert go(sequences=0) == q4rdna.OK


def test_structures_have_the_header_s_layout():
    assert ctypes.sizeof(_lib.RotateDesc) == 176 and ctypes.sizeof(_lib.TreeDesc) == 128
    assert ctypes.sizeof(_lib.BeamDesc) == 80 and ctypes.sizeof(_lib.ForkDesc) == 56
    for packer, structure in ((_lib.ROTATE, _lib.RotateDesc), (_lib.TREE, _lib.TreeDesc), (_lib.BEAM, _lib.BeamDesc),
                              (_lib.FORK, _lib.ForkDesc)):
        assert packer.size == ctypes.sizeof(structure)


def test_tensors_on_the_host():
    """The Python calls look at their tensors before anything else."""
    import torch
    from q4rdna import api
    x = torch.zeros((2, 4, 64))
    with pytest.raises(ValueError):
        api.rotate(x, None, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        api.rotate(None, None, None)
    with pytest.raises(ValueError):
        api.beam_select(x, None, 1)
