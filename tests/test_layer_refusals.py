"""What the decoder-layer entry points refuse, before any device call."""
import ctypes

import pytest

import q4rdna
from q4rdna import _lib

P = 1 << 20  # an aligned address that is never followed


def cache(**changes):
    c = _lib.CacheDesc()
    c.pages = c.scales = c.open = c.open_scales = P
    c.page_count, c.slot_count, c.kv_heads, c.head_dim, c.device = 4, 2, 2, 64, 0
    for name, value in changes.items():
        setattr(c, name, value)
    return c


def batch(**changes):
    b = _lib.BatchDesc()
    b.past = b.table = P
    b.sequences = b.tokens = 2
    b.max_tokens, b.table_width = 1, 4
    for name, value in changes.items():
        setattr(b, name, value)
    return b


def rows(address=P):
    return _lib.Rows(address, 64, 64)


def append(**changes):
    d = _lib.AppendDesc()
    d.k = d.v = d.q = d.q_out = rows()
    d.q_heads, d.cos, d.sin, d.positions, d.rotary = 4, P, P, 8, 64
    for name, value in changes.items():
        setattr(d, name, value)
    return d


def attend(**changes):
    d = _lib.AttendDesc()
    d.q = d.out = rows()
    d.q_heads, d.scale = 4, 0.125
    for name, value in changes.items():
        setattr(d, name, value)
    return d


def norm(**changes):
    d = _lib.AddNormDesc()
    d.rows, d.width = 2, 64
    d.residual, d.y, d.h, d.n = P, P + 4096, P + 8192, P + 12288
    d.weight = P
    for name in ("residual", "y", "h", "n"):
        setattr(d, name + "_stride", 64)
    for name, value in changes.items():
        setattr(d, name, value)
    return d


def refused(status, word):
    assert status == q4rdna.ERR_ARGUMENT
    assert word in q4rdna.last_error(), q4rdna.last_error()


CACHES = [(dict(pages=None), "null cache"), (dict(scales=None), "null cache"), (dict(open=None), "null cache"),
          (dict(open_scales=None), "null cache"), (dict(head_dim=96), "head_dim"), (dict(head_dim=0), "head_dim"),
          (dict(kv_heads=0), "kv heads"), (dict(page_count=0), "pages"), (dict(page_count=2 ** 31), "pages"),
          (dict(slot_count=0), "slots"), (dict(pages=P + 8), "misaligned"), (dict(scales=P + 4), "misaligned"),
          (dict(open=P + 1), "misaligned"), (dict(open_scales=P + 8), "misaligned"), (dict(faults=P + 2), "misaligned")]
BATCHES = [(dict(past=None), "null past"), (dict(table=None), "null past or table"), (dict(past=P + 1), "misaligned"),
           (dict(cu_tokens=P + 2), "misaligned"), (dict(slots=P + 3), "misaligned"), (dict(table_width=0), "table columns"),
           (dict(table_width=2 ** 24 + 1), "table columns"), (dict(sequences=65536, tokens=65536), "sequences"),
           (dict(max_tokens=0), "tokens"), (dict(tokens=3), "without cu_tokens"), (dict(max_tokens=2), "without cu_tokens")]


@pytest.mark.parametrize("call", ["append", "attend", "read"])
def test_caches_and_batches(call):
    L = q4rdna.load()

    def go(c, b):
        c, b = ctypes.byref(c) if c else None, ctypes.byref(b) if b else None
        if call == "append":
            return L.q4rdna_kv_append(c, b, ctypes.byref(append()), None)
        if call == "attend":
            return L.q4rdna_kv_attend(c, b, ctypes.byref(attend()), None)
        return L.q4rdna_kv_read(c, b, _lib.F32, ctypes.byref(rows()), ctypes.byref(rows()), None)

    refused(go(None, batch()), "null cache")
    refused(go(cache(), None), "null batch")
    for changes, word in CACHES:
        refused(go(cache(**changes), batch()), word)
    for changes, word in BATCHES:
        refused(go(cache(), batch(**changes)), word)
    assert go(cache(), batch(tokens=0, cu_tokens=P)) == q4rdna.OK
    assert go(cache(), batch(sequences=0, tokens=0, past=None, table=None)) == q4rdna.OK


def test_append_arguments():
    L = q4rdna.load()
    go = lambda **c: L.q4rdna_kv_append(ctypes.byref(cache()), ctypes.byref(batch()), ctypes.byref(append(**c)), None)  # noqa: E731
    refused(L.q4rdna_kv_append(ctypes.byref(cache()), ctypes.byref(batch()), None, None), "null descriptor")
    for changes, word in [(dict(dtype=3), "dtype"), (dict(k=rows(None)), "null k"), (dict(v=rows(P + 2)), "misaligned v"),
                          (dict(q=rows(None)), "null q"), (dict(q_out=rows(None)), "null q_out"), (dict(q_heads=3), "query heads"),
                          (dict(rotary=12), "rotary"), (dict(rotary=72), "rotary"), (dict(cos=None), "cos"), (dict(sin=P + 8), "sin"),
                          (dict(q_norm=P + 4), "norm"), (dict(k_norm=P + 8), "norm")]:
        refused(go(**changes), word)


def test_attend_arguments():
    L = q4rdna.load()
    go = lambda **c: L.q4rdna_kv_attend(ctypes.byref(cache()), ctypes.byref(batch()), ctypes.byref(attend(**c)), None)  # noqa: E731
    refused(L.q4rdna_kv_attend(ctypes.byref(cache()), ctypes.byref(batch()), None, None), "null descriptor")
    for changes, word in [(dict(dtype=7), "dtype"), (dict(q=rows(None)), "null q"), (dict(out=rows(None)), "null out"),
                          (dict(q=rows(P + 1)), "misaligned q"), (dict(q_heads=0), "query heads"), (dict(q_heads=5), "query heads"),
                          (dict(scale=float("nan")), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"),
                          (dict(lse=P + 2), "lse")]:
        refused(go(**changes), word)


def test_read_arguments():
    L = q4rdna.load()
    c, b = ctypes.byref(cache()), ctypes.byref(batch())
    refused(L.q4rdna_kv_read(c, b, 9, ctypes.byref(rows()), ctypes.byref(rows()), None), "dtype")
    refused(L.q4rdna_kv_read(c, b, 0, None, ctypes.byref(rows()), None), "null rows")
    refused(L.q4rdna_kv_read(c, b, 0, ctypes.byref(rows()), ctypes.byref(rows(None)), None), "null v")


def test_norm_arguments():
    L = q4rdna.load()
    go = lambda **c: L.q4rdna_add_norm(ctypes.byref(norm(**c)), None)  # noqa: E731
    refused(L.q4rdna_add_norm(None, None), "null descriptor")
    for changes, word in [(dict(dtype=3), "dtype"), (dict(width=0), "numbers a row"), (dict(width=16385), "numbers a row"),
                          (dict(residual=None), "residual"), (dict(weight=None), "weight"), (dict(y=None, gate=P), "without y"),
                          (dict(y=None, post_weight=P), "without y"), (dict(y=P + 2), "misaligned"), (dict(weight=P + 2), "weight"),
                          (dict(h=P + 12288), "one buffer"), (dict(h=P, h_stride=128), "another stride"),
                          (dict(gate=P + 8192), "over the gate"), (dict(reserved=1), "reserved")]:
        refused(go(**changes), word)
    assert go(rows=0) == q4rdna.OK and go(h=None, n=None) == q4rdna.OK


def test_structures_have_the_header_s_layout():
    """Sizes that a C compiler gives the header's structures on this ABI."""
    assert ctypes.sizeof(_lib.CacheDesc) == 64 and ctypes.sizeof(_lib.BatchDesc) == 48 and ctypes.sizeof(_lib.Rows) == 24
    assert ctypes.sizeof(_lib.AppendDesc) == 152 and ctypes.sizeof(_lib.AttendDesc) == 72
    assert ctypes.sizeof(_lib.AddNormDesc) == 120
    for packer, structure in ((_lib.ROWS, _lib.Rows), (_lib.APPEND, _lib.AppendDesc), (_lib.ATTEND, _lib.AttendDesc),
                              (_lib.ADD_NORM, _lib.AddNormDesc)):
        assert packer.size == ctypes.sizeof(structure)
