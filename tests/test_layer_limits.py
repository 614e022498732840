"""Steps with more workgroups than a launch may have (2^32 threads) are refused
as arguments, before any device call."""
import ctypes

import q4rdna
from q4rdna import _lib
from test_layer_refusals import P, append, attend, batch, cache, refused, rows

MANY = dict(sequences=65535, tokens=65535)


def test_too_many_workgroups():
    L = q4rdna.load()
    # 65535 sequences of 1024 heads: 2^26 workgroups of 256 threads
    c, b = ctypes.byref(cache(kv_heads=1024)), ctypes.byref(batch(**MANY))
    refused(L.q4rdna_kv_append(c, b, ctypes.byref(append(q_heads=0)), None), "too many")
    refused(L.q4rdna_kv_attend(c, b, ctypes.byref(attend(q_heads=1024)), None), "too many")
    refused(L.q4rdna_kv_read(c, b, _lib.F32, ctypes.byref(rows()), ctypes.byref(rows()), None), "too many")
    # q alone: 2^30 - 1 tokens of 32768 heads
    c = ctypes.byref(cache(kv_heads=1))
    b = ctypes.byref(batch(sequences=1, tokens=2 ** 30 - 1, max_tokens=2 ** 30 - 1, cu_tokens=P))
    refused(L.q4rdna_kv_append(c, b, ctypes.byref(append(q_heads=32768)), None), "too many")
    # long prompts of a group of 32 query heads: 2^28 row groups of 128
    b = ctypes.byref(batch(sequences=1, tokens=2 ** 24, max_tokens=2 ** 24, cu_tokens=P, table_width=2 ** 20))
    c = ctypes.byref(cache(kv_heads=1024))
    refused(L.q4rdna_kv_attend(c, b, ctypes.byref(attend(q_heads=32768)), None), "too many")
