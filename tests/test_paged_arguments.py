"""Paged K/V cache operators: arguments that no kernel may get, refused on the
host before any CUDA call (no GPU)."""
import ctypes
import random

import pytest

from helpers import abi, lfm3

P = 0x10000  # never dereferenced
INVALID = -1


def cache(**over):
    d = dict(k=P, v=P, table=P, lengths=P, pages=10, page_rows=16, kv_heads=2,
             dim=64, sequences=2, table_pages=4, table_stride=4)
    return abi.PagedCache(**{**d, **over})


def batch(**over):
    return abi.PagedBatch(**{**dict(starts=P, positions=None, rows=4, max_rows=4),
                             **over})


def heads(c=None, b=None, kind=0, q=P, qs=256, k=4 * P, ks=128, v=5 * P, vs=128,
          o=2 * P, os=256, qn=P, kn=P, freq=P, fac=None):
    return lfm3.library().lfm3_cuda_paged_heads(
        ctypes.byref(c or cache()), ctypes.byref(b or batch()), kind, q, qs, k,
        ks, v, vs, o, os, 4, qn, kn, freq, fac, 1e-5, None)


def attention(c=None, b=None, kind=0, q=P, qs=256, gate=None, o=2 * P, os=256,
              lse=None):
    return lfm3.library().lfm3_cuda_paged_attention(
        ctypes.byref(c or cache()), ctypes.byref(b or batch()), kind, q, qs, gate,
        4, o, os, lse, 4, 0, P, 1 << 40, None)


def weights(c=None, b=None, lse=P, w=P):
    return lfm3.library().lfm3_cuda_paged_key_weights(
        ctypes.byref(c or cache()), ctypes.byref(b or batch()), 0, P, 256, lse, w,
        4, 0, P, 1 << 40, None)


def evict(c=None, out_table=P, out_lengths=P, w=P, kept=P):
    return lfm3.library().lfm3_cuda_paged_evict(
        ctypes.byref(c or cache()), out_table, out_lengths, w, kept, 8, 2, None)


def refused(code, text):
    message = lfm3.library().lfm3_last_error()
    return code == INVALID and text in message


@pytest.mark.parametrize("name", ["table", "lengths"])
def test_misaligned_tables(name):
    c = cache(**{name: P + 2})
    for call in (heads, attention, weights, evict):
        assert refused(call(c), b"table or lengths are not aligned")


def test_misaligned_batch():
    for call in (heads, attention, weights):
        assert refused(call(b=batch(starts=P + 1)), b"starts are not aligned")
    # heads alone read positions
    assert refused(heads(b=batch(positions=P + 1)), b"are not aligned")
    for call in (attention, weights):
        assert not refused(call(b=batch(positions=P + 1)), b"aligned")


def test_misaligned_arrays():
    for name in ("qn", "kn", "freq", "fac"):
        assert refused(heads(**{name: P + 2}), b"are not aligned")
    assert refused(attention(lse=P + 2), b"gate or lse")
    assert refused(attention(gate=P + 2), b"gate or lse")        # FP32
    assert refused(attention(kind=1, gate=P + 1), b"gate or lse")
    for name in ("lse", "w"):
        assert refused(weights(**{name: P + 2}), b"lse or weights")
    for name in ("out_table", "out_lengths", "w", "kept"):
        assert refused(evict(**{name: P + 3}), b"an array is not aligned")


def overlap(a, sa, wa, b, sb, wb, rows):
    """Whether row i of a and row j of b share a byte, for some i and j < rows."""
    return any(a + i * sa < b + j * sb + wb and b + j * sb < a + i * sa + wa
               for i in range(rows) for j in range(rows))


def test_overlapping_rows_are_refused():
    """Exactly the calls whose rows overlap: columns of one buffer are fine."""
    rng = random.Random(0)
    base, text = 1 << 32, b"overlaps"
    seen = [0, 0]
    for _ in range(3000):
        rows = rng.choice([1, 2, 3, 7, 12])
        kind, size = rng.choice([(0, 4), (1, 2), (30, 2)])
        width = 4 * 64 * size
        sq = rng.choice([256, 264, 512, 768, 1024])
        so = rng.choice([sq, sq, 256, 328, 600, 2048])
        q = base + 16 * rng.randint(0, 40)
        o = q + 16 * rng.choice([rng.randint(-400, 400), rng.randint(-9000, 9000)])
        if o == q:
            continue
        want = overlap(q, sq * size, width, o, so * size, width, rows)
        seen[want] += 1
        b = batch(rows=rows)
        far = dict(k=1 << 40, v=1 << 41)
        for call in (lambda: attention(b=b, kind=kind, q=q, qs=sq, o=o, os=so),
                     lambda: heads(b=b, kind=kind, q=q, qs=sq, o=o, os=so, **far)):
            code = call()
            # calls that are not refused end at the first CUDA call here, or at
            # the pointers that are not the device's
            assert (code == INVALID and
                    text in lfm3.library().lfm3_last_error()) == want, (
                        rows, kind, sq, so, o - q)
            assert code != 0
    assert min(seen) > 300
    # keys and values, and a fused buffer [q k v] worked on in place
    q, row = base, (256 + 128 + 128)
    fused = dict(q=q, qs=row, k=q + 1024, ks=row, v=q + 1536, vs=row, os=row)
    assert not refused(heads(o=q, **fused), text)
    assert refused(heads(o=q + 1024, **fused), text)
    assert refused(heads(o=q + 512, **fused), text)
    assert refused(heads(**{**fused, "q": 1 << 40, "o": q + 1280}), text)
