"""Paged K/V cache operators, host side (no GPU): refusals of every entry point
come before any CUDA call, and lfm3_paged_check applies the kernels' own rules
on the tables to host copies."""
import ctypes

import numpy as np
import pytest

from helpers import abi, lfm3

P = 0x10000  # never dereferenced: the calls below are refused first
INVALID, UNSUPPORTED = -1, -3


def cache(**over):
    d = dict(k=P, v=P, table=P, lengths=P, pages=10, page_rows=16, kv_heads=2,
             dim=64, sequences=2, table_pages=4, table_stride=4)
    d.update(over)
    return abi.PagedCache(**d)


def batch(**over):
    d = dict(starts=P, positions=None, rows=4, max_rows=4)
    d.update(over)
    return abi.PagedBatch(**d)


def heads(c=None, b=None, kind=0, q=P, qs=256, k=P, ks=128, v=P, vs=128, o=P,
          os=256, h=4, freq=P, eps=1e-5):
    c, b = c or cache(), b or batch()
    return lfm3.library().lfm3_cuda_paged_heads(
        ctypes.byref(c), ctypes.byref(b), kind, q, qs, k, ks, v, vs, o, os, h,
        P, P, freq, None, eps, None)


def attention(c=None, b=None, kind=0, q=P, qs=256, gate=None, gs=0, o=2 * P,
              os=256, h=4, window=0, ws=P, size=1 << 40):
    c, b = c or cache(), b or batch()
    return lfm3.library().lfm3_cuda_paged_attention(
        ctypes.byref(c), ctypes.byref(b), kind, q, qs, gate, gs, o, os, None, h,
        window, ws, size, None)


def weights(c=None, b=None, kind=0, q=P, qs=256, lse=P, w=P, h=4, window=0,
            ws=P, size=1 << 40):
    c, b = c or cache(), b or batch()
    return lfm3.library().lfm3_cuda_paged_key_weights(
        ctypes.byref(c), ctypes.byref(b), kind, q, qs, lse, w, h, window, ws,
        size, None)


def evict(c=None, out_table=P, out_lengths=P, w=P, kept=P, keep=8, recent=2):
    c = c or cache()
    return lfm3.library().lfm3_cuda_paged_evict(
        ctypes.byref(c), out_table, out_lengths, w, kept, keep, recent, None)


@pytest.mark.parametrize("over,code", [
    (dict(dim=96), UNSUPPORTED), (dict(dim=0), UNSUPPORTED),
    (dict(kv_heads=0), UNSUPPORTED), (dict(kv_heads=-2), UNSUPPORTED),
    (dict(page_rows=0), UNSUPPORTED), (dict(page_rows=8), UNSUPPORTED),
    (dict(page_rows=40), UNSUPPORTED), (dict(page_rows=-16), UNSUPPORTED),
    (dict(sequences=-1), UNSUPPORTED), (dict(sequences=4097), UNSUPPORTED),
    (dict(pages=0), INVALID), (dict(table_pages=0), INVALID),
    (dict(table_stride=3), INVALID),
    (dict(pages=1 << 27), UNSUPPORTED),
    (dict(table_pages=1 << 27, table_stride=1 << 27), UNSUPPORTED),
    (dict(k=None), INVALID), (dict(v=None), INVALID),
    (dict(table=None), INVALID), (dict(lengths=None), INVALID),
    (dict(k=P + 8), INVALID), (dict(v=P + 2), INVALID),
])
def test_cache_refusals(over, code):
    c = cache(**over)
    assert [heads(c), attention(c), weights(c), evict(c)] == [code] * 4
    assert lfm3.library().lfm3_last_error() != b""
    lib, b = lfm3.library(), batch()
    for size in (lib.lfm3_cuda_paged_attention_workspace_bytes,
                 lib.lfm3_cuda_paged_key_weights_workspace_bytes):
        assert size(ctypes.byref(c), ctypes.byref(b), 4) == 0


@pytest.mark.parametrize("over", [dict(starts=None), dict(rows=-1),
                                  dict(max_rows=-1)])
def test_batch_refusals(over):
    b = batch(**over)
    assert [heads(b=b), attention(b=b), weights(b=b)] == [INVALID] * 3


def test_missing_descriptors():
    lib, c, b = lfm3.library(), cache(), batch()
    at, bt = ctypes.byref(c), ctypes.byref(b)
    assert lib.lfm3_paged_check(None, bt, 0) == INVALID
    assert lib.lfm3_paged_check(at, None, 1) == INVALID
    assert lib.lfm3_cuda_paged_evict(None, P, P, P, P, 8, 2, None) == INVALID
    assert lib.lfm3_cuda_paged_attention_workspace_bytes(None, bt, 4) == 0
    assert lib.lfm3_cuda_paged_key_weights_workspace_bytes(at, None, 4) == 0


@pytest.mark.parametrize("call", [heads, attention, weights])
def test_shared_refusals(call):
    for kind in (2, 8, 99):  # Q8_0 and unknown types
        assert call(kind=kind) == UNSUPPORTED
    for h in (0, -4, 3, 2 * 129):
        assert call(h=h, qs=1 << 16) == UNSUPPORTED
    assert call(q=None) == INVALID
    assert call(q=P + 8) == INVALID      # alignment
    assert call(qs=248) == INVALID       # narrower than the heads
    assert call(qs=260) == INVALID       # not a multiple of 8
    assert call(qs=1 << 50) == INVALID


def test_operator_refusals():
    assert heads(k=None) == heads(v=P + 4) == heads(ks=120) == INVALID
    assert heads(o=None) == heads(o=2 * P, os=130) == INVALID
    assert heads(freq=None) == heads(eps=float("nan")) == INVALID
    assert heads(eps=-1.0) == heads(eps=float("inf")) == INVALID
    assert heads(os=264) == INVALID      # in place at another stride
    assert attention(o=None) == attention(os=100) == INVALID
    assert attention(o=P) == INVALID      # out over q
    assert b"may not be q" in lfm3.library().lfm3_last_error()
    assert attention(window=-1) == weights(window=-1) == INVALID
    assert attention(gate=P, gs=3) == INVALID
    assert attention(ws=P + 16) == weights(ws=P + 16) == INVALID
    assert attention(size=0) == attention(ws=None) == INVALID
    assert weights(lse=None) == weights(w=None) == INVALID
    assert evict(out_table=None) == evict(w=None) == INVALID
    assert evict(out_lengths=None) == evict(kept=None) == INVALID
    assert evict(keep=0) == evict(recent=-1) == evict(recent=9) == INVALID
    assert evict(keep=65) == INVALID     # four pages of 16 rows hold 64


def test_nothing_to_do_needs_no_arrays():
    for b in (batch(rows=0), batch(max_rows=0)):
        assert heads(b=b, q=None) == attention(b=b, q=None) == 0
        assert weights(b=b, q=None) == 0
    c = cache(sequences=0)
    assert heads(c, q=None) == attention(c, q=None) == weights(c, q=None) == 0
    assert evict(c) == 0


# ---- tables ------------------------------------------------------------------------
def check(starts, lengths, table, pages=10, page_rows=16, rows=40, max_rows=40,
          table_pages=None, shared=0):
    starts = np.array(starts, np.int32)
    lengths = np.array(lengths, np.int32)
    table = np.array(table, np.int32)
    c = cache(table=table.ctypes.data, lengths=lengths.ctypes.data, pages=pages,
              page_rows=page_rows, sequences=len(lengths),
              table_pages=table_pages or table.shape[1],
              table_stride=table.shape[1])
    b = batch(starts=starts.ctypes.data, rows=rows, max_rows=max_rows)
    return lfm3.library().lfm3_paged_check(ctypes.byref(c), ctypes.byref(b),
                                           shared)


def test_sound_tables():
    # unused entries may hold anything; lengths of 0 and n > length are fine
    assert check([0, 1, 1, 21], [33, 0, 16], [[0, 1, 9], [-1, -1, -1],
                                              [4, 99, 99]]) == 0
    assert check([3, 4, 5], [0, 0], [[-1], [77]]) == 0
    assert check([0], [], np.zeros((0, 1))) == 0


def test_shared_pages():
    two = ([0, 1, 2], [33, 20], [[4, 5, 6], [4, 7, 4]])  # a common prefix
    assert check(*two, shared=1) == 0
    assert check(*two) == INVALID
    assert b"sequence 1: page of row 0 is held already" in \
        lfm3.library().lfm3_last_error()
    assert check([0, 1], [17], [[3, 3]]) == INVALID
    # entries past the rows held do not count
    assert check([0, 1, 2], [16, 16], [[4, 5], [5, 4]]) == 0


@pytest.mark.parametrize("starts,lengths,table,more", [
    ([0, 1], [17], [[3, 10]], {}),            # page id past the pool
    ([0, 1], [17], [[-1, 3]], {}),            # negative page id
    ([0, 1], [33], [[1, 2]], {}),             # longer than the table row
    ([0, 1], [33], [[1, 2, 3]], {"table_pages": 2}),
    ([0, 1], [-1], [[1, 2]], {}),             # negative length
    ([1, 0], [5], [[1, 2]], {}),              # starts decrease
    ([-1, 3], [5], [[1, 2]], {}),
    ([0, 41], [5], [[1, 2]], {}),             # past the tensors' rows
    ([0, 9], [20], [[1, 2]], {"max_rows": 8}),
    ([0, 2 ** 31 - 1], [5], [[1, 2]], {}),
])
def test_broken_tables(starts, lengths, table, more):
    assert check(starts, lengths, table, **more) == INVALID
    assert b"sequence 0" in lfm3.library().lfm3_last_error()
