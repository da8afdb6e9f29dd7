"""Paged K/V cache operators on the GPU against their definitions in FP64
(tests/paged.py): ragged batches, odd sizes, empty rows and sequences, windows,
strides, every type, pages that end inside a key tile, and the operators run
together as a serving loop uses them."""
import ctypes

import numpy as np
import pytest

from helpers import abi, lfm3
from paged import HALF_STEP, TYPES, Paged, torch_type

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def setup_module(module):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def broken():
    torch.cuda.synchronize()
    return lfm3.library().lfm3_cuda_take_device_error()


# ---- attention -----------------------------------------------------------------
# Tolerances. A score is a sum of dim products: Q carries 22 bits (F32) or is
# exact (16-bit types), the products are exact in FP32 and the sum of dim / 16
# steps rounds to FP32 (tensor cores may truncate: a full step each), so a
# score is off by at most size * (2^-22 + 2 (dim / 16 + 16) 2^-24), size the
# sum of |q_d k_d| / sqrt(dim). The scaled exponential adds 2^-21 relative, the
# probabilities' rounding 2^-22 (F32) or 2^-11, the sums over keys a step of
# 2^-23 per 16 keys, and every relative error of a probability enters the
# output (numerator and denominator) at most twice, times max |v|. The output
# rounds once.
def check_attention(p, window=0, gate=False):
    out, lse = p.attention(window, gate)
    got = p.host(out)[:, :p.heads * p.dim].reshape(p.rows, p.heads, p.dim)
    got_lse = p.host(lse)
    covered = np.zeros(p.rows, bool)
    square_off = square = 0.0
    for s in range(p.seqs):
        b, e = p.starts[s], p.starts[s + 1]
        covered[b:e] = True
        if b == e:
            continue
        want, want_lse, size = p.expect_attention(s, window, gate)
        top = p.host(p.v[torch.isfinite(p.v)].abs().max())
        score = size * (2.0 ** -22 + 2 * (p.dim / 16 + 16) * 2.0 ** -24)
        rel = (score + 2.0 ** -21 + (2.0 ** -22 if p.kind == "f32" else 2.0 ** -11)
               + (p.lengths[s] / 16 + 2) * 2.0 ** -23)
        limit = 2 * rel * top + HALF_STEP[p.kind] * np.abs(want) * (1 + 2.0 ** -7)
        # fp16 outputs below its normal range round in steps of 2^-24
        limit = limit + (2.0 ** -25 if p.kind == "f16" else 0)
        off = np.abs(got[b:e] - want)
        assert (off <= limit).all(), (s, float((off - limit).max()), float(off.max()))
        empty = np.isneginf(want_lse)
        assert (np.isneginf(got_lse[b:e]) == empty).all()
        assert (got[b:e][empty] == 0).all()
        z = np.abs(got_lse[b:e][~empty] - want_lse[~empty])
        if z.size:
            # (probabilities' roundings enter the sum as relative errors)
            assert z.max() <= rel + 2.0 ** -22 * np.abs(want_lse[~empty]).max()
        square_off += float((off ** 2).sum())
        square += float((want ** 2).sum())
    # together, independent roundings: in the 2-norm at most the output's half
    # step and the probabilities', and for F32 the score's 2^-22 size (taken
    # as 10) and a few steps
    if square:
        norm = (square_off / square) ** 0.5
        bound = {"f32": 8e-6, "f16": 2.0 ** -11 + 2.0 ** -11,
                 "bf16": 2.0 ** -8 + 2.0 ** -11}[p.kind]
        assert norm <= bound, norm
    # rows outside the sequences and columns past the heads are untouched
    assert (got[~covered] == 77).all() and (got_lse[~covered] == 55).all()
    assert (p.host(out)[:, p.heads * p.dim:] == 77).all()
    assert broken() == 0


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 4, 128), (32, 8, 64),
                                                (4, 4, 128), (8, 1, 64)])
def test_decode_edges(kind, heads, kv_heads, dim):
    lengths = [1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 257, 1000]
    check_attention(Paged([1] * len(lengths), lengths, heads, kv_heads, dim,
                          page=16, kind=kind), gate=True)


@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_decode_long(page, kind):
    check_attention(Paged([1, 1, 1], [9001, 33, 4096], page=page, kind=kind))


def test_decode_many_sequences():
    rng = np.random.default_rng(5)
    lengths = rng.integers(0, 300, 333)
    check_attention(Paged([1] * 333, lengths, 4, 2, 64, page=16, kind="f16"),
                    gate=True)


@pytest.mark.parametrize("heads,kv_heads", [(3, 1), (10, 2), (12, 2), (7, 1),
                                            (9, 1), (16, 1), (128, 1),
                                            (25, 5)])
@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_odd_groups(heads, kv_heads, kind):
    check_attention(Paged([1, 5, 0, 40], [70, 5, 12, 200], heads, kv_heads, 64,
                          page=32, kind=kind, seed=3))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,length", [(2, 2), (3, 130), (17, 17), (31, 400),
                                      (32, 32), (33, 97), (64, 64), (65, 65),
                                      (127, 128), (128, 129), (129, 1000),
                                      (512, 700)])
def test_chunk_edges(kind, n, length):
    check_attention(Paged([n], [length], page=16 if n % 2 else 128, kind=kind,
                          seed=n), gate=n % 3 == 0)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_chunk_over_long_history(kind, dim):
    check_attention(Paged([77, 200], [9000, 5003], 8, 2, dim, page=48,
                          kind=kind))


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("window", [1, 2, 17, 64, 128, 129, 700])
def test_windows(kind, window):
    check_attention(Paged([1, 130, 1, 3, 64], [1000, 600, 30, 3, 2000], 8, 2,
                          128, page=32, kind=kind, seed=window), window,
                    gate=True)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_mixed_ragged_batch(kind):
    """Chunks, single tokens, idle sequences, rows before and behind."""
    check_attention(Paged([1, 0, 300, 1, 2, 0, 77, 1], [500, 90, 1300, 1, 2, 0,
                          77, 4000], page=64, kind=kind, before=3, behind=9,
                          stride_pad=24), gate=True)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_without_keys(kind):
    """Idle slots of a fixed-shape graph (length 0, one row) and chunks whose
    first rows have no key."""
    check_attention(Paged([1, 1, 1, 200, 20], [0, 5, 0, 150, 0], page=16,
                          kind=kind), gate=True)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("window", [0, 100])
def test_uneven_lengths(kind, window):
    """Shares of the work that end between and behind stretches: many short
    sequences beside a few long ones, single tokens and chunks from row 0."""
    lengths = [9000] + list(range(1, 60)) * 2 + [4000, 16, 17]
    check_attention(Paged([1] * len(lengths), lengths, 8, 4, 64, page=32,
                          kind=kind), window)
    new = [400, 30, 2, 70, 150]
    p = Paged(new, [400, 30, 900, 70, 151], 16, 8, 64, page=16, kind=kind)
    check_attention(p, window, gate=True)
    check_weights(p, window)
    new = [1, 65, 1] * 15
    check_attention(Paged(new, [n + i for i, n in enumerate(new)], 4, 2, 128,
                          page=16, kind=kind), window)


def test_max_rows_is_only_a_bound():
    check_attention(Paged([1, 1, 1], [100, 200, 300], max_rows=500, behind=600))
    check_attention(Paged([40], [100], max_rows=4000, kind="bf16"))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 150])
def test_wide_scores(kind, n):
    """Large queries (scores of +-1000: nearly one-hot rows), tiny ones and
    zeros; and scores that grow along the sequence, so that every tile moves
    the running maximum."""
    p = Paged([n, n, n], [700, 700, 700], 8, 2, 128, kind=kind)
    p.q[p.starts[0]:p.starts[1]] *= 60 / 1.3
    p.q[p.starts[1]:p.starts[2]] *= 2.0 ** -12
    p.q[p.starts[1]] = 0
    i = np.arange(700)
    at = torch.from_numpy(p.table[2, i // p.page].astype(np.int64)).cuda()
    ramp = torch.linspace(0.01, 1.5, 700, device="cuda")[:, None, None]
    p.k[at, torch.from_numpy(i % p.page).cuda()] = (
        ramp * torch.ones(1, 2, 128, device="cuda")).half()
    p.q[p.starts[2]:p.starts[3]] = 2.0
    check_attention(p)


def test_infinite_values_in_other_rows_stay_there():
    """A NaN key or value reaches only the rows that see it."""
    p = Paged([40, 1], [300, 300], 8, 2, 128, kind="f16")
    row = 290  # visible to the last new rows of sequence 0 only
    p.v[int(p.table[0, row // p.page]), row % p.page] = float("inf")
    out, lse = p.attention()
    got = p.host(out)[:, :p.heads * p.dim]
    first = p.starts[0] + row - (300 - 40)
    assert np.isfinite(got[:first]).all()
    assert not np.isfinite(got[first:p.starts[1]]).any()
    assert np.isfinite(got[p.starts[1]:]).all()
    assert np.isfinite(p.host(lse)).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_infinite_keys_and_queries(kind):
    """A NaN query spoils its own rows; a NaN key the rows that see it; their
    weights and nothing else."""
    p = Paged([70, 1], [500, 300], 8, 2, 128, kind=kind)
    p.q[5, 128:256] = float("nan")          # row 5, head 1
    row = 480                               # seen from new row 50 on
    p.k[int(p.table[0, row // p.page]), row % p.page, 1] = float("nan")
    out, lse = p.attention()
    got = p.host(out)[:, :p.heads * p.dim].reshape(p.rows, p.heads, p.dim)
    bad = np.zeros((p.rows, p.heads), bool)
    bad[5, 1] = True
    bad[50:70, 4:] = True                   # the KV head's four heads
    assert (np.isnan(got).all(2) == bad).all()
    assert (np.isfinite(got).all(2) == ~bad).all()


def test_same_bits_every_time_and_on_another_stream():
    p = Paged([1, 200, 1], [5000, 3000, 40], kind="bf16")
    a, la = p.attention()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b, lb = p.attention()
    side.synchronize()
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_captured_call_reads_tables_afresh():
    p = Paged([1, 1], [900, 300], kind="f32")
    space = torch.empty(
        lfm3.library().lfm3_cuda_paged_attention_workspace_bytes(
            ctypes.byref(p.cache()), ctypes.byref(p.batch()), p.heads),
        dtype=torch.uint8, device="cuda")
    out = torch.zeros(p.rows, p.heads * p.dim + 8, device="cuda")
    p.attention(workspace=space, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.attention(workspace=space, out=out, lse=False)
    p.dlengths.copy_(torch.tensor([700, 299]))
    p.lengths = [700, 299]
    out.fill_(0)
    graph.replay()
    want = p.attention()[0]
    assert torch.equal(out[:, :-8], want[:, :-8])


def test_sequences_may_share_pages():
    """A common prefix: three sequences whose first pages are the same."""
    p = Paged([1, 70, 1], [900, 600, 300], 8, 2, 128, page=64, kind="f16")
    for s in (1, 2):
        p.table[s, :4] = p.table[0, :4]
    p.dtable = torch.from_numpy(p.table).cuda()
    check_attention(p)


@pytest.mark.parametrize("page,heads,kv_heads", [(256, 16, 4), (1040, 8, 2),
                                                 (32, 192, 192),
                                                 (4096, 384, 3)])
def test_large_pages_and_many_heads(page, heads, kv_heads):
    p = Paged([1, 140, 3], [700, 1100, 90], heads, kv_heads, 64, page=page,
              kind="f16")
    check_attention(p, gate=True)
    check_weights(p)


def test_outputs_have_to_be_on_the_device():
    p = Paged([4], [40])
    host = torch.empty(p.rows, p.heads * p.dim + 8).pin_memory()
    with pytest.raises(RuntimeError, match="out is not on the current device"):
        p.attention(out=host)
    lib, c, b = lfm3.library(), p.cache(), p.batch()
    f = torch.ones(p.dim // 2, device="cuda")
    k = torch.zeros(p.rows, p.kv_stride, device="cuda")
    with pytest.raises(RuntimeError, match="q_out is not on the current"):
        lfm3.check(lib.lfm3_cuda_paged_heads(
            ctypes.byref(c), ctypes.byref(b), TYPES["f32"], p.q.data_ptr(),
            p.q_stride, k.data_ptr(), p.kv_stride, k.data_ptr(), p.kv_stride,
            host.data_ptr(), host.shape[1], p.heads, None, None, f.data_ptr(),
            None, 1e-5, p.stream()))
    check_attention(p)


def test_two_calls_at_once():
    """Calls on two streams, each with its own workspace and outputs."""
    one = Paged([1, 300, 1], [4000, 2000, 70], kind="f32", seed=1)
    two = Paged([1] * 20, list(range(100, 2100, 100)), kind="bf16", seed=2)
    want = [x.attention() for x in (one, two)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for t in streams:
        t.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(4):
        for i, x in enumerate((one, two)):
            with torch.cuda.stream(streams[i]):
                got[i].append(x.attention())
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])


def test_queries_written_just_before():
    """Mixed batches run two kernels that overlap: both must see queries that
    the work queued right before the call wrote."""
    p = Paged([1, 200, 1, 90], [3000, 1500, 70, 400], kind="bf16")
    a, b = p.q.clone(), torch.randn_like(p.q)
    want = []
    for x in (a, b):
        p.q.copy_(x)
        torch.cuda.synchronize()
        want.append(p.attention()[0].clone())
    torch.cuda.synchronize()
    got = []
    for i in range(20):
        p.q.copy_((a, b)[i % 2])
        got.append(p.attention()[0])
    torch.cuda.synchronize()
    for i in range(20):
        assert torch.equal(got[i], want[i % 2])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_long_chunk_rows(kind):
    """Rows whose keys fill hundreds of tiles of one block (where fp16 rows
    move their sums out of tensor memory): some rows against FP64."""
    heads, n, length, dim = 8, 4096, 40960, 64
    p = Paged([n], [length], heads, heads, dim, page=128, kind=kind)
    out, lse = p.attention()
    k, v = p.cached(p.k, 0, length), p.cached(p.v, 0, length)
    for row in (0, 1, 777, 2048, n - 1):
        q = p.host(p.q[row, :heads * dim]).reshape(heads, dim)
        own = length - n + row
        x = np.einsum("hd,thd->ht", q, k[:own + 1]) / np.sqrt(dim)
        m = x.max(1, keepdims=True)
        e = np.exp(x - m)
        want = np.einsum("ht,thd->hd", e / e.sum(1, keepdims=True), v[:own + 1])
        got = p.host(out[row, :heads * dim]).reshape(heads, dim)
        off = np.linalg.norm(got - want) / np.linalg.norm(want)
        # the two half steps, and for fp16 256 tiles' losses in tensor memory
        # (a step of at most 2^-23 each, 8 a tile)
        assert off <= HALF_STEP[kind] + 2.0 ** -11 + 2048 * 2.0 ** -23
        assert np.abs(p.host(lse[row]) - (m[:, 0] + np.log(e.sum(1)))).max() < 1e-4
    assert broken() == 0


# ---- broken tables: nothing faults, the error word says so ---------------------
@pytest.mark.parametrize("what", ["page", "length", "starts", "max_rows"])
def test_broken_tables_are_reported(what):
    p = Paged([1, 40, 1], [500, 400, 300], kind="f16")
    if what == "page":
        p.dtable[1, 2] = p.pages
        p.dtable[0, 3] = -1
    elif what == "length":
        p.dlengths[1] = p.width * p.page + 1
    elif what == "starts":
        p.dstarts[2] = 10 ** 6
    else:
        p.max_rows = 39
    fine = p.expect_attention(2)[0] if what != "starts" else None
    out, lse = p.attention()
    assert broken() == 6
    if fine is not None:  # the other sequences are right
        got = p.host(out)[p.starts[2]:, :p.heads * p.dim]
        assert np.abs(got.reshape(fine.shape) - fine).max() < 4e-3
    weights = torch.zeros(p.pages, p.page, device="cuda")
    p.key_weights(lse, weights)
    assert broken() == 6
    # heads: only pages that hold new rows are needed
    q = p.q.clone()
    k = torch.zeros(p.rows, p.kv_stride, dtype=p.q.dtype, device="cuda")
    freq = torch.ones(p.dim // 2, device="cuda")
    if what == "page":
        p.dtable[1, (400 - 1) // p.page] = -5
    c, b = p.cache(), p.batch()
    before = p.k.clone()
    lfm3.check(lfm3.library().lfm3_cuda_paged_heads(
        ctypes.byref(c), ctypes.byref(b), TYPES["f16"], q.data_ptr(),
        p.q_stride, k.data_ptr(), p.kv_stride, k.data_ptr(), p.kv_stride,
        q.data_ptr(), p.q_stride, p.heads, None, None, freq.data_ptr(), None,
        0.0, p.stream()))
    assert broken() == 6
    # nothing but the new rows' places in sound pages was written
    changed = (p.k != before) & ~(p.k.isnan() & before.isnan())
    pages = set(changed.flatten(1).any(1).nonzero().flatten().tolist())
    fine = {int(x) for s in range(3) for x in p.table[s] if 0 <= x < p.pages}
    assert pages <= fine


@pytest.mark.parametrize("what", ["page", "length", "negative"])
def test_evict_broken_tables(what):
    p = Paged([0, 0], [500, 400], 4, 2, 64, page=16)
    p.k, p.v = torch.nan_to_num(p.k), torch.nan_to_num(p.v)
    if what == "page":
        p.dtable[1, 3] = p.pages + 5
    else:
        p.dlengths[1] = -1 if what == "negative" else p.width * 16 + 1
    w = torch.rand(p.pages, 16, device="cuda")
    kept = torch.full((2, 100), -1, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    host = w.cpu().numpy()
    c = p.cache()
    lfm3.check(lfm3.library().lfm3_cuda_paged_evict(
        ctypes.byref(c), p.dtable.data_ptr(), lengths.data_ptr(), w.data_ptr(),
        kept.data_ptr(), 100, 10, p.stream()))
    assert broken() == 6
    i = np.arange(500)
    want = expect_kept(host[p.table[0, i // 16], i % 16], 100, 10)
    assert (kept[0].cpu().numpy() == want).all()
    assert lengths[1].item() == (100 if what == "page" else 0)


# ---- heads -----------------------------------------------------------------------
def run_heads(p, seed=0, norms=True, factors=True, positions=None,
              in_place=False):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t, d = p.q.dtype, p.dim
    k = (torch.randn(p.rows, p.kv_stride, generator=g, device="cuda") * 0.7).to(t)
    v = (torch.randn(p.rows, p.kv_stride, generator=g, device="cuda") * 0.7).to(t)
    qn = 1 + 0.1 * torch.randn(d, generator=g, device="cuda") if norms else None
    kn = 1 + 0.1 * torch.randn(d, generator=g, device="cuda") if norms else None
    freq = (1e6 ** (torch.arange(d // 2, device="cuda", dtype=torch.float64)
                    * (-2.0 / d))).float()
    fac = torch.linspace(1, 8, d // 2, device="cuda") if factors else None
    p.positions = positions
    q = p.q.clone()
    out = q if in_place else torch.full_like(q, 33.0)
    pk, pv = p.k.clone(), p.v.clone()
    lib, c, b = lfm3.library(), p.cache(), p.batch()
    c.k, c.v = pk.data_ptr(), pv.data_ptr()

    def at(x):
        return x.data_ptr() if x is not None else None

    lfm3.check(lib.lfm3_cuda_paged_heads(
        ctypes.byref(c), ctypes.byref(b), TYPES[p.kind], q.data_ptr(),
        p.q_stride, k.data_ptr(), p.kv_stride, v.data_ptr(), p.kv_stride,
        out.data_ptr(), p.q_stride, p.heads, at(qn), at(kn), at(freq), at(fac),
        1e-5, p.stream()))
    got = p.host(out)
    want_k, want_v = p.host(p.k), p.host(p.v)
    want_q = p.host(p.q) if in_place else np.full(got.shape, 33.0)
    f = p.host(freq) / (p.host(fac) if factors else 1.0)
    pos_all = positions.cpu().numpy() if positions is not None else None

    def turn(x, w, pos):
        if norms:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * p.host(w)
        a, b = x[..., :d // 2], x[..., d // 2:]
        angle = np.asarray(pos, np.float64)[:, None, None] * f
        return np.concatenate([a * np.cos(angle) - b * np.sin(angle),
                               b * np.cos(angle) + a * np.sin(angle)], -1)

    if not norms:  # norms of 1: the formula without them
        qn = kn = None
    for s in range(p.seqs):
        b0, e0 = p.starts[s], p.starts[s + 1]
        number = p.lengths[s] - p.new[s] + np.arange(p.new[s])
        pos = pos_all[b0:e0] if pos_all is not None else number
        if b0 == e0:
            continue
        x = p.host(p.q[b0:e0, :p.heads * d]).reshape(-1, p.heads, d)
        want_q[b0:e0, :p.heads * d] = turn(x, qn, pos).reshape(e0 - b0, -1)
        x = p.host(k[b0:e0, :p.kv_heads * d]).reshape(-1, p.kv_heads, d)
        y = turn(x, kn, pos)
        z = p.host(v[b0:e0, :p.kv_heads * d]).reshape(-1, p.kv_heads, d)
        for i, row in enumerate(number):
            if row >= 0:
                place = int(p.table[s, row // p.page]), row % p.page
                want_k[place], want_v[place] = y[i], z[i]
    # FP32 arithmetic (sum of squares of dim terms, root, quotient, products)
    # on values of at most 10, angles reduced to 2^-23 of a radian; one
    # rounding to the type (F16 in the pages, whose steps below 2^-14 are
    # 2^-24)
    for x, y, half in ((got, want_q, HALF_STEP[p.kind]),
                       (p.host(pk), want_k, 2.0 ** -11),
                       (p.host(pv), want_v, 2.0 ** -11)):
        fine = np.isfinite(y)
        assert (np.isfinite(x) == fine).all()
        limit = half * np.abs(y[fine]) * (1 + 2.0 ** -7) + 2.0 ** -25 + 10 * 2.0 ** -21
        assert (np.abs(x[fine] - y[fine]) <= limit).all()
    assert broken() == 0


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 4, 128), (32, 8, 64),
                                                (3, 1, 64), (5, 5, 128)])
def test_heads(kind, heads, kv_heads, dim):
    run_heads(Paged([1, 0, 50, 3, 1], [77, 5, 50, 400, 1], heads, kv_heads,
                    dim, page=16, kind=kind, before=2, behind=5, stride_pad=8))


def test_heads_far_positions_and_idle_rows():
    p = Paged([1, 30, 2, 1], [0, 20, 9, 40], page=32)
    run_heads(p, positions=torch.randint(0, 10 ** 6, (p.rows,), dtype=torch.int32,
                                         device="cuda"))


def test_heads_without_norms_in_place():
    run_heads(Paged([5, 9], [5, 100], 8, 2, 64, kind="bf16"), norms=False,
              factors=False, in_place=True)


def test_heads_many_sequences():
    run_heads(Paged([1] * 200, list(range(1, 201)), 4, 2, 64, page=16,
                    kind="f16"))


# ---- key weights -----------------------------------------------------------------
def check_weights(p, window=0):
    lse = p.attention(window)[1]
    start = torch.rand(p.pages, p.page, device="cuda") + 0.5
    got = p.host(p.key_weights(lse, start.clone(), window))
    want, z = p.host(start), p.host(lse)
    scale = 1.0
    for s in range(p.seqs):
        if not p.new[s] or not p.lengths[s]:
            continue
        i = np.arange(p.lengths[s])
        place = p.table[s, i // p.page], i % p.page
        had = want[place]
        had[max(0, p.lengths[s] - p.new[s]):] = 0
        want[place] = had + p.expect_weights(s, z, window)
        scale = max(scale, p.expect_attention(s, window)[2])
    # each probability carries its score's error (see check_attention) and
    # the exponential's; all terms are positive, sums of n * heads of them in
    # FP32 and their FP32 partial sums round by a step of 2^-24 each
    rel = (scale * (2.0 ** -22 + 2 * (p.dim / 16 + 16) * 2.0 ** -24) + 2.0 ** -20
           + (max(p.new) * p.heads + 8) * 2.0 ** -24
           + 2.0 ** -23 * np.abs(z[np.isfinite(z)]).max())
    off = np.abs(got - want)
    assert (off <= rel * np.abs(want) + 1e-30).all(), float((off / np.abs(want)).max())
    assert broken() == 0


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 4, 128), (32, 8, 64),
                                                (12, 4, 128), (7, 1, 64)])
def test_weights_ragged(kind, heads, kv_heads, dim):
    check_weights(Paged([1, 0, 70, 1, 5, 1, 33], [500, 90, 300, 1, 5, 0, 1000],
                        heads, kv_heads, dim, page=16, kind=kind, before=1,
                        behind=4, stride_pad=16))


@pytest.mark.parametrize("window", [1, 30, 128, 500])
def test_weights_window(window):
    check_weights(Paged([1, 130, 2], [900, 700, 64], 8, 2, 128, page=48,
                        kind="bf16"), window)


def test_weights_long():
    check_weights(Paged([1, 300], [9000, 5000], page=64, kind="f32"))


def test_weights_rows_without_keys():
    check_weights(Paged([1, 1, 60], [0, 7, 40], page=16, kind="f32"))


def test_weights_sum_to_the_heads():
    """Every row's probabilities sum to 1 per head: the chunk adds
    new rows * heads in all."""
    p = Paged([200], [1500], kind="f32")
    lse = p.attention()[1]
    w = p.key_weights(lse, torch.zeros(p.pages, p.page, device="cuda"))
    assert abs(p.host(w).sum() / (200 * p.heads) - 1) < 1e-5


# ---- eviction ----------------------------------------------------------------------
def expect_kept(w, keep, recent):
    n = len(w)
    if n <= keep:
        return np.arange(n)
    old = n - recent
    order = sorted(range(old), key=lambda t: (not np.isnan(w[t]), -w[t] if not
                                              np.isnan(w[t]) else 0, t))
    return np.array(sorted(order[:keep - recent]) + list(range(old, n)))


def run_evict(lengths, keep, recent, in_place, page=16, kv_heads=2, dim=64,
              weights=None, own_lengths=False, seed=0):
    p = Paged([0] * len(lengths), lengths, kv_heads * 2, kv_heads, dim, page,
              seed=seed, extra_pages=3 + sum(-(-min(n, keep) // page)
                                             for n in lengths))
    p.k = torch.nan_to_num(p.k)
    p.v = torch.nan_to_num(p.v)
    p.width = max(p.width, -(-keep // page))
    if p.table.shape[1] < p.width:
        p.table = np.pad(p.table, ((0, 0), (0, p.width - p.table.shape[1])),
                         constant_values=-7)
        p.dtable = torch.from_numpy(p.table).cuda()
    rng = np.random.default_rng(seed)
    out_table = p.table.copy()
    if not in_place:
        free = sorted(set(range(p.pages)) - {int(x) for s, n in
                                             enumerate(lengths) for x in
                                             p.table[s, :-(-n // page)]})
        rng.shuffle(free)
        at = 0
        for s, n in enumerate(lengths):
            m = -(-min(n, keep) // page)
            out_table[s, :m] = free[at:at + m]
            at += m
    if weights is None:  # many ties
        weights = rng.integers(0, 40, (p.pages, page)).astype(np.float32) / 8
    w = torch.from_numpy(weights.copy()).cuda()
    before = p.k.cpu().numpy(), p.v.cpu().numpy(), weights
    dout = torch.from_numpy(out_table).cuda() if not in_place else p.dtable
    out_lengths = p.dlengths if own_lengths else torch.full_like(p.dlengths, -5)
    kept = torch.full((len(lengths), keep), -1, dtype=torch.int32, device="cuda")
    c = p.cache()
    lfm3.check(lfm3.library().lfm3_cuda_paged_evict(
        ctypes.byref(c), dout.data_ptr(), out_lengths.data_ptr(), w.data_ptr(),
        kept.data_ptr(), keep, recent, p.stream()))
    torch.cuda.synchronize()
    after = p.k.cpu().numpy(), p.v.cpu().numpy(), w.cpu().numpy()
    got_kept, got_len = kept.cpu().numpy(), out_lengths.cpu().numpy()
    touched = [x.copy() for x in before]
    for s, n in enumerate(lengths):
        i = np.arange(n)
        place = p.table[s, i // page], i % page
        want = expect_kept(weights[place], keep, recent)
        assert got_len[s] == want.size
        assert (got_kept[s, :want.size] == want).all()
        assert (got_kept[s, want.size:] == -1).all()
        j = np.arange(want.size)
        to = out_table[s, j // page], j % page
        for x, y in zip(touched, before):
            x[to] = y[place][want]
    for x, y in zip(after, touched):  # moved exactly, nothing else touched
        assert np.array_equal(x.view(np.uint8), y.view(np.uint8))
    assert broken() == 0


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (50, 0), (50, 50),
                                         (100, 7), (1000, 3)])
def test_evict(in_place, keep, recent):
    run_evict([0, 1, 49, 50, 51, 100, 101, 777, 1500], keep, recent, in_place,
              own_lengths=in_place)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("kv_heads,dim,page", [(4, 128, 64), (1, 64, 48),
                                               (3, 64, 32), (8, 128, 16)])
def test_evict_shapes(in_place, kv_heads, dim, page):
    run_evict([3000, 64, 900], 400, 30, in_place, page, kv_heads, dim, seed=4)


def test_evict_long():
    run_evict([20000], 5000, 100, True, page=64, seed=9)


def test_evict_many_sequences():
    """A block a sequence, one of them with more rows than it stages."""
    run_evict([20000] + [30 + i for i in range(80)], 60, 7, True, page=64)
    run_evict([17] * 149 + [600], 100, 0, False)


def test_evict_in_place_through_a_copy_of_the_table():
    p = Paged([0, 0], [700, 300], 4, 2, 64, page=16)
    p.k, p.v = torch.nan_to_num(p.k), torch.nan_to_num(p.v)
    w = torch.rand(p.pages, 16, device="cuda")
    kept = torch.full((2, 200), -1, dtype=torch.int32, device="cuda")
    before, host = p.k.clone(), w.cpu().numpy()
    c = p.cache()
    lfm3.check(lfm3.library().lfm3_cuda_paged_evict(
        ctypes.byref(c), p.dtable.clone().data_ptr(), p.dlengths.data_ptr(),
        w.data_ptr(), kept.data_ptr(), 200, 20, p.stream()))
    torch.cuda.synchronize()
    for s, n in enumerate((700, 300)):
        i, j = np.arange(n), np.arange(200)
        want = expect_kept(host[p.table[s, i // 16], i % 16], 200, 20)
        at = torch.from_numpy(p.table[s].astype(np.int64)).cuda()
        src, dst = torch.from_numpy(want).cuda(), torch.from_numpy(j).cuda()
        assert torch.equal(p.k[at[dst // 16], dst % 16],
                           before[at[src // 16], src % 16])


def test_evict_weights_of_every_kind():
    rng = np.random.default_rng(2)
    w = rng.choice(np.array([0.0, -0.0, 1e-45, 1e-38, 1.0, 3.4e38, np.inf,
                             -1.0, -np.inf, np.nan], np.float32), (200, 16))
    run_evict([700, 300], 200, 5, True, weights=w[:3 + 44 + 19 + 13 + 13])
    run_evict([700, 300], 200, 0, False, weights=w[:3 + 44 + 19 + 13 + 13])


# ---- together ----------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_serving_loop(kind):
    """Prompt chunks, decode steps, weights and an eviction, twice: the cache
    after each step matches a plain restatement that keeps every sequence's
    keys, values, positions and weights as Python lists of rows."""
    heads, kv_heads, dim, page, width = 4, 2, 64, 16, 16
    seqs, lib = 3, lfm3.library()
    rng = np.random.default_rng(0)
    t = torch_type(kind)
    pages = seqs * width
    k = torch.zeros(pages, page, kv_heads, dim, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    weights = torch.full((pages, page), 9.0, device="cuda")
    table = rng.permutation(pages).reshape(seqs, width).astype(np.int32)
    dtable = torch.from_numpy(table).cuda()
    freq = torch.from_numpy((1e4 ** (-np.arange(dim // 2) * 2 / dim)
                             ).astype(np.float32)).cuda()
    lengths, seen = np.zeros(seqs, np.int32), np.zeros(seqs, np.int32)
    rows_of = [[] for _ in range(seqs)]  # (key, value, weight) per cached row
    keep, recent = 60, 10

    def host(x):
        torch.cuda.synchronize()
        return x.double().cpu().numpy()

    for new in ([70, 33, 5], [1, 1, 1], [1, 0, 90], [1, 1, 1], None,
                [1, 1, 1], [20, 2, 1], None, [1, 1, 1]):
        dl = torch.from_numpy(lengths.copy()).cuda()
        c = abi.PagedCache(k.data_ptr(), v.data_ptr(), dtable.data_ptr(),
                           dl.data_ptr(), pages, page, kv_heads, dim, seqs,
                           width, width)
        if new is None:
            kept = torch.full((seqs, keep), -1, dtype=torch.int32, device="cuda")
            lfm3.check(lib.lfm3_cuda_paged_evict(
                ctypes.byref(c), dtable.data_ptr(), dl.data_ptr(),
                weights.data_ptr(), kept.data_ptr(), keep, recent,
                torch.cuda.current_stream().cuda_stream))
            lengths = host(dl).astype(np.int32)
            got = host(weights)
            for s in range(seqs):
                n = len(rows_of[s])
                chosen = host(kept)[s, :lengths[s]].astype(int)
                # the device's own weights decide (they differ from the
                # restatement's in the last bits)
                w = np.array([x[2] for x in rows_of[s]], np.float32)
                assert (chosen == expect_kept(w, keep, recent)).all()
                rows_of[s] = [rows_of[s][i] for i in chosen]
                assert lengths[s] == min(n, keep)
        else:
            n = np.array(new)
            starts = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
            rows = int(starts[-1])
            lengths = (lengths + n).astype(np.int32)
            dl.copy_(torch.from_numpy(lengths))
            pos = np.concatenate([seen[s] + np.arange(n[s]) for s in range(seqs)])
            seen = (seen + n).astype(np.int32)
            x = [torch.from_numpy(rng.standard_normal((rows, m * dim)).astype(
                np.float32)).cuda().to(t) for m in (heads, kv_heads, kv_heads)]
            ds = torch.from_numpy(starts).cuda()
            dp = torch.from_numpy(pos.astype(np.int32)).cuda()
            b = abi.PagedBatch(ds.data_ptr(), dp.data_ptr(), rows, int(n.max()))
            at, bt = ctypes.byref(c), ctypes.byref(b)
            st = torch.cuda.current_stream().cuda_stream
            raw = [host(y) for y in x]
            lfm3.check(lib.lfm3_cuda_paged_heads(
                at, bt, TYPES[kind], x[0].data_ptr(), heads * dim,
                x[1].data_ptr(), kv_heads * dim, x[2].data_ptr(),
                kv_heads * dim, x[0].data_ptr(), heads * dim, heads, None, None,
                freq.data_ptr(), None, 1e-5, st))
            size = lib.lfm3_cuda_paged_attention_workspace_bytes(at, bt, heads)
            more = lib.lfm3_cuda_paged_key_weights_workspace_bytes(at, bt, heads)
            space = torch.empty(max(size, more), dtype=torch.uint8, device="cuda")
            out = torch.empty(rows, heads * dim, dtype=t, device="cuda")
            lse = torch.empty(rows, heads, device="cuda")
            lfm3.check(lib.lfm3_cuda_paged_attention(
                at, bt, TYPES[kind], x[0].data_ptr(), heads * dim, None, 0,
                out.data_ptr(), heads * dim, lse.data_ptr(), heads, 0,
                space.data_ptr(), size, st))
            lfm3.check(lib.lfm3_cuda_paged_key_weights(
                at, bt, TYPES[kind], x[0].data_ptr(), heads * dim,
                lse.data_ptr(), weights.data_ptr(), heads, 0, space.data_ptr(),
                more, st))
            got_w, got_out, q = host(weights), host(out), host(x[0])
            pk, pv = host(k), host(v)
            for s in range(seqs):
                for i in range(n[s]):
                    angle = pos[starts[s] + i] * host(freq)
                    kx = raw[1][starts[s] + i].reshape(kv_heads, dim)
                    a, bb = kx[:, :dim // 2], kx[:, dim // 2:]
                    key = np.concatenate([a * np.cos(angle) - bb * np.sin(angle),
                                          bb * np.cos(angle) + a * np.sin(angle)], 1)
                    row = lengths[s] - n[s] + i
                    place = table[s, row // page], row % page
                    assert np.abs(pk[place] - key).max() < 4e-3  # F16 step at 4
                    rows_of[s].append([pk[place], pv[place], 0.0])
                assert len(rows_of[s]) == lengths[s]
                if not n[s]:
                    continue
                i = np.arange(lengths[s])
                place = table[s, i // page], i % page
                # rows moved as they were stored
                assert np.array_equal(pk[place], np.stack([y[0] for y in rows_of[s]]))
                assert np.array_equal(pv[place], np.stack([y[1] for y in rows_of[s]]))
                gain = np.zeros(lengths[s])
                for h in range(heads):
                    kk, vv = pk[place][:, h // 2], pv[place][:, h // 2]
                    qq = q[starts[s]:starts[s + 1]].reshape(-1, heads, dim)[:, h]
                    z = qq @ kk.T / np.sqrt(dim)
                    z[i[None] > (lengths[s] - n[s] + np.arange(n[s]))[:, None]] = -np.inf
                    e = np.exp(z - z.max(1, keepdims=True))
                    e /= e.sum(1, keepdims=True)
                    gain += e.sum(0)
                    o = got_out[starts[s]:starts[s + 1]].reshape(-1, heads, dim)[:, h]
                    # |v| < 5: twice 2^-11 (bf16: and its half step) of it
                    limit = 1e-4 if kind == "f32" else 5 * (2 * 2.0 ** -11 + 2.0 ** -8)
                    assert np.abs(o - e @ vv).max() < limit
                old = np.array([y[2] for y in rows_of[s]])
                assert np.abs(got_w[place] - (old + gain)).max() < 1e-4 * heads
                for y, w in zip(rows_of[s], got_w[place]):
                    y[2] = w
    assert broken() == 0
