"""Paged K/V cache operators on the GPU where numbers or sizes are extreme:
rows of unlike sizes beside each other, infinite scores, idle rows that hold
anything, windows past every length, sums that move out of tensor memory many
times, pools beyond 32-bit offsets. Against the definitions in FP64."""
import ctypes

import numpy as np
import pytest

from helpers import lfm3
from paged import HALF_STEP, TYPES, Paged

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def setup_module(module):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def broken():
    torch.cuda.synchronize()
    return lfm3.library().lfm3_cuda_take_device_error()


# Tolerances of single rows. A score is off by at most e = size * (2^-22 +
# 2 (dim / 16 + 16) 2^-24), size the row's largest sum of |q_d k_d| / sqrt(dim):
# Q carries 22 bits (F32) or is exact, sums of dim / 16 steps may truncate. The
# scaled exponential adds 2^-21, the probabilities' rounding 2^-22 (F32) or
# 2^-11, the sums over keys a step of 2^-23 per 16 keys. Each relative error of
# a probability enters twice (numerator, denominator), times max |v|, and the
# output rounds once. Where e is not small, a row whose first score is ahead of
# the second by 2 e + 40 still has one probability of 1 and others below
# exp(-40) < 2^-57; rows in between are not compared (but have to be finite).
def check_rows(p, out, lse, skip=None, window=0):
    """Every row but those of skip [rows][heads]; returns how many (row, head)
    pairs were compared, and how many were one-hot."""
    d, group = p.dim, p.heads // p.kv_heads
    got = p.host(out)[:, :p.heads * d].reshape(p.rows, p.heads, d)
    got_lse = p.host(lse)
    compared = single = 0
    for s in range(p.seqs):
        b, length = p.starts[s], p.lengths[s]
        if not p.new[s]:
            continue
        q = p.queries(s)
        k, v = p.cached(p.k, s, length), p.cached(p.v, s, length)
        see, top = p.visible(s, window), np.abs(v).max() if length else 0
        for h in range(p.heads):
            live = see.any(1)
            if skip is not None:
                live &= ~skip[b:b + p.new[s], h]
            idle = ~see.any(1)
            assert (got[b:b + p.new[s], h][idle] == 0).all()
            assert np.isneginf(got_lse[b:b + p.new[s], h][idle]).all()
            if not live.any():
                continue
            kh, vh, qh, sh = k[:, h // group], v[:, h // group], q[live, h], see[live]
            x = np.where(sh, qh @ kh.T / np.sqrt(d), -np.inf)
            size = np.where(sh, np.abs(qh) @ np.abs(kh).T / np.sqrt(d), 0).max(1)
            m = x.max(1, keepdims=True)
            w = np.exp(x - m)
            total = w.sum(1, keepdims=True)
            want, want_lse = w / total @ vh, (m + np.log(total))[:, 0]
            e = size * (2.0 ** -22 + 2 * (d / 16 + 16) * 2.0 ** -24)
            x.sort(1)
            gap = x[:, -1] - x[:, -2] if length > 1 else np.full(len(x), np.inf)
            small, hot = e < 2.0 ** -6, gap - 2 * e > 40
            rel = (np.where(hot, 0, np.expm1(np.minimum(e, 1))) + 2.0 ** -21
                   + (2.0 ** -22 if p.kind == "f32" else 2.0 ** -11)
                   + (length / 16 + 2) * 2.0 ** -23)
            y, z = got[b:b + p.new[s], h][live], got_lse[b:b + p.new[s], h][live]
            assert np.isfinite(y).all() and np.isfinite(z).all()
            ok = small | hot
            limit = 2 * rel[:, None] * top + HALF_STEP[p.kind] * np.abs(want) * (
                1 + 2.0 ** -7) + (2.0 ** -25 if p.kind == "f16" else 0)
            off = np.abs(y - want)
            assert (off <= limit)[ok].all(), (s, h, float((off - limit)[ok].max()))
            assert (np.abs(z - want_lse) <= e + rel + 2.0 ** -22 * np.abs(
                want_lse))[ok].all()
            compared += int(ok.sum())
            single += int((ok & hot).sum())
    assert broken() == 0
    return compared, single


@pytest.mark.parametrize("kind,power", [("f16", 26), ("f32", 18), ("f32", 21),
                                        ("f32", 22), ("f32", 24), ("f32", 27),
                                        ("f32", 60), ("f32", 100), ("bf16", 20),
                                        ("bf16", 25), ("bf16", 30),
                                        ("bf16", 110)])
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_of_any_size(kind, power, dim):
    """Scores past 2^24, where a step of FP32 is 1 or more: rows become one-hot,
    not infinite."""
    p = Paged([150, 1, 1, 2], [700, 900, 16, 2], 8, 2, dim, kind=kind, seed=power)
    if kind == "f16":
        p.k *= 2.0 ** (power // 2)
        power -= power // 2
    p.q *= 2.0 ** power
    out, lse = p.attention()
    compared, single = check_rows(p, out, lse)
    assert compared >= 0.9 * p.rows * p.heads and single > 0.8 * compared


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (32, 8, 64),
                                                (3, 1, 128), (16, 1, 64)])
@pytest.mark.parametrize("power", [18, 24, 32, 40, 100])
def test_rows_of_unlike_sizes(kind, heads, kv_heads, dim, power):
    """Heads and queries beside each other whose sizes differ by 2^power: each
    row keeps its own bits."""
    p = Paged([150, 1], [400, 200], heads, kv_heads, dim, kind=kind, seed=power)
    big = torch.zeros(p.rows, heads, dtype=torch.bool, device="cuda")
    big.view(-1)[2::5] = True
    q = p.q.view(p.rows, heads, dim)
    q[big] *= 2.0 ** power
    out, lse = p.attention()
    compared, single = check_rows(p, out, lse)
    # the rows of ordinary size, at least, and most of the others
    assert compared >= 0.8 * p.rows * heads
    assert power < 24 or single > 0


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_rows_beside_infinite_queries(kind, dim, value):
    """A query that is not finite spoils its own rows only, whatever the size of
    those beside it."""
    p = Paged([150, 1], [400, 200], 8, 2, dim, kind=kind)
    bad = np.zeros((p.rows, p.heads), bool)
    bad.reshape(-1)[2::5] = True
    q = p.q.view(p.rows, p.heads, dim)
    q.view(-1, dim)[3::5] *= 2.0 ** 24  # above fp16's largest number
    q.view(-1, dim)[4::5] *= 2.0 ** -30
    q.view(-1, dim)[2::5, 7] = value
    out, lse = p.attention()
    compared, single = check_rows(p, out, lse, skip=bad)
    assert compared >= 0.75 * (~bad).sum() and single > 0
    got = p.host(out)[:, :p.heads * dim].reshape(p.rows, p.heads, dim)
    assert np.isnan(got[bad]).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("value", [3e4, 1e30, float("inf"), float("nan")])
def test_idle_rows_may_hold_anything(kind, value):
    """Rows with negative numbers, and rows that no sequence has, reach no
    result whatever they hold."""
    p = Paged([200, 1, 40], [150, 0, 30], 8, 2, 128, kind=kind, before=3,
              behind=5)
    idle = list(range(3)) + list(range(p.starts[0], p.starts[0] + 50)) + [
        int(p.starts[1])] + list(range(p.starts[2], p.starts[2] + 10)) + list(
        range(p.starts[3], p.rows))
    p.q[idle] = value
    out, lse = p.attention()
    check_rows(p, out, lse)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 60, 2 ** 30])
def test_windows_past_every_length(kind, window):
    """A window that no row fills is no window, in chunks whose first rows have
    no key, too."""
    p = Paged([200, 1, 40, 300], [150, 9, 30, 300], 8, 2, 64, kind=kind)
    out, lse = p.attention(window)
    want, want_lse = p.attention()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    check_rows(p, out, lse)
    start = torch.rand(p.pages, p.page, device="cuda")
    assert torch.equal(p.key_weights(lse, start.clone(), window),
                       p.key_weights(lse, start.clone()))
    assert broken() == 0


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("hidden", [16, 40, 200])
def test_scores_of_minus_infinity(kind, dim, hidden):
    """Keys whose score is -infinity (an infinite key, or an FP32 score past
    the largest number) weigh nothing, in single tokens as in chunks; a row that
    sees no other key is a row without keys."""
    p = Paged([1, 40, 1], [200, 240, 200], 8, 2, dim, page=16, kind=kind)
    if kind == "f16":
        low, p.q[:, :] = float("-inf"), 1.0
    else:  # -1e38 * 1000 * dim / sqrt(dim)
        low, p.q[:, :] = 1000.0, -1e38
    for s, n in enumerate((hidden, hidden, 200)):
        for t in range(p.lengths[s]):
            at = int(p.table[s, t // p.page]), t % p.page
            p.k[at] = low if t < n else 0.0
    out, lse = p.attention()
    got = p.host(out)[:, :8 * dim].reshape(p.rows, 8, dim)
    got_lse = p.host(lse)
    for s in range(3):
        v, see = p.cached(p.v, s, p.lengths[s]), p.visible(s, 0)
        see[:, :200 if s == 2 else hidden] = False
        for i in range(p.new[s]):
            r, count = p.starts[s] + i, see[i].sum()
            if count == 0:
                assert (got[r] == 0).all() and np.isneginf(got_lse[r]).all()
                continue
            want = v[see[i]].mean(0).repeat(4, 0)  # scores of 0: the mean
            # probabilities are equal numbers, exact in fp16: the sums' steps
            # (2^-23 per 16 keys), 1 / l and the output's rounding remain
            limit = 17 * 2.0 ** -23 * np.abs(v).max() + HALF_STEP[kind] * np.abs(
                want) * (1 + 2.0 ** -7) + (2.0 ** -25 if kind == "f16" else 0)
            assert (np.abs(got[r] - want) <= limit).all()
            assert np.abs(got_lse[r] - np.log(count)).max() <= 8 * 2.0 ** -21
    assert broken() == 0


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), 1.0])
def test_weights_of_rows_without_lse(kind, value):
    """A query whose lse is -infinity adds nothing, whatever it and the keys
    hold: among others, a whole column block of them, single tokens."""
    p = Paged([150, 1, 1, 70], [900, 300, 290, 600], 8, 2, 128, kind=kind)
    lse = p.attention()[1]
    off = torch.zeros(p.rows, 8, dtype=torch.bool, device="cuda")
    off.view(-1)[5::7] = True
    off[32:64] = True            # queries 32 .. 63: a column block
    off[p.starts[2]] = True
    q = p.q.view(p.rows, 8, 128)
    q[off] = value
    lse[off] = float("-inf")
    # a key that only such rows see: sequence 3's last
    off[p.rows - 1] = True
    lse[p.rows - 1] = float("-inf")
    last = int(p.table[3, 599 // p.page]), 599 % p.page
    p.k[last] = float("-inf") if value == 1.0 else value
    start = torch.rand(p.pages, p.page, device="cuda") + 0.5
    got = p.host(p.key_weights(lse, start.clone()))
    z, want = p.host(lse), p.host(start)
    p.q = torch.where(off[:, :, None], torch.zeros_like(q), q).view(p.rows, -1)
    p.k[last] = 0.0
    scale = 1.0
    for s in range(p.seqs):
        i = np.arange(p.lengths[s])
        place = p.table[s, i // p.page], i % p.page
        had = want[place]
        had[p.lengths[s] - p.new[s]:] = 0
        want[place] = had + p.expect_weights(s, z)
        scale = max(scale, p.expect_attention(s)[2])
    assert got[last] == 0
    # a probability carries its score's error and the exponential's, and sums
    # of n * heads of them round by a step of 2^-24 each
    rel = (scale * (2.0 ** -22 + 2 * (128 / 16 + 16) * 2.0 ** -24) + 2.0 ** -20
           + (150 * 8 + 8) * 2.0 ** -24 + 2.0 ** -23 * np.abs(
               z[np.isfinite(z)]).max())
    assert (np.abs(got - want) <= rel * np.abs(want) + 1e-30).all()
    assert broken() == 0


# ---- sums that move out of tensor memory -----------------------------------------
def spikes(p, s):
    """Every 600 keys of sequence s one whose score is 6.5 or 12.5 above the
    others', in turn: rows move their reference, and what they have summed up
    before still counts."""
    b, e = p.starts[s], p.starts[s + 1]
    p.q[b:e].view(e - b, -1)[:, :p.heads * p.dim:p.dim] = 8.0
    at = torch.from_numpy(p.table[s].astype(np.int64)).cuda()
    pages = -(-p.lengths[s] // p.page)
    p.k[at[:pages], :, :, 0] = 0.0
    for j, t in enumerate(range(300, p.lengths[s], 600)):
        p.k[int(p.table[s, t // p.page]), t % p.page, :, 0] = (
            (6.5, 12.5)[j % 2] * p.dim ** 0.5 / 8)


# In the 2-norm. FP32 rows: 64 additions in tensor memory (4 tiles of 8 steps and
# two terms) drop half a step of 2^-23 each, of a sum that grows from 0: 1.9e-6;
# the scores' sums shrink by 8 such halves in 16 steps, 5e-7 of scores of size
# 1.3 to 2; Q's and P's roundings of 2^-23 are independent and a tenth of that.
# 4e-6 bounds their sum. Spikes: scores of 12.5 instead of 2, 8e-6. A flush that
# is lost or counted twice changes the sums by a tile's share or more: 1e-2.
def norm_off(p, s, rows, out, lse):
    """The rows' error in the 2-norm against FP64, and the lse's largest."""
    d, group = p.dim, p.heads // p.kv_heads
    k, v = p.cached(p.k, s, p.lengths[s]), p.cached(p.v, s, p.lengths[s])
    base = p.lengths[s] - p.new[s]
    q = p.queries(s)
    square = off = worst = 0.0
    for i in rows:
        own = base + i
        for h in range(p.heads):
            x = k[:own + 1, h // group] @ q[i, h] / np.sqrt(d)
            m = x.max()
            w = np.exp(x - m)
            want = w @ v[:own + 1, h // group] / w.sum()
            got = p.host(out[p.starts[s] + i, h * d:(h + 1) * d])
            off += float(((got - want) ** 2).sum())
            square += float((want ** 2).sum())
            z = float(lse[p.starts[s] + i, h])
            worst = max(worst, abs(z - (m + np.log(w.sum()))) / max(1, abs(z)))
    return (off / square) ** 0.5, worst


@pytest.mark.parametrize("moving", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,n,length", [
    (16, 4, 128, 512, 8704), (32, 8, 64, 512, 8300), (8, 8, 64, 2300, 5000),
    (4, 4, 128, 256, 12000)])
def test_sums_moved_many_times(moving, heads, kv_heads, dim, n, length):
    """FP32 rows over segments of 9 to 40 key tiles: their sums leave tensor
    memory every 4 tiles and are added up, with the reference unmoved or moved
    in between."""
    p = Paged([n], [length], heads, kv_heads, dim, page=128)
    if moving:
        spikes(p, 0)
    out, lse = p.attention()
    off, worst = norm_off(p, 0, (0, 1, n // 3, n // 2 + 7, n - 1), out, lse)
    assert off <= (8e-6 if moving else 4e-6) and worst <= 4e-6
    assert broken() == 0


# ---- offsets past 32 bits -------------------------------------------------------
def test_pools_past_32_bit_offsets():
    """Pools of 5 GB whose held pages lie at both ends: element and byte offsets
    pass 2^32."""
    p = Paged([60, 1, 0], [300, 700, 0], 8, 2, 128, page=64, kind="bf16",
              extra_pages=5)
    small, pages = p.pages, 5 * 2 ** 30 // (64 * 2 * 128 * 2)
    for name in ("k", "v"):
        x = torch.zeros(pages, 64, 2, 128, dtype=torch.float16, device="cuda")
        x[:8] = getattr(p, name)[:8]
        x[pages - (small - 8):] = getattr(p, name)[8:]
        setattr(p, name, x)
    assert p.k.numel() > 2 ** 31 and p.k.numel() * 2 > 2 ** 32
    p.table[p.table >= 8] += pages - small
    p.pages, p.dtable = pages, torch.from_numpy(p.table).cuda()
    out, lse = p.attention()
    check_rows(p, out, lse)
    start = torch.rand(pages, 64, device="cuda")
    got = p.host(p.key_weights(lse, start.clone()))
    want, z = p.host(start), p.host(lse)
    for s in range(2):
        i = np.arange(p.lengths[s])
        place = p.table[s, i // 64], i % 64
        had = want[place]
        had[p.lengths[s] - p.new[s]:] = 0
        want[place] = had + p.expect_weights(s, z)
    assert (np.abs(got - want) <= 1e-4 * np.abs(want)).all()
    # heads: the keys as they are (no norm, angles of 0) into the same places
    new = torch.randn(p.rows, 256, device="cuda").to(p.q.dtype)
    q, zero = p.q.clone(), torch.zeros(64, device="cuda")
    c, b = p.cache(), p.batch()
    lfm3.check(lfm3.library().lfm3_cuda_paged_heads(
        ctypes.byref(c), ctypes.byref(b), TYPES["bf16"], q.data_ptr(),
        p.q_stride, new.data_ptr(), 256, new.data_ptr(), 256, q.data_ptr(),
        p.q_stride, 8, None, None, zero.data_ptr(), None, 0.0, p.stream()))
    held = [p.cached(p.k, s, p.lengths[s]) for s in range(2)]
    for s in range(2):
        x = p.host(new[p.starts[s]:p.starts[s + 1]].half()).reshape(-1, 2, 128)
        assert np.array_equal(held[s][p.lengths[s] - p.new[s]:], x)
    # eviction in place
    weights = torch.rand(pages, 64, device="cuda")
    kept = torch.full((3, 100), -1, dtype=torch.int32, device="cuda")
    lfm3.check(lfm3.library().lfm3_cuda_paged_evict(
        ctypes.byref(c), p.dtable.data_ptr(), p.dlengths.data_ptr(),
        weights.data_ptr(), kept.data_ptr(), 100, 10, p.stream()))
    for s in range(2):
        rows = kept[s].cpu().numpy()
        assert (np.diff(rows) > 0).all() and rows[-10:].min() == p.lengths[s] - 10
        assert np.array_equal(p.cached(p.k, s, 100), held[s][rows])
    assert p.dlengths.tolist() == [100, 100, 0]
    assert broken() == 0
