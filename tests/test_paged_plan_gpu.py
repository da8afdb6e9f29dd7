"""How the paged kernels share out a batch (paged_plan.cuh), run on tables
without tensors: the blocks' shares have to hold every unit of the batch, for
any mix of lengths and for sizes that no test could give tensors to."""
import ctypes
import os
import random
import subprocess

import pytest

from helpers import ROOT

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
CSRC = os.path.join(ROOT, "lfm3-gufo-extension_b200", "csrc")
CHUNKS, WEIGHTS, DECODE = 0, 1, 2
BLOCKS = {CHUNKS: 148, WEIGHTS: 148, DECODE: 296}


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    so = str(tmp_path_factory.mktemp("plan") / "probe.so")
    cmd = [os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc"), "-gencode",
           "arch=compute_100a,code=sm_100a", "-std=c++20", "-O2", "-rdc=true",
           "-Xcompiler", "-fPIC", "-shared", "--expt-relaxed-constexpr",
           "-diag-suppress", "20044",
           os.path.join(ROOT, "tests", "paged_plan_probe.cu"),
           os.path.join(CSRC, "device_error.cu"), "-o", so]
    done = subprocess.run(cmd, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    call = ctypes.CDLL(so).paged_plan_probe

    def run(what, new, lengths, kv_heads, group, window=0, extra=0, walk=True):
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        s = torch.tensor(starts, dtype=torch.int32, device="cuda")
        le = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        out = torch.zeros(5, dtype=torch.int64, device="cuda")
        assert call(what, ctypes.c_void_p(s.data_ptr()),
                    ctypes.c_void_p(le.data_ptr()), len(new), kv_heads, group,
                    window, extra, int(walk), max(lengths) // 16 + 1, 16,
                    starts[-1], max(new), ctypes.c_void_p(out.data_ptr())) == 0
        return out.tolist()

    return run


def chunk_units(n, length, group, window, pair):
    """Key tiles of 128 that a pair of row tiles sees."""
    queries = 2 * (128 // group)
    base, q0 = length - n, pair * queries
    last = base + min(n, q0 + queries) - 1
    first = max(0, base + q0 - window + 1) if window else 0
    return 0 if last < first else last // 128 - first // 128 + 1


def weight_blocks(n, length, group, window, pair):
    """Column blocks that a pair of key tiles is seen by."""
    queries = 128 // group
    base, k0 = length - n, pair * 256
    k1 = min(k0 + 256, length) - 1
    first, last = max(0, k0 - base), n - 1
    if window:
        last = min(last, k1 + window - 1 - base)
    return 0 if last < first else last // queries - first // queries + 1


def units(what, new, lengths, kv_heads, group, window):
    """(units, stretches) of a batch."""
    total = stretches = 0
    for n, length in zip(new, lengths):
        if what == CHUNKS:
            if n == 0 or (n == 1 and group <= 16):
                continue
            count = -(-n // (2 * (128 // group)))
            per = [chunk_units(n, length, group, window, p) for p in range(count)]
        else:
            count = -(-length // 256) if n else 0
            per = [weight_blocks(n, length, group, window, p) * kv_heads
                   for p in range(count)]
        many = kv_heads if what == CHUNKS else 1
        total += sum(per) * many
        stretches += sum(1 for x in per if x) * many
    return total, stretches


@pytest.mark.parametrize("what", [CHUNKS, WEIGHTS])
def test_every_unit_is_in_a_segment(probe, what):
    rng = random.Random(what)
    for _ in range(300):
        seqs = rng.choice([1, 2, 5, 8, 9, 31, 32, 33, 70])
        group = rng.choice([1, 3, 4, 16, 17, 65, 128])
        kv_heads = rng.choice([1, 2, 8, 40])
        window = rng.choice([0, 0, 1, 100, 256, 5000, 2 ** 31 - 1])
        most = rng.choice([3, 40, 700, 5000])
        new = [rng.choice([0, 1, rng.randint(0, most)]) for _ in range(seqs)]
        lengths = [max(0, n + rng.choice([0, -5, rng.randint(0, 9000)]))
                   for n in new]
        if not any(new) or not any(lengths):
            continue
        extra = rng.choice([4, 6]) if what == CHUNKS else 0
        share, total, held, begun, _ = probe(what, new, lengths, kv_heads, group,
                                             window, extra)
        want, stretches = units(what, new, lengths, kv_heads, group, window)
        case = (new, lengths, kv_heads, group, window)
        assert share * BLOCKS[what] >= total >= want, case
        assert held == want and begun == stretches, case


@pytest.mark.parametrize("rows,kv_heads,group,window", [
    (700_000, 4, 65, 64),      # two rows a stretch: 1.4 M stretches
    (2_200_000, 128, 1, 16),
    (1_000_000, 8, 128, 128),
    (300_000, 1024, 1, 256),
])
@pytest.mark.parametrize("extra", [4, 6])
def test_more_than_a_million_stretches(probe, rows, kv_heads, group, window,
                                       extra):
    share, total, _, _, _ = probe(CHUNKS, [rows], [rows], kv_heads, group,
                                  window, extra, walk=False)
    assert share * BLOCKS[CHUNKS] >= total
    # (a pair's tiles do not depend on it beyond the window, but their sum does)
    want, _ = units(CHUNKS, [rows], [rows], kv_heads, group, window)
    assert total >= want
    share, total, _, _, _ = probe(WEIGHTS, [rows], [rows], kv_heads, group,
                                  window, walk=False)
    assert total == units(WEIGHTS, [rows], [rows], kv_heads, group, window)[0]
    assert share * BLOCKS[WEIGHTS] >= total


def test_shares_of_single_tokens(probe):
    rng = random.Random(7)
    for _ in range(300):
        seqs = rng.choice([1, 3, 32, 40, 700, 4096])
        top = rng.choice([20, 3000, 2 ** 20, 2 ** 31 - 5000])
        lengths = [rng.randint(0, top) for _ in range(seqs)]
        if not any(lengths):
            continue
        kv_heads, group = rng.choice([1, 4, 64, 1024]), rng.choice([1, 4, 16])
        window = rng.choice([0, 0, 500, 2 ** 31 - 1])
        share, total, _, _, _ = probe(DECODE, [1] * seqs, lengths, kv_heads,
                                      group, window)
        want = sum(-(-n // 16) if not window or n <= window else
                   (n - 1) // 16 - (n - window) // 16 + 1
                   for n in lengths) * kv_heads
        assert share * BLOCKS[DECODE] >= total >= want, (lengths, kv_heads)
