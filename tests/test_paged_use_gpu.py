"""Paged K/V cache operators as a server calls them: a whole step captured once
and replayed over changed tables, calls of every operator at once on several
streams, the largest batches and head counts the header allows."""
import ctypes

import numpy as np
import pytest

from helpers import lfm3
from paged import TYPES, Paged
from test_paged_extremes_gpu import check_rows
from test_paged_gpu import expect_kept

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def setup_module(module):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def broken():
    torch.cuda.synchronize()
    return lfm3.library().lfm3_cuda_take_device_error()


class Step:
    """heads, attention, key weights and eviction of one batch, with buffers of
    their own."""

    def __init__(self, seed=0, kind="bf16", new=(1, 70, 1, 0, 1), window=0,
                 lengths=(900, 300, 64, 20, 0)):
        p = self.p = Paged(new, lengths, 8, 2, 64, page=16, kind=kind, seed=seed)
        p.k, p.v = torch.nan_to_num(p.k), torch.nan_to_num(p.v)
        lib, c, b = lfm3.library(), p.cache(), p.batch()
        at, bt = ctypes.byref(c), ctypes.byref(b)
        sizes = [f(at, bt, 8) for f in (
            lib.lfm3_cuda_paged_attention_workspace_bytes,
            lib.lfm3_cuda_paged_key_weights_workspace_bytes)]
        self.window, self.keep = window, 100
        self.space = [torch.empty(n, dtype=torch.uint8, device="cuda")
                      for n in sizes]
        f = p.normal
        self.new = [f(p.rows, 128).to(p.q.dtype) for _ in range(2)]
        self.freq = torch.rand(32, device="cuda")
        self.norm = 1 + 0.1 * f(64)
        self.q = torch.zeros_like(p.q)
        self.out = torch.zeros(p.rows, 512, dtype=p.q.dtype, device="cuda")
        self.lse = torch.zeros(p.rows, 8, device="cuda")
        self.weights = torch.rand(p.pages, 16, device="cuda")
        self.kept = torch.full((p.seqs, self.keep), -1, dtype=torch.int32,
                               device="cuda")
        self.lengths = torch.zeros_like(p.dlengths)
        self.buffers = [p.k, p.v, self.q, self.out, self.lse, self.weights,
                        self.kept, self.lengths]
        self.first = [x.clone() for x in self.buffers]

    def reset(self):
        for x, y in zip(self.buffers, self.first):
            x.copy_(y)

    def __call__(self):
        p, lib, s = self.p, lfm3.library(), self.p.stream()
        at, bt = ctypes.byref(p.cache()), ctypes.byref(p.batch())
        kind, ld = TYPES[p.kind], p.q_stride
        lfm3.check(lib.lfm3_cuda_paged_heads(
            at, bt, kind, p.q.data_ptr(), ld, self.new[0].data_ptr(), 128,
            self.new[1].data_ptr(), 128, self.q.data_ptr(), ld, 8,
            self.norm.data_ptr(), self.norm.data_ptr(), self.freq.data_ptr(),
            None, 1e-5, s))
        lfm3.check(lib.lfm3_cuda_paged_attention(
            at, bt, kind, self.q.data_ptr(), ld, None, 0, self.out.data_ptr(),
            512, self.lse.data_ptr(), 8, self.window, self.space[0].data_ptr(),
            self.space[0].numel(), s))
        lfm3.check(lib.lfm3_cuda_paged_key_weights(
            at, bt, kind, self.q.data_ptr(), ld, self.lse.data_ptr(),
            self.weights.data_ptr(), 8, self.window, self.space[1].data_ptr(),
            self.space[1].numel(), s))
        lfm3.check(lib.lfm3_cuda_paged_evict(
            at, p.dtable.data_ptr(), self.lengths.data_ptr(),
            self.weights.data_ptr(), self.kept.data_ptr(), self.keep, 10, s))

    def results(self):
        torch.cuda.synchronize()
        return [x.clone() for x in self.buffers]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_a_captured_step_reads_tables_afresh(kind):
    step = Step(kind=kind)
    step()  # (kernels are loaded before the capture)
    step.results()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for lengths in ((900, 300, 64, 20, 0), (400, 70, 1, 0, 0),
                    (880, 60, 64, 20, 0), (0, 0, 0, 0, 0)):
        step.p.dlengths.copy_(torch.tensor(lengths))
        step.reset()
        step()
        want = step.results()
        for _ in range(3):
            step.reset()
            graph.replay()
            assert same(step.results(), want), lengths
    assert broken() == 0


def test_steps_on_three_streams():
    """Eager calls and replayed graphs at once, each with its own buffers."""
    steps = [Step(1, "f32"), Step(2, "bf16", window=50),
             Step(3, "f16", (300, 1, 1), lengths=(2000, 500, 0))]
    want, graphs = [], []
    for s in steps:
        s()
        want.append(s.results())
        g = torch.cuda.CUDAGraph()
        s.reset()
        with torch.cuda.graph(g):
            s()
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in steps]
    for turn in range(6):
        torch.cuda.synchronize()
        for i, s in enumerate(steps):
            with torch.cuda.stream(streams[i]):
                s.reset()
                if (turn + i) % 2:
                    graphs[i].replay()
                else:
                    s()
        for i, s in enumerate(steps):
            assert same(s.results(), want[i]), (turn, i)
    assert broken() == 0


@pytest.mark.parametrize("new", ["single", "mixed"])
def test_as_many_sequences_as_allowed(new):
    """4096 sequences, of 0 to 40 rows each."""
    rng = np.random.default_rng(4)
    lengths = rng.integers(0, 41, 4096)
    lengths[7], lengths[4095] = 700, 300
    rows = np.ones(4096, int) if new == "single" else rng.integers(0, 3, 4096)
    p = Paged(rows.tolist(), lengths.tolist(), 2, 1, 64, page=16, kind="f32")
    p.k, p.v = torch.nan_to_num(p.k), torch.nan_to_num(p.v)
    out, lse = p.attention()
    check_rows(p, out, lse)
    start = torch.rand(p.pages, 16, device="cuda")
    got = p.host(p.key_weights(lse, start.clone()))
    want, z = p.host(start), p.host(lse)
    for s in range(4096):
        if not rows[s]:
            continue
        i = np.arange(lengths[s])
        place = p.table[s, i // 16], i % 16
        had = want[place]
        had[max(0, lengths[s] - rows[s]):] = 0
        want[place] = had + p.expect_weights(s, z)
    assert (np.abs(got - want) <= 1e-4 * np.abs(want) + 1e-30).all()
    keep, recent = 20, 3
    w, before = start.cpu().numpy(), p.k.clone()
    kept = torch.full((4096, keep), -1, dtype=torch.int32, device="cuda")
    lfm3.check(lfm3.library().lfm3_cuda_paged_evict(
        ctypes.byref(p.cache()), p.dtable.data_ptr(), p.dlengths.data_ptr(),
        start.data_ptr(), kept.data_ptr(), keep, recent, p.stream()))
    assert broken() == 0
    got, left = kept.cpu().numpy(), p.dlengths.cpu().numpy()
    after, before = p.k.cpu().numpy(), before.cpu().numpy()
    for s in range(4096):
        i = np.arange(lengths[s])
        chosen = expect_kept(w[p.table[s, i // 16], i % 16], keep, recent)
        assert left[s] == len(chosen) and (got[s, :len(chosen)] == chosen).all()
        j = np.arange(len(chosen))
        assert np.array_equal(after[p.table[s, j // 16], j % 16],
                              before[p.table[s, chosen // 16], chosen % 16])


@pytest.mark.parametrize("heads,kv_heads", [(1024, 1024), (4096, 32)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_as_many_heads_as_allowed(heads, kv_heads, kind):
    """1024 KV heads, and groups of 128."""
    p = Paged([1, 5, 140], [70, 40, 200], heads, kv_heads, 64, page=32, kind=kind)
    out, lse = p.attention()
    check_rows(p, out, lse)
    w = p.host(p.key_weights(lse, torch.zeros(p.pages, 32, device="cuda")))
    assert abs(w.sum() / (146 * heads) - 1) < 1e-5
