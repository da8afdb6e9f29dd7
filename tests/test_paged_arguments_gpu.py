"""Paged K/V cache operators: memory that the current device's kernels cannot
read is refused on the host; pinned host memory serves for the small arrays."""
import ctypes

import numpy as np
import pytest

from helpers import lfm3
from paged import TYPES, Paged

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
INVALID = -1


def setup_module(module):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


class Call:
    """The four operators over one small batch, any pointer replaced."""

    def __init__(self):
        p = self.p = Paged([3, 1], [40, 20], 4, 2, 64, page=16)
        p.k, p.v = torch.nan_to_num(p.k), torch.nan_to_num(p.v)
        f = lambda *shape: torch.ones(*shape, device="cuda")  # noqa: E731
        self.own = dict(
            k=p.k, v=p.v, table=p.dtable, lengths=p.dlengths, starts=p.dstarts,
            positions=torch.arange(4, dtype=torch.int32, device="cuda"), q=p.q,
            gate=f(4, 4), lse=f(4, 4) * 3, out=torch.empty_like(p.q),
            knew=f(4, p.kv_stride), vnew=f(4, p.kv_stride), q_norm=f(64),
            k_norm=f(64), freq=f(32), factors=f(32), weights=f(p.pages, 16),
            space=torch.empty(1 << 26, dtype=torch.uint8, device="cuda"),
            out_table=p.dtable, out_lengths=p.dlengths.clone(),
            kept=torch.zeros(2, 30, dtype=torch.int32, device="cuda"))

    def __call__(self, op, **other):
        p, lib = self.p, lfm3.library()
        a = {name: x.data_ptr() for name, x in self.own.items()}
        a.update(other)
        c = ctypes.byref(p.cache(k=a["k"], v=a["v"], table=a["table"],
                                 lengths=a["lengths"]))
        b = ctypes.byref(p.batch(starts=a["starts"], positions=a["positions"]))
        kind, s = TYPES["f32"], p.stream()
        if op == "heads":
            return lib.lfm3_cuda_paged_heads(
                c, b, kind, a["q"], p.q_stride, a["knew"], p.kv_stride, a["vnew"],
                p.kv_stride, a["out"], p.q_stride, 4, a["q_norm"], a["k_norm"],
                a["freq"], a["factors"], 1e-5, s)
        if op == "attention":
            return lib.lfm3_cuda_paged_attention(
                c, b, kind, a["q"], p.q_stride, a["gate"], 4, a["out"],
                p.q_stride, a["lse"], 4, 0, a["space"], 1 << 26, s)
        if op == "weights":
            return lib.lfm3_cuda_paged_key_weights(
                c, b, kind, a["q"], p.q_stride, a["lse"], a["weights"], 4, 0,
                a["space"], 1 << 26, s)
        return lib.lfm3_cuda_paged_evict(
            c, a["out_table"], a["out_lengths"], a["weights"], a["kept"], 30, 2, s)


BATCH = ["k", "table", "lengths", "starts"]
ARRAYS = {
    "heads": BATCH + ["v", "positions", "q", "out", "knew", "vnew", "q_norm",
                      "k_norm", "freq", "factors"],
    "attention": BATCH + ["v", "q", "out", "gate", "lse", "space"],
    "weights": BATCH + ["q", "lse", "weights", "space"],
    "evict": ["k", "v", "table", "lengths", "out_table", "out_lengths", "weights",
              "kept"],
}


@pytest.mark.parametrize("op,name", [(op, name) for op in ARRAYS
                                     for name in ARRAYS[op]])
def test_pageable_memory_is_refused(op, name):
    call = Call()
    host = np.zeros(1 << 16, np.uint8)
    at = (host.ctypes.data + 255) // 256 * 256
    # the runtime knows nothing of it (else the check could not tell, and the
    # call below is not made)
    kind = ctypes.create_string_buffer(64)
    runtime = torch.cuda.cudart()
    assert runtime is not None
    lib = ctypes.CDLL("libcudart.so.12")
    assert lib.cudaPointerGetAttributes(kind, ctypes.c_void_p(at)) == 0
    assert ctypes.c_int.from_buffer(kind).value == 0  # unregistered
    assert call(op, **{name: at}) == INVALID
    assert b"current device" in lfm3.library().lfm3_last_error()
    assert call(op) == 0
    torch.cuda.synchronize()
    assert lfm3.library().lfm3_cuda_take_device_error() == 0


@pytest.mark.parametrize("op", ["heads", "attention", "weights", "evict"])
def test_small_arrays_may_be_pinned(op):
    """The same bits as with the arrays on the device."""
    results = []
    for pinned in (False, True):
        torch.manual_seed(0)
        call = Call()
        if pinned:
            for name in ARRAYS[op]:
                if name in ("table", "lengths", "starts", "positions", "gate",
                            "lse", "q_norm", "k_norm", "freq", "factors", "kept",
                            "out_lengths", "out_table"):
                    call.own[name] = call.own[name].cpu().pin_memory()
        assert call(op) == 0
        torch.cuda.synchronize()
        names = {"heads": ["out", "k", "v"], "attention": ["out", "lse"],
                 "weights": ["weights"],
                 "evict": ["k", "v", "weights", "kept", "out_lengths"]}[op]
        results.append([call.own[name].cpu().clone() for name in names])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("op,name", [("attention", "positions"),
                                     ("weights", "positions"), ("weights", "v")])
def test_what_an_operator_does_not_read_may_be_anything(op, name):
    call = Call()
    assert call(op, **{name: 0x10000}) == 0
    torch.cuda.synchronize()
    assert lfm3.library().lfm3_cuda_take_device_error() == 0
