"""A paged K/V cache on the GPU for the paged operators' tests, its calls
through the C ABI, and the operators' definitions in FP64 (numpy)."""
import ctypes

import numpy as np

from helpers import abi, lfm3

TYPES = {"f32": abi.F32, "f16": abi.F16, "bf16": abi.BF16}
# a rounding to the type is off by at most half a step
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def torch_type(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16,
            "bf16": torch.bfloat16}[name]


class Paged:
    """Sequences of lengths[s] rows, the last new[s] of them this call's."""

    def __init__(self, new, lengths, heads=16, kv_heads=4, dim=128, page=64,
                 kind="f32", seed=0, extra_pages=3, before=0, behind=0,
                 max_rows=None, stride_pad=0):
        import torch
        self.torch = torch
        self.new, self.lengths = list(new), list(lengths)
        self.heads, self.kv_heads, self.dim, self.page = heads, kv_heads, dim, page
        self.kind, self.before = kind, before
        self.seqs = len(self.new)
        rng = np.random.default_rng(seed)
        used = [-(-n // page) for n in self.lengths]
        self.width = max(used + [1])
        self.pages = sum(used) + extra_pages
        order = rng.permutation(self.pages)
        # table rows are wider than used, unused entries are not page ids
        self.table = np.full((self.seqs, self.width + 2), -7, np.int32)
        at = 0
        for s, n in enumerate(used):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.starts = (before + np.concatenate([[0], np.cumsum(self.new)])
                       ).astype(np.int32)
        self.rows = int(self.starts[-1]) + behind
        self.max_rows = max(self.new + [0]) if max_rows is None else max_rows
        g = torch.Generator(device="cuda")
        g.manual_seed(seed + 1)

        def normal(*shape, scale=1.0):
            return torch.randn(*shape, generator=g, device="cuda") * scale

        t = torch_type(kind)
        self.k = normal(self.pages, page, kv_heads, dim).half()
        self.v = normal(self.pages, page, kv_heads, dim).half()
        # rows that no sequence holds must never reach a result
        held = np.zeros((self.pages, page), bool)
        for s, n in enumerate(self.lengths):
            i = np.arange(n)
            held[self.table[s, i // page], i % page] = True
        free = torch.from_numpy(~held).cuda()
        self.k[free] = float("nan")
        self.v[free] = float("nan")
        self.q_stride = heads * dim + stride_pad
        self.kv_stride = kv_heads * dim + stride_pad
        self.q = normal(self.rows, self.q_stride, scale=1.3).to(t)
        self.gate = normal(self.rows, heads + 3).to(t)
        self.dtable = torch.from_numpy(self.table).cuda()
        self.dlengths = torch.tensor(self.lengths, dtype=torch.int32,
                                     device="cuda")
        self.dstarts = torch.from_numpy(self.starts).cuda()
        self.positions = None
        self.normal = normal

    def cache(self, **over):
        d = dict(k=self.k.data_ptr(), v=self.v.data_ptr(),
                 table=self.dtable.data_ptr(), lengths=self.dlengths.data_ptr(),
                 pages=self.pages, page_rows=self.page, kv_heads=self.kv_heads,
                 dim=self.dim, sequences=self.seqs, table_pages=self.width,
                 table_stride=self.table.shape[1])
        d.update(over)
        return abi.PagedCache(**d)

    def batch(self, **over):
        d = dict(starts=self.dstarts.data_ptr(),
                 positions=(self.positions.data_ptr()
                            if self.positions is not None else None),
                 rows=self.rows, max_rows=self.max_rows)
        d.update(over)
        return abi.PagedBatch(**d)

    def stream(self):
        return self.torch.cuda.current_stream().cuda_stream

    # ---- calls -----------------------------------------------------------
    def attention(self, window=0, gate=False, lse=True, workspace=None,
                  out=None, poison=True):
        torch, lib = self.torch, lfm3.library()
        c, b = self.cache(), self.batch()
        need = lib.lfm3_cuda_paged_attention_workspace_bytes(
            ctypes.byref(c), ctypes.byref(b), self.heads)
        if workspace is None:  # contents are arbitrary: NaN patterns
            workspace = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
        if out is None:
            out = torch.full((self.rows, self.heads * self.dim + 8), 77.0,
                             dtype=self.q.dtype, device="cuda")
        ls = torch.full((self.rows, self.heads), 55.0, device="cuda") if lse else None
        lfm3.check(lib.lfm3_cuda_paged_attention(
            ctypes.byref(c), ctypes.byref(b), TYPES[self.kind],
            self.q.data_ptr(), self.q_stride,
            self.gate.data_ptr() if gate else None, self.heads + 3,
            out.data_ptr(), out.shape[1], ls.data_ptr() if lse else None,
            self.heads, window, workspace.data_ptr(), workspace.numel(),
            self.stream()))
        return out, ls

    def key_weights(self, lse, weights, window=0):
        torch, lib = self.torch, lfm3.library()
        c, b = self.cache(), self.batch()
        need = lib.lfm3_cuda_paged_key_weights_workspace_bytes(
            ctypes.byref(c), ctypes.byref(b), self.heads)
        space = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
        lfm3.check(lib.lfm3_cuda_paged_key_weights(
            ctypes.byref(c), ctypes.byref(b), TYPES[self.kind],
            self.q.data_ptr(), self.q_stride, lse.data_ptr(),
            weights.data_ptr(), self.heads, window, space.data_ptr(), need,
            self.stream()))
        return weights

    # ---- definitions -------------------------------------------------------
    def host(self, x):
        self.torch.cuda.synchronize()
        return x.double().cpu().numpy()

    def cached(self, pool, s, n):
        """The first n rows of sequence s [n][kv_heads][dim] in FP64."""
        i = np.arange(n)
        at = self.torch.from_numpy(
            self.table[s, i // self.page].astype(np.int64)).cuda()
        off = self.torch.from_numpy(i % self.page).cuda()
        return self.host(pool[at, off])

    def queries(self, s):
        """Sequence s's new queries [n][heads][dim] in FP64."""
        b, e = self.starts[s], self.starts[s + 1]
        q = self.host(self.q[b:e, :self.heads * self.dim])
        return q.reshape(e - b, self.heads, self.dim)

    def visible(self, s, window):
        """[n][length]: the keys each new row sees."""
        n, length = self.new[s], self.lengths[s]
        own = (length - n + np.arange(n))[:, None]
        t = np.arange(length)[None, :]
        see = t <= own
        if window:
            see &= t > own - window
        return see

    def expect_attention(self, s, window=0, gate=False):
        """(out [n][heads][dim], lse [n][heads]) of sequence s in FP64, and
        the largest sum of |q_d k_d| / sqrt(dim) of a visible pair."""
        n, length, group = self.new[s], self.lengths[s], self.heads // self.kv_heads
        q = self.queries(s)
        k, v = self.cached(self.k, s, length), self.cached(self.v, s, length)
        see = self.visible(s, window)
        out = np.zeros((n, self.heads, self.dim))
        lse = np.full((n, self.heads), -np.inf)
        size = 0.0
        rows = see.any(axis=1)
        for h in range(self.heads):
            if not rows.any():
                break
            kh, vh = k[:, h // group], v[:, h // group]
            x = q[:, h] @ kh.T / np.sqrt(self.dim)
            size = max(size, float((np.abs(q[:, h]) @ np.abs(kh).T)[see].max()
                                   / np.sqrt(self.dim)))
            x[~see] = -np.inf
            x = x[rows]
            m = x.max(axis=1, keepdims=True)
            p = np.exp(x - m)
            total = p.sum(axis=1, keepdims=True)
            out[rows, h] = (p / total) @ vh
            lse[rows, h] = (m + np.log(total))[:, 0]
        if gate:
            b, e = self.starts[s], self.starts[s + 1]
            g = self.host(self.gate[b:e, :self.heads])
            out /= (1 + np.exp(-g))[:, :, None]
        return out, lse, size

    def expect_weights(self, s, lse, window=0):
        """What each cached row of s gains, from the lse given [rows][heads]."""
        length, group = self.lengths[s], self.heads // self.kv_heads
        q, k = self.queries(s), self.cached(self.k, s, length)
        see = self.visible(s, window)
        b, e = self.starts[s], self.starts[s + 1]
        gain = np.zeros(length)
        for h in range(self.heads):
            x = q[:, h] @ k[:, h // group].T / np.sqrt(self.dim)
            z = lse[b:e, h][:, None]
            with np.errstate(invalid="ignore", over="ignore"):
                p = np.exp(x - z)
            p[~see | ~np.isfinite(z).repeat(length, 1)] = 0
            gain += p.sum(axis=0)
        return gain
