"""Cases and plain forms of the paged K/V cache operators.

The cache of one attention layer is a pool of pages, F16 [pages][page_rows]
[kv_heads][dim] for keys and for values; sequence s holds lengths[s] rows in
the pages table[s][0], table[s][1], ... A call advances the sequences by
ragged chunks of new rows (starts[s] .. starts[s + 1] - 1 of its tensors),
which are the last of their sequence's rows:

  heads      per-head RMSNorm and rotation of queries and keys, keys and
             values stored in the pages
  attention  causal (optionally sliding-window) attention of the new rows
             over the pages, optionally gated, with its log sum of exponentials
  weights    the attention weight every cached key receives from the new
             rows, added to what it has accumulated
  evict      the keys of least accumulated weight leave, the others move to
             other pages, in order

`own` selects the library's operators; otherwise the plain forms run."""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ABI_TYPES = {"f32": 0, "f16": 1, "bf16": 30}
EPS = 1e-5


# ---- cases -------------------------------------------------------------------

def listed():
    model = {"heads": 16, "kv_heads": 4, "dim": 128}   # the default geometry
    narrow = {"heads": 32, "kv_heads": 8, "dim": 64}   # 32 / 8 heads of 64
    return [
        # one new row for each of 8 sessions of the decode round
        {"name": "heads decode 8", "op": "heads", "type": "f32", **model,
         "page": 64, "seqs": 8, "single": 8, "hist_lo": 64, "hist_hi": 4096,
         "new_lo": 1, "new_hi": 1, "shape": 1},
        # a 512-row prompt pass of one session
        {"name": "heads pass 512", "op": "heads", "type": "f32", **model,
         "page": 64, "seqs": 1, "single": 0, "hist_lo": 2048, "hist_hi": 2048,
         "new_lo": 512, "new_hi": 512, "shape": 2},
        # prefill of a ragged batch of prompts, 16-bit activations
        {"name": "heads prefill ragged", "op": "heads", "type": "bf16", **narrow,
         "page": 32, "seqs": 12, "single": 0, "hist_lo": 1, "hist_hi": 30000,
         "new_lo": 301, "new_hi": 2049, "shape": 3},
        # a decode round of 8 sessions at ragged depths
        {"name": "attn decode 8", "op": "attention", "type": "f32", **model,
         "page": 64, "seqs": 8, "single": 8, "hist_lo": 64, "hist_hi": 4096,
         "new_lo": 1, "new_hi": 1, "window": 0, "gate": True, "shape": 4},
        # a serving batch's decode step over long, ragged histories
        {"name": "attn decode 32 long", "op": "attention", "type": "bf16",
         **model, "page": 32, "seqs": 32, "single": 32, "hist_lo": 512,
         "hist_hi": 32768, "new_lo": 1, "new_hi": 1, "window": 0,
         "gate": False, "shape": 5},
        # a 512-row prompt pass at depth 8192, 32-bit activations
        {"name": "attn pass 512 at 8K", "op": "attention", "type": "f32",
         **model, "page": 64, "seqs": 1, "single": 0, "hist_lo": 8192,
         "hist_hi": 8192, "new_lo": 512, "new_hi": 512, "window": 0,
         "gate": True, "shape": 6},
        # prompt chunks between single tokens, sliding-window layer
        {"name": "attn mixed window", "op": "attention", "type": "f16",
         **narrow, "page": 16, "seqs": 20, "single": 16, "hist_lo": 33,
         "hist_hi": 5000, "new_lo": 77, "new_hi": 700, "window": 256,
         "gate": True, "shape": 7},
        # long prompt chunks deep in their histories
        {"name": "attn chunks 2K at 16K", "op": "attention", "type": "bf16",
         **model, "page": 128, "seqs": 2, "single": 0, "hist_lo": 14000,
         "hist_hi": 16384, "new_lo": 1900, "new_hi": 2048, "window": 0,
         "gate": False, "shape": 8},
        # weight bookkeeping of a decode step
        {"name": "weights decode 16", "op": "weights", "type": "f32", **model,
         "page": 64, "seqs": 16, "single": 16, "hist_lo": 1024,
         "hist_hi": 8192, "new_lo": 1, "new_hi": 1, "window": 0, "shape": 9},
        # weight bookkeeping of a prompt pass
        {"name": "weights pass 512", "op": "weights", "type": "bf16", **model,
         "page": 64, "seqs": 1, "single": 0, "hist_lo": 8192, "hist_hi": 8192,
         "new_lo": 512, "new_hi": 512, "window": 0, "shape": 10},
        # one session shrunk from a long history to a quarter
        {"name": "evict one", "op": "evict", **model, "page": 64, "seqs": 1,
         "single": 0, "hist_lo": 32000, "hist_hi": 32000, "new_lo": 0,
         "new_hi": 0, "keep": 8192, "recent": 256, "shape": 11},
        # a batch shrunk at once, some sequences already short enough
        {"name": "evict batch", "op": "evict", **model, "page": 16, "seqs": 24,
         "single": 0, "hist_lo": 900, "hist_hi": 9000, "new_lo": 0,
         "new_hi": 0, "keep": 2000, "recent": 100, "shape": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["heads", "attention", "attention", "weights", "evict"])
    heads, kv_heads, dim = rng.choice(
        [(16, 4, 128), (32, 8, 64), (16, 2, 128), (8, 8, 64), (12, 4, 128),
         (24, 8, 64)])
    case = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": rng.choice([16, 32, 48, 64, 128]),
            "shape": rng.randrange(1 << 20)}
    if op == "evict":
        case["seqs"] = _log(rng, 1, 24)
        case["hist_lo"] = _log(rng, 64, 8000)
        case["hist_hi"] = case["hist_lo"] + _log(rng, 1, 8000)
        case["keep"] = max(1, int(case["hist_hi"] * rng.uniform(0.1, 0.9)))
        case["recent"] = rng.randint(0, case["keep"])
        case.update(single=0, new_lo=0, new_hi=0)
        return case
    case["type"] = rng.choice(["f32", "f16", "bf16"])
    kind = rng.choice(["decode", "chunk", "mixed"])
    if kind == "decode":
        case["seqs"] = case["single"] = _log(rng, 1, 32)
        case.update(hist_lo=_log(rng, 1, 2000), new_lo=1, new_hi=1)
        case["hist_hi"] = case["hist_lo"] + _log(rng, 1, 20000)
    elif kind == "chunk":
        case["seqs"], case["single"] = rng.randint(1, 3), 0
        case["new_lo"] = _log(rng, 2, 400)
        case["new_hi"] = case["new_lo"] + _log(rng, 1, 800)
        case["hist_lo"] = _log(rng, 1, 4000)
        case["hist_hi"] = case["hist_lo"] + _log(rng, 1, 8000)
    else:
        case["seqs"] = rng.randint(3, 12)
        case["single"] = rng.randint(1, case["seqs"] - 1)
        case["new_lo"] = _log(rng, 2, 100)
        case["new_hi"] = case["new_lo"] + _log(rng, 1, 400)
        case["hist_lo"] = _log(rng, 1, 1000)
        case["hist_hi"] = case["hist_lo"] + _log(rng, 1, 4000)
    if op != "heads":
        case["window"] = rng.choice([0, 0, 0, rng.randint(1, 1000)])
    if op == "attention":
        case["gate"] = rng.random() < 0.5
    return case


def _shape(case):
    """(new rows, length with them) of each sequence: of the case alone."""
    rng = random.Random(case["shape"])
    new, lengths = [], []
    for s in range(case["seqs"]):
        n = rng.randint(case["new_lo"], case["new_hi"])
        n = 1 if s < case["single"] else n
        new.append(n)
        lengths.append(n + _log(rng, case["hist_lo"], case["hist_hi"]))
    order = list(range(case["seqs"]))
    rng.shuffle(order)
    return [new[i] for i in order], [lengths[i] for i in order]


def _pairs(case):
    """(visible (row, key) pairs of one head, cached rows some row sees)."""
    window, pairs, seen = case.get("window", 0), 0, 0
    for n, length in zip(*_shape(case)):
        first = length - n + 1  # keys the first new row sees without a window
        if window:
            short = max(0, min(n, window - first + 1))  # rows seeing < window
            pairs += short * first + short * (short - 1) // 2
            pairs += (n - short) * window
            seen += min(length, window + n - 1)
        else:
            pairs += n * first + n * (n - 1) // 2
            seen += length
    return pairs, seen


def work(case):
    new, lengths = _shape(case)
    rows, h, kv, d = sum(new), case["heads"], case["kv_heads"], case["dim"]
    size = 4 if case.get("type") == "f32" else 2
    if case["op"] == "heads":
        return {"bytes": rows * ((2 * h + 2 * kv) * d * size + 2 * kv * d * 2 + 4),
                "flops": rows * (h + kv) * d * 8}
    if case["op"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lengths)
        return {"bytes": sum(lengths) * 4 + kept * (2 * (2 * kv * d * 2) + 8),
                "flops": sum(lengths)}
    pairs, seen = _pairs(case)
    if case["op"] == "weights":
        return {"bytes": rows * h * (d * size + 4) + seen * kv * d * 2 +
                sum(lengths) * 8, "flops": pairs * h * d * 2}
    return {"bytes": rows * h * (2 * d * size + 4 + (size if case["gate"] else 0))
            + seen * kv * d * 2 * 2, "flops": pairs * h * d * 4}


# ---- inputs --------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    new, lengths = _shape(case)
    page, kv, d, h = case["page"], case["kv_heads"], case["dim"], case["heads"]
    seqs, rows = case["seqs"], sum(new)
    # the sequences' pages lie scattered in the pool; eviction has as many
    # free pages besides
    used = [-(-n // page) for n in lengths]
    width = max(used)
    copies = 2 if case["op"] == "evict" else 1
    pages = copies * sum(used) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    tables, at = [], 0
    for _ in range(copies):
        t = torch.zeros(seqs, width, dtype=torch.int32, device=dev)
        for s in range(seqs):
            t[s, :used[s]] = order[at:at + used[s]]
            at += used[s]
        tables.append(t)
    state = {
        "case": case, "table": tables[0],
        "lengths": torch.tensor(lengths, dtype=torch.int32, device=dev),
        "pages": pages, "width": width, "rows": rows, "max_rows": max(new),
        "starts": torch.tensor(np.concatenate([[0], np.cumsum(new)]),
                               dtype=torch.int32, device=dev),
        # row r is row row_off[r] of sequence row_seq[r]'s chunk
        "row_seq": torch.tensor(np.repeat(np.arange(seqs), new), device=dev),
        "row_off": torch.tensor(np.concatenate([np.arange(n) for n in new]),
                                dtype=torch.int64, device=dev),
    }

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev) * scale

    state["k"] = normal(pages, page, kv, d).half()
    state["v"] = normal(pages, page, kv, d).half()
    op = case["op"]
    if op == "evict":
        state["out_table"] = tables[1]
        # accumulated weights are heavy-tailed; some rows tie (never seen)
        w = torch.exp(normal(pages, page, scale=2.0))
        state["weights"] = torch.where(w < 0.05, torch.zeros_like(w), w)
        return state
    t = TYPES[case["type"]]
    state["q"] = normal(rows, h, d, scale=1.3).to(t)
    if op == "heads":
        state["knew"] = normal(rows, kv, d, scale=0.7).to(t)
        state["vnew"] = normal(rows, kv, d, scale=0.7).to(t)
        state["q_norm"] = 1 + normal(d, scale=0.1)
        state["k_norm"] = 1 + normal(d, scale=0.1)
        theta = torch.arange(d // 2, dtype=torch.float64, device=dev) * (-2.0 / d)
        state["freq"] = (1e6 ** theta).float()
        factors = torch.ones(d // 2, device=dev)
        factors[d // 4:] = 8.0  # far wavelengths are stretched
        state["factors"] = factors
        # evicted rows leave positions ahead of the cache's lengths
        pos = state["lengths"].long()[state["row_seq"]] + state["row_off"]
        state["positions"] = (pos + 1000).to(torch.int32)
        state["q_out"] = torch.empty_like(state["q"])
        return state
    if op == "attention" and case["gate"]:
        state["gate"] = normal(rows, h).to(t)
    if op == "weights":
        state["weights"] = torch.rand(pages, page, generator=g, device=dev)
        # the lse that the step's attention returned
        state["lse"] = _attention(state)[1]
    return state


# ---- plain forms ---------------------------------------------------------------

def _rows_of(s, table, count):
    """Pool rows of slots 0 .. count - 1 of every sequence [seqs][count]
    (slots past a sequence's pages: some row of the pool)."""
    page = s["case"]["page"]
    t = torch.arange(count, device=table.device)
    return table.long()[:, t // page] * page + t % page


def _scores(s):
    """(scores [seqs][kv][rows * group][slots] masked by -inf, pool rows)."""
    c = s["case"]
    kv, d, h, page = c["kv_heads"], c["dim"], c["heads"], c["page"]
    seqs, n, group = c["seqs"], s["max_rows"], h // kv
    slots = s["width"] * page
    idx = _rows_of(s, s["table"], slots)
    k = s["k"].view(-1, kv, d)[idx].float()
    i = torch.arange(n, device=idx.device)
    starts, lengths = s["starts"].long(), s["lengths"].long()
    src = (starts[:-1, None] + i).clamp(max=s["rows"] - 1)
    q = s["q"][src].float().view(seqs, n, kv, group, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(seqs, kv, n * group, d)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
    count = starts[1:] - starts[:-1]
    pos = (lengths - count)[:, None] + i  # a row's own slot
    t = torch.arange(slots, device=idx.device)
    seen = (t <= pos[:, :, None]) & (i < count[:, None])[:, :, None]
    if c["window"]:
        seen &= t > pos[:, :, None] - c["window"]
    hide = torch.where(seen, 0.0, -math.inf)
    x.view(seqs, kv, n, group, slots).add_(hide[:, None, :, None, :])
    return x, idx


def _per_row(s, x):
    """[seqs][kv][rows * group][...] back to the tensors' rows [rows][heads][...]."""
    c = s["case"]
    kv, n = c["kv_heads"], s["max_rows"]
    x = x.reshape(c["seqs"], kv, n, c["heads"] // kv, -1)
    x = x[s["row_seq"], :, s["row_off"]]
    return x.reshape(s["rows"], c["heads"], -1)


def _attention(s):
    c = s["case"]
    x, idx = _scores(s)
    m = x.amax(-1, keepdim=True).clamp(min=-3e38)
    p = x.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    v = s["v"].view(-1, c["kv_heads"], c["dim"])[idx].float()
    o = torch.matmul(p, v.permute(0, 2, 1, 3))
    o = o / total.clamp(min=1e-38)
    out = _per_row(s, o)
    if c.get("gate"):
        out = out / (1 + torch.exp(-s["gate"].float()))[:, :, None]
    lse = _per_row(s, m + torch.log(total))[:, :, 0].contiguous()
    return out.to(s["q"].dtype), lse


def _weights(s):
    c = s["case"]
    x, idx = _scores(s)
    kv, n, h = c["kv_heads"], s["max_rows"], c["heads"]
    i = torch.arange(n, device=x.device)
    starts, lengths = s["starts"].long(), s["lengths"].long()
    src = (starts[:-1, None] + i).clamp(max=s["rows"] - 1)
    lse = s["lse"][src].view(c["seqs"], n, kv, h // kv).permute(0, 2, 1, 3)
    p = x.sub_(lse.reshape(c["seqs"], kv, -1, 1)).exp_()
    got = p.sum((1, 2), dtype=torch.float64).float()
    t = torch.arange(x.shape[-1], device=x.device)
    old = lengths - (starts[1:] - starts[:-1])  # rows before this chunk
    pool = torch.cat([s["weights"].view(-1), s["weights"].new_zeros(1)])
    value = torch.where(t < old[:, None], pool[idx], 0.0) + got
    to = torch.where(t < lengths[:, None], idx, pool.numel() - 1)
    pool[to] = value
    return pool[:-1].view(s["weights"].shape)


def _heads(s):
    c = s["case"]
    d = c["dim"]
    angle = (s["positions"].double()[:, None] * s["freq"].double() /
             s["factors"].double())
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        a, b = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    q = turn(s["q"], s["q_norm"]).to(s["q"].dtype)
    # the new rows are the last of their sequences
    seq, kv = s["row_seq"], c["kv_heads"]
    slot = (s["lengths"].long() - (s["starts"][1:] - s["starts"][:-1]).long())[seq]
    slot = slot + s["row_off"]
    row = s["table"].long()[seq, slot // c["page"]] * c["page"] + slot % c["page"]
    s["k"].view(-1, kv, d)[row] = turn(s["knew"], s["k_norm"]).half()
    s["v"].view(-1, kv, d)[row] = s["vnew"].half()
    return q, s["k"], s["v"]


def _evict(s):
    c = s["case"]
    keep, recent, kv, d = c["keep"], c["recent"], c["kv_heads"], c["dim"]
    page, lengths = c["page"], s["lengths"].long()
    slots = s["width"] * page
    src = _rows_of(s, s["table"], slots)
    w = s["weights"].view(-1)[src]
    t = torch.arange(slots, device=w.device)
    # the last `recent` rows first, then by weight, then the empty slots
    w = torch.where(t >= lengths[:, None] - recent, math.inf, w)
    w = torch.where(t < lengths[:, None], w, -math.inf)
    top = torch.sort(w, dim=1, descending=True, stable=True)[1][:, :keep]
    count = lengths.clamp(max=keep)
    j = torch.arange(top.shape[1], device=w.device)
    top = torch.sort(torch.where(j < count[:, None], top, slots), dim=1)[0]
    live = j < count[:, None]
    kept = torch.full((c["seqs"], keep), -1, dtype=torch.int32, device=w.device)
    kept[:, :top.shape[1]] = torch.where(live, top, -1).to(torch.int32)
    dst = _rows_of(s, s["out_table"], top.shape[1])
    from_ = torch.where(live, src.gather(1, top.clamp(max=slots - 1)), dst)
    live = live.unsqueeze(-1)
    # slots past a sequence's rows point at pages of others: they go nowhere
    trash = s["weights"].numel()
    dst = torch.where(live[..., 0], dst, trash)
    pools = []
    for pool, shape in ((s["k"], (-1, kv, d)), (s["v"], (-1, kv, d)),
                        (s["weights"], (-1,))):
        flat = pool.view(shape)
        new = torch.cat([flat, torch.zeros_like(flat[:1])])
        new[dst] = flat[from_]
        pools.append(new[:-1].view(pool.shape))
    return pools[0], pools[1], pools[2], count.to(torch.int32), kept


# ---- the library's operators -----------------------------------------------------

def _own(s):
    import ctypes
    import importlib
    lfm3 = importlib.import_module("lfm3-gufo-extension_b200")
    lib, abi, c = lfm3.library(), lfm3.abi, s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    cache = abi.PagedCache(
        s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(),
        s["lengths"].data_ptr(), s["pages"], c["page"], c["kv_heads"],
        c["dim"], c["seqs"], s["width"], s["width"])
    at = ctypes.byref(cache)
    op = c["op"]
    if op == "evict":
        # eviction writes the pages of out_table and the weights' rows there
        kept = torch.full((c["seqs"], c["keep"]), -1, dtype=torch.int32,
                          device="cuda")
        lengths = torch.empty_like(s["lengths"])
        lfm3.check(lib.lfm3_cuda_paged_evict(
            at, s["out_table"].data_ptr(), lengths.data_ptr(),
            s["weights"].data_ptr(), kept.data_ptr(), c["keep"], c["recent"],
            stream))
        return s["k"], s["v"], s["weights"], lengths, kept
    kind, h, d, kv = ABI_TYPES[c["type"]], c["heads"], c["dim"], c["kv_heads"]
    positions = s["positions"].data_ptr() if op == "heads" else None
    batch = abi.PagedBatch(s["starts"].data_ptr(), positions, s["rows"],
                           s["max_rows"])
    rows = ctypes.byref(batch)
    if op == "heads":
        lfm3.check(lib.lfm3_cuda_paged_heads(
            at, rows, kind, s["q"].data_ptr(), h * d, s["knew"].data_ptr(),
            kv * d, s["vnew"].data_ptr(), kv * d, s["q_out"].data_ptr(), h * d,
            h, s["q_norm"].data_ptr(), s["k_norm"].data_ptr(),
            s["freq"].data_ptr(), s["factors"].data_ptr(), EPS, stream))
        return s["q_out"], s["k"], s["v"]
    if op == "attention":
        size = lib.lfm3_cuda_paged_attention_workspace_bytes(at, rows, h)
        space = torch.empty(size, dtype=torch.uint8, device="cuda")
        out = torch.empty_like(s["q"])
        lse = torch.empty(s["rows"], h, device="cuda")
        gate = s["gate"].data_ptr() if c["gate"] else None
        lfm3.check(lib.lfm3_cuda_paged_attention(
            at, rows, kind, s["q"].data_ptr(), h * d, gate, h, out.data_ptr(),
            h * d, lse.data_ptr(), h, c["window"], space.data_ptr(), size,
            stream))
        return out, lse
    size = lib.lfm3_cuda_paged_key_weights_workspace_bytes(at, rows, h)
    space = torch.empty(size, dtype=torch.uint8, device="cuda")
    weights = s["weights"].clone()  # the case is run again on its state
    lfm3.check(lib.lfm3_cuda_paged_key_weights(
        at, rows, kind, s["q"].data_ptr(), h * d, s["lse"].data_ptr(),
        weights.data_ptr(), h, c["window"], space.data_ptr(), size, stream))
    return weights


def run(state):
    if own:
        return _own(state)
    return {"heads": _heads, "attention": _attention, "weights": _weights,
            "evict": _evict}[state["case"]["op"]](state)


# ---- the definitions in 64 bits ----------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    page, kv, d, h = case["page"], case["kv_heads"], case["dim"], case["heads"]
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()

    def cached(pool, q, first, last):
        """Rows first .. last - 1 of sequence q, [rows][kv][d]."""
        table = s["table"][q].long()[:-(-last // page)]
        return pool[table].reshape(-1, kv, d)[first:last].double()

    if case["op"] == "heads":
        out = s["q"].double().clone()
        k, v = s["k"].double(), s["v"].double()
        for q, length in enumerate(lengths):
            b, e = starts[q], starts[q + 1]
            angle = s["positions"][b:e].double().unsqueeze(1) * s["freq"].double()
            angle = angle / s["factors"].double()
            z = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)

            def rotated(x, w):
                x = x.double()
                x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / d + EPS)
                x = x * w.double()
                y = torch.complex(x[..., :d // 2].contiguous(),
                                  x[..., d // 2:].contiguous()) * z
                return torch.cat([y.real, y.imag], -1)

            out[b:e] = rotated(s["q"][b:e], s["q_norm"])
            slot = torch.arange(length - (e - b), length, device="cuda")
            where = (s["table"][q].long()[slot // page], slot % page)
            k[where] = rotated(s["knew"][b:e], s["k_norm"])
            v[where] = s["vnew"][b:e].double()
        return out, k, v
    if case["op"] == "evict":
        weights = s["weights"].cpu().numpy().astype(np.float64)
        src, dst = s["table"].cpu().numpy(), s["out_table"].cpu().numpy()
        moved, kept = weights.copy(), np.full((case["seqs"], case["keep"]), -1)
        count = []
        for q, length in enumerate(lengths):
            w = weights[src[q, np.arange(length) // page],
                        np.arange(length) % page]
            old = max(0, length - case["recent"])
            free = case["keep"] - (length - old)
            best = np.lexsort((np.arange(old), -w[:old]))[:max(0, free)]
            chosen = np.sort(np.concatenate([best, np.arange(old, length)]))
            chosen = chosen[-case["keep"]:].astype(np.int64)
            kept[q, :chosen.size] = chosen
            count.append(chosen.size)
            j = np.arange(chosen.size)
            moved[dst[q, j // page], j % page] = w[chosen]
        # keys and values only move
        return None, None, torch.from_numpy(moved), torch.tensor(count), \
            torch.from_numpy(kept)
    group, window = h // kv, case["window"]
    out = torch.zeros(s["rows"], h, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["rows"], h, dtype=torch.float64, device="cuda")
    weights = s["weights"].double() if case["op"] == "weights" else None
    for q, length in enumerate(lengths):
        b, e = starts[q], starts[q + 1]
        n = e - b
        first = max(0, length - n - window + 1) if window else 0
        k = cached(s["k"], q, first, length)
        own_slot = torch.arange(length - n, length, device="cuda").unsqueeze(1)
        t = torch.arange(first, length, device="cuda").unsqueeze(0)
        hidden = t > own_slot
        if window:
            hidden = hidden | (t <= own_slot - window)
        gained = torch.zeros(length, dtype=torch.float64, device="cuda")
        values = cached(s["v"], q, first, length) if weights is None else None
        for head in range(h):
            x = s["q"][b:e, head].double() @ k[:, head // group].T / d ** 0.5
            x.masked_fill_(hidden, -math.inf)
            if weights is not None:
                x = x - s["lse"][b:e, head].double().unsqueeze(1)
                gained[first:] += x.exp().sum(0)
                continue
            z = torch.logsumexp(x, 1)
            lse[b:e, head] = z
            y = (x - z.unsqueeze(1)).exp() @ values[:, head // group]
            if case["gate"]:
                y = y * torch.sigmoid(s["gate"][b:e, head].double()).unsqueeze(1)
            out[b:e, head] = y
        if weights is not None:
            slot = torch.arange(length, device="cuda")
            where = (s["table"][q].long()[slot // page], slot % page)
            had = weights[where]
            had[length - n:] = 0
            weights[where] = had + gained
    return weights if weights is not None else (out, lse)
