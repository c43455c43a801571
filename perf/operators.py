"""The paged KV cache's operators as a serving program calls them: append of new rows to pages, attention of one new
token per sequence over its pages (with and without accumulating the attention weights), and eviction of the rows
with the least accumulated weight.

Pages are FP16, [page][layer][K|V][kv_head][row][128]; a sequence's rows are listed by a table of page ids; attention
weights are FP32, [page][layer][kv_head][row]. Query heads are twice the KV heads. With ``own`` the framework's calls
run; without it, the same results come from elementary torch operations in 32 bits.
"""
import math
import random

import torch

own = False

D, GROUP = 128, 2
EPS, THETA = 1e-6, 1e6


# ---- cases ---------------------------------------------------------------------------------------
def listed():
    return [
        # one new token in one layer: an engine's layer loop, single user; latency counts
        {"name": "append_token_1layer", "op": "append", "n": 1, "seqs": 1, "layers": 1, "hkv": 8, "page": 16, "pos0": 4000, "padded": 0},
        # one token for each of 64 users, every layer, caches kept short by eviction while positions go on
        {"name": "append_batch64_28layers", "op": "append", "n": 64, "seqs": 64, "layers": 28, "hkv": 8, "page": 16, "pos0": 20000, "padded": 3},
        # prompts of several users (ragged, 3968 rows in all) into pages, every layer
        {"name": "append_prompts_3968x28", "op": "append", "n": 3968, "seqs": 5, "layers": 28, "hkv": 8, "page": 64, "pos0": 0, "padded": 0},
        # one layer of one user's step in a short chat; latency counts
        {"name": "attn_1layer_452", "op": "attn", "n": 1, "rows": 452, "ragged": False, "padded": 0, "layers": 1, "hkv": 8, "page": 16, "add_weights": False},
        # one user's step, every layer, near the end of a 4K context
        {"name": "attn_28layers_3970", "op": "attn", "n": 1, "rows": 3970, "ragged": False, "padded": 0, "layers": 28, "hkv": 8, "page": 32, "add_weights": False},
        # one layer of a batch of 64 users with histories of any length and two padded rows
        {"name": "attn_batch64_ragged", "op": "attn", "n": 64, "rows": 4096, "ragged": True, "padded": 2, "layers": 1, "hkv": 8, "page": 16, "add_weights": False},
        # two very long histories, one layer
        {"name": "attn_long_131071", "op": "attn", "n": 2, "rows": 131071, "ragged": True, "padded": 0, "layers": 1, "hkv": 8, "page": 64, "add_weights": False},
        # the same kinds of step while the weights for a later eviction are gathered
        {"name": "attn_weights_28layers_2049", "op": "attn", "n": 1, "rows": 2049, "ragged": False, "padded": 0, "layers": 28, "hkv": 8, "page": 16, "add_weights": True},
        {"name": "attn_weights_batch33", "op": "attn", "n": 33, "rows": 3001, "ragged": True, "padded": 1, "layers": 1, "hkv": 4, "page": 128, "add_weights": True},
        # eviction after a prompt in one layer's cache
        {"name": "evict_1layer_1025", "op": "evict", "n": 1, "rows": 1025, "ragged": False, "layers": 1, "hkv": 8, "page": 16, "keep": 512, "recent": 64},
        # one user's full 4K cache halved, every layer
        {"name": "evict_28layers_4096", "op": "evict", "n": 1, "rows": 4096, "ragged": False, "layers": 28, "hkv": 8, "page": 32, "keep": 2048, "recent": 256},
        # a batch of users brought under one budget; some are under it already
        {"name": "evict_batch24_ragged", "op": "evict", "n": 24, "rows": 2777, "ragged": True, "layers": 4, "hkv": 8, "page": 16, "keep": 1000, "recent": 37},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append", "attn", "attn", "attn", "evict", "evict"])
    hkv = rng.choice([1, 2, 4, 8, 8])
    layers = rng.choice([1, 2, 3, 7, 28])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "append":
        if rng.random() < 0.5:          # one token per sequence
            n = _log(rng, 1, 200)
            return {"op": op, "n": n, "seqs": n, "layers": layers, "hkv": hkv, "page": page if n < 32 else 16,
                    "pos0": rng.randrange(0, 30000), "padded": rng.randrange(0, 3) if n > 4 else 0}
        n = _log(rng, 2, 3968)          # prompts
        return {"op": op, "n": n, "seqs": rng.randrange(1, min(n, 9) + 1), "layers": layers, "hkv": hkv, "page": page,
                "pos0": rng.randrange(0, 2000), "padded": 0}
    if op == "attn":
        n = _log(rng, 1, 128)
        rows = _log(rng, 1, min(131072, max(1, 1500000 // (n * layers * hkv))))
        return {"op": op, "n": n, "rows": rows, "ragged": rng.random() < 0.7, "padded": rng.randrange(0, 3) if n > 4 else 0,
                "layers": layers, "hkv": hkv, "page": page, "add_weights": rng.random() < 0.4}
    n = _log(rng, 1, 32)
    rows = _log(rng, 4, min(40000, max(4, 700000 // (n * layers * hkv))))
    keep = max(1, int(rows * rng.uniform(0.1, 0.9)))
    return {"op": op, "n": n, "rows": rows, "ragged": rng.random() < 0.5, "layers": layers, "hkv": hkv, "page": page,
            "keep": keep, "recent": rng.randrange(0, keep + 1) if rng.random() < 0.5 else keep // 8}


def _lengths(case):
    """Rows of each sequence: the longest first, the others anywhere below it where the case is ragged; padded rows hold 0."""
    r = random.Random("%s %d %d" % (case["op"], case["n"], case["rows"]))
    n, top = case["n"], case["rows"]
    got = [top] + [r.randrange(1, top + 1) if case["ragged"] else top for _ in range(n - 1)]
    for i in range(case.get("padded", 0)):
        got[n - 1 - 2 * i] = 0
    return got


def _append_rows(case):
    """(sequence, rows its sequence holds with this one, RoPE position) of each new row."""
    r = random.Random("append %d %d %d" % (case["n"], case["seqs"], case["pos0"]))
    n, seqs = case["n"], case["seqs"]
    if seqs == n:                                       # one token each; caches of 1 to 128 rows
        held = [r.randrange(1, 129) for _ in range(n)]
        for i in range(case["padded"]):
            held[n - 1 - 2 * i] = 0
        return list(range(n)), held, [case["pos0"] + r.randrange(0, 2000) for _ in range(n)]
    cuts = [0] + sorted(r.sample(range(1, n), seqs - 1)) + [n]
    seq, held, pos = [], [], []
    for s in range(seqs):
        m = cuts[s + 1] - cuts[s]
        seq += [s] * m
        held += range(1, m + 1)
        pos += range(case["pos0"], case["pos0"] + m)
    return seq, held, pos


def _ceil(a, b):
    return -(-a // b)


# ---- inputs --------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dev, layers, hkv, page = "cuda", case["layers"], case["hkv"], case["page"]

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, device=dev, dtype=dtype, generator=g)

    def i32(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    def table_of(cols_used, first, cols):
        """Pages handed out in a shuffled order, as after a while of allocating and freeing."""
        total = sum(cols_used)
        ids = (torch.randperm(total, device=dev, generator=g) + first).to(torch.int32)
        table = torch.zeros(len(cols_used), cols, dtype=torch.int32, device=dev)
        at = 0
        for b, c in enumerate(cols_used):
            table[b, :c] = ids[at:at + c]
            at += c
        return table, total

    s = dict(case)
    if case["op"] == "append":
        seq, held, pos = _append_rows(case)
        most = [1] * case["seqs"]
        for b, h in zip(seq, held):
            most[b] = max(most[b], h)
        used = [_ceil(m, page) for m in most]
        s["table"], pages = table_of(used, 0, max(used))
        n = case["n"]
        s["kv"] = torch.zeros(pages, layers, 2, hkv, page, D, dtype=torch.float16, device=dev)
        s["row_seq"], s["row_len"], s["row_pos"] = i32(seq), i32(held), i32(pos)
        # rows as projections give them: channels of unlike size, before their normalisation
        s["q"] = randn(layers, n, GROUP * hkv, D) * 1.7
        s["k"] = randn(layers, n, hkv, D) * 0.6
        s["v"] = randn(layers, n, hkv, D)
        s["norms"] = 1 + 0.3 * randn(layers, 2, D)
        s["q_out"] = torch.zeros_like(s["q"])
    else:
        lengths = _lengths(case)
        used = [_ceil(max(m, 1), page) for m in lengths]
        s["table"], pages = table_of(used, 0, max(used))
        s["lengths"], s["cols"] = i32(lengths), max(used)
        n = case["n"]
        if case["op"] == "attn":
            s["kv"] = randn(pages, layers, 2, hkv, page, D, dtype=torch.float16)
            # normalised queries whose norm weights are above one: some rows take much of the weight
            s["q"] = 2.5 * randn(layers, n, GROUP * hkv, D)
            s["out"] = torch.empty_like(s["q"])
            if case["add_weights"]:
                s["weights0"] = 0.1 * torch.rand(pages, layers, hkv, page, device=dev, generator=g)
                s["weights"] = torch.empty_like(s["weights0"])
        else:
            keep = case["keep"]
            kept_cols = _ceil(keep, page)
            s["dst"], more = table_of([kept_cols] * n, pages, kept_cols)
            s["kv"] = randn(pages + more, layers, 2, hkv, page, D, dtype=torch.float16)
            # few heavy rows, many light ones, and a tenth that no query looked at (ties)
            w = torch.rand(pages + more, layers, hkv, page, device=dev, generator=g) ** 6
            s["weights"] = w * (torch.rand(w.shape, device=dev, generator=g) > 0.1)
            s["kept"] = torch.empty(n, layers, hkv, keep, dtype=torch.int32, device=dev)
            s["new_lengths"] = torch.empty(n, dtype=torch.int32, device=dev)
    if own:
        from fpga_qwen_b200 import qattn
        ctx = qattn.Context(n_layers=layers, n_q_heads=GROUP * hkv, n_kv_heads=hkv, context=1)
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        if case["op"] == "append":
            ctx.rope_positions(32768)
            for layer, w in enumerate(s["norms"].cpu().numpy()):
                ctx.set_norms(layer, w[0].ctypes.data, w[1].ctypes.data)
        if case["op"] == "attn":
            s["bytes"] = ctx.paged_workspace(case["n"], layers, s["cols"] * page, case["add_weights"])
            s["workspace"] = torch.empty(s["bytes"], dtype=torch.uint8, device=dev)
        weights = s["weights"].data_ptr() if "weights" in s else 0
        s["ctx"], s["pages"] = ctx, qattn.Pages(s["kv"].data_ptr(), weights, s["kv"].shape[0], page)
    return s


# ---- the operators -------------------------------------------------------------------------------
def run(s):
    if s["op"] == "append":
        return _append(s)
    if s["op"] == "attn":
        return _attn(s)
    return _evict(s)


def _append(s):
    if own:
        s["ctx"].paged_append(s["pages"], s["table"].data_ptr(), s["seqs"], s["table"].shape[1], s["row_seq"].data_ptr(),
                              s["row_len"].data_ptr(), s["row_pos"].data_ptr(), s["n"], 0, s["layers"],
                              s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["q_out"].data_ptr())
        return s["q_out"], s["kv"]
    kv, page, dev = s["kv"], s["page"], s["kv"].device
    j = torch.arange(D // 2, device=dev, dtype=torch.float64)
    angle = s["row_pos"].double()[:, None] / THETA ** (2.0 * j / D)
    cos, sin = torch.cos(angle).float()[None, :, None], torch.sin(angle).float()[None, :, None]

    def norm_rope(x, w):
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w[:, None, None]
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    q = norm_rope(s["q"], s["norms"][:, 0])
    k = norm_rope(s["k"], s["norms"][:, 1])
    there = s["row_len"] > 0
    q = torch.where(there[None, :, None, None], q, torch.zeros((), device=dev))
    at = (s["row_len"] - 1).clamp(min=0).long()
    ids = s["table"].long()[s["row_seq"].long(), at // page]
    layer = torch.arange(s["layers"], device=dev)[:, None, None]
    head = torch.arange(s["hkv"], device=dev)[None, None]
    for half, rows in ((0, k), (1, s["v"])):
        to = (ids[None, :, None], layer, half, head, (at % page)[None, :, None])
        kv[to] = torch.where(there[None, :, None, None], rows.half(), kv[to])
    return q, kv


def _attn(s):
    weights = s.get("weights")
    if weights is not None:
        weights.copy_(s["weights0"])       # a pass adds to the weights: every pass starts from the same ones
    if own:
        s["ctx"].paged_attn(s["pages"], s["table"].data_ptr(), s["cols"], s["lengths"].data_ptr(), s["n"], 0, s["layers"],
                            s["q"].data_ptr(), s["out"].data_ptr(), weights is not None, s["workspace"].data_ptr(), s["bytes"])
        return (s["out"],) if weights is None else (s["out"], weights)
    n, layers, hkv, page, cols = s["n"], s["layers"], s["hkv"], s["page"], s["cols"]
    ids = s["table"].long()
    rows = s["kv"][ids].permute(3, 0, 2, 4, 1, 5, 6).reshape(2, n, layers, hkv, cols * page, D).float()
    q = s["q"].view(layers, n, hkv, GROUP, D).transpose(0, 1)
    logits = q @ rows[0].transpose(-1, -2) / math.sqrt(D)
    there = torch.arange(cols * page, device=q.device) < s["lengths"][:, None]
    there = there[:, None, None, None]
    logits = logits.masked_fill(~there, -math.inf)
    most = logits.amax(-1, keepdim=True)
    p = torch.where(there, torch.exp(logits - most), torch.zeros((), device=q.device))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros((), device=q.device))
    out = (p @ rows[1]).transpose(0, 1).reshape(layers, n, GROUP * hkv, D)
    if weights is None:
        return (out,)
    add = p.sum(3).view(n, layers, hkv, cols, page).permute(0, 3, 1, 2, 4)
    weights.index_add_(0, ids.flatten(), add.reshape(n * cols, layers, hkv, page))
    return out, weights


def _evict(s):
    if own:
        s["ctx"].paged_evict(s["pages"], s["table"].data_ptr(), s["cols"], s["dst"].data_ptr(), s["dst"].shape[1],
                             s["lengths"].data_ptr(), s["new_lengths"].data_ptr(), s["n"], s["keep"], s["recent"],
                             s["kept"].data_ptr())
        return s["kv"], s["weights"], s["new_lengths"], s["kept"]
    kv, weights, dev = s["kv"], s["weights"], s["kv"].device
    n, layers, hkv, page, cols, keep = s["n"], s["layers"], s["hkv"], s["page"], s["cols"], s["keep"]
    w = weights[s["table"].long()].permute(0, 2, 3, 1, 4).reshape(n, layers, hkv, cols * page)
    t = torch.arange(cols * page, device=dev)
    length = s["lengths"][:, None, None, None]
    w = w.masked_fill(t >= length - s["recent"], math.inf).masked_fill(t >= length, -1.0)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :keep]
    if order.shape[-1] < keep:
        order = torch.cat([order, order.new_full((n, layers, hkv, keep - order.shape[-1]), cols * page)], -1)
    slot = torch.arange(keep, device=dev)
    there = slot < length
    kept = torch.sort(torch.where(there, order, cols * page), dim=-1).values
    to = (s["dst"].long()[:, slot // page][:, None, None], slot % page)
    source = torch.where(there, kept, 0)
    row = torch.arange(n, device=dev)[:, None, None, None]
    layer = torch.arange(layers, device=dev)[None, :, None, None]
    head = torch.arange(hkv, device=dev)[None, None, :, None]
    ids = torch.where(there, s["table"].long()[row, source // page], to[0])
    at = torch.where(there, source % page, to[1])
    weights[to[0], layer, head, to[1]] = weights[ids, layer, head, at]
    kv[to[0], layer, 0, head, to[1]] = kv[ids, layer, 0, head, at]
    kv[to[0], layer, 1, head, to[1]] = kv[ids, layer, 1, head, at]
    kept = torch.where(there, kept, -1).int()
    return kv, weights, s["lengths"].clamp(max=keep), kept


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    layers, hkv = case["layers"], case["hkv"]
    if case["op"] == "append":
        n = sum(1 for h in _append_rows(case)[1] if h)
        return {"bytes": n * layers * hkv * D * (2 * 4 * GROUP + 2 * 4 + 2 * 2) + 12 * n, "flops": n * layers * hkv * D * 10 * (GROUP + 1)}
    keys = sum(_lengths(case)) * layers * hkv
    if case["op"] == "attn":
        rows = case["n"] * layers * hkv * GROUP
        return {"bytes": keys * (512 + (8 if case["add_weights"] else 0)) + rows * D * 8, "flops": keys * GROUP * D * 4}
    kept = sum(min(m, case["keep"]) for m in _lengths(case)) * layers * hkv
    return {"bytes": keys * 4 + kept * (2 * 512 + 8), "flops": 0}


# ---- 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    """The operators from their definitions, one sequence at a time, in 64 bits."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    kv, page, layers, hkv = s["kv"], case["page"], case["layers"], case["hkv"]
    if case["op"] == "append":
        out, pool = torch.zeros_like(s["q"], dtype=torch.float64), kv.double()
        seq, held, pos = _append_rows(case)
        place = [(r, int(s["table"][b, (h - 1) // page]), (h - 1) % page, p) for r, (b, h, p) in enumerate(zip(seq, held, pos)) if h]
        r, ids, at, p = (torch.tensor(v, device=kv.device) for v in zip(*place))
        freq = torch.tensor([THETA ** (-2.0 * j / D) for j in range(D // 2)], dtype=torch.float64, device=kv.device)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=kv.device), p.double()[:, None] * freq)
        for layer in range(layers):
            for name, which in (("q", 0), ("k", 1)):
                x = s[name][layer, r].double()
                x = x * (x.square().sum(-1, keepdim=True) / D + EPS).rsqrt() * s["norms"][layer, which].double()
                z = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous()) * turn[:, None]
                z = torch.cat([z.real, z.imag], -1)
                if which == 0:
                    out[layer, r] = z
                else:
                    pool[ids, layer, 0, :, at] = z
            pool[ids, layer, 1, :, at] = s["v"][layer, r].double()
        return out, pool
    lengths, table = _lengths(case), s["table"].long()
    if case["op"] == "attn":
        out = torch.zeros_like(s["q"], dtype=torch.float64)
        total = s["weights0"].double() if case["add_weights"] else None
        for b, m in enumerate(lengths):
            ids = table[b, :_ceil(m, page)]
            for layer in range(layers if m else 0):
                k, v = (kv[ids, layer, i].double().transpose(0, 1).reshape(hkv, -1, D)[:, :m] for i in (0, 1))
                q = s["q"][layer, b].double().view(hkv, GROUP, D)
                p = torch.softmax(torch.einsum("hgd,htd->hgt", q, k) / math.sqrt(D), -1)
                out[layer, b] = torch.einsum("hgt,htd->hgd", p, v).reshape(GROUP * hkv, D)
                if total is not None:
                    t = torch.arange(m, device=kv.device)
                    total[ids[t // page], layer, :, t % page] += p.sum(1).T
        return (out,) if total is None else (out, total)
    keep, recent = case["keep"], case["recent"]
    pool, weights = kv.double(), s["weights"].double()
    kept = torch.full((case["n"], layers, hkv, keep), -1, dtype=torch.int32, device=kv.device)
    slots = torch.arange(keep, device=kv.device)
    for b, m in enumerate(lengths):
        c = min(m, keep)
        to, to_row = s["dst"][b].long()[slots[:c] // page], slots[:c] % page
        for layer in range(layers):
            w = s["weights"][table[b, :_ceil(m, page)], layer].transpose(0, 1).reshape(hkv, -1)[:, :m].cpu().tolist()
            for h in range(hkv):
                old = range(max(0, m - recent)) if m > keep else range(m)
                best = sorted(old, key=lambda i: (-w[h][i], i))[:keep - recent] if m > keep else list(old)
                mine = torch.tensor(sorted(best) + (list(range(m - recent, m)) if m > keep else []), device=kv.device)
                kept[b, layer, h, :c] = mine.int()
                ids, at = table[b][mine // page], mine % page
                pool[to, layer, :, h, to_row] = kv[ids, layer, :, h, at].double()
                weights[to, layer, h, to_row] = s["weights"][ids, layer, h, at].double()
    return pool, weights, torch.tensor([min(m, keep) for m in lengths], dtype=torch.int32, device=kv.device), kept
