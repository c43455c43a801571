"""GPU: the paged KV cache (qa_paged_append, qa_paged_attn, qa_paged_evict) against the oracle, 64-bit
arithmetic and the slot calls.

Tolerances count roundings of at most half a step, u = 2^-24 relative in FP32, summed as a random
walk, with a factor of 8 on top:
* a logit is a chain of 128 fused multiply-adds whose partial sums are about the 2-norm P of its 128
  products, so it is off by u * sqrt(128) * P (and u times its own size for the scale), absolutely,
  and that is the relative error of its softmax weight;
* a weight passes through exp2f and one rescaling per 16-row block that raises the maximum (at most
  a few u each): u * (8 + sqrt(L / 16)); the sums over L rows add u * sqrt(L) to either factor;
* so an output is off by that relative error times sum_t p_t |v_t|, and an accumulated weight by it
  times the weight, plus u times the sum for its addition.
Copies, indices and FP16 rows are compared bit for bit.
"""
import math

import numpy as np
import pytest
import torch

from fpga_qwen_b200 import qattn
from oracle import oracle as O
from tests import helpers as H

pytestmark = pytest.mark.gpu

D, U = 128, 2.0 ** -24


def make(layers=1, hkv=8, context=1, **kw):
    ctx = qattn.Context(n_layers=layers, n_q_heads=2 * hkv, n_kv_heads=hkv, context=context, **kw)
    if not kw.get("io_host"):
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    return ctx


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Cache:
    """A pool of pages handed out in shuffled order, with junk (NaN, infinities) in every row that
    no sequence holds and in spare pages."""

    def __init__(self, lengths, layers=1, hkv=8, page=16, seed=0, spare=3, extra_cols=1, weights=True, room=0):
        g = torch.Generator("cuda").manual_seed(seed)
        self.lengths, self.layers, self.hkv, self.page = list(lengths), layers, hkv, page
        used = [-(-max(m + room, 1) // page) for m in lengths]
        self.cols = max(used) + extra_cols
        self.n_pages = sum(used) + spare
        ids = torch.randperm(self.n_pages, device="cuda", generator=g)[:sum(used)].to(torch.int32)
        self.table = torch.full((len(used), self.cols), -7, dtype=torch.int32, device="cuda")   # past the end: never read
        at = 0
        for b, c in enumerate(used):
            self.table[b, :c] = ids[at:at + c]
            at += c
        junk = torch.tensor([float("nan"), float("inf"), float("-inf"), 60000.0], dtype=torch.float16, device="cuda")
        self.kv = junk[torch.randint(0, 4, (self.n_pages, layers, 2, hkv, page, D), device="cuda", generator=g)]
        self.w = torch.full((self.n_pages, layers, hkv, page), float("nan"), device="cuda") if weights else None
        for b, m in enumerate(lengths):
            rows = torch.randn(layers, 2, hkv, m, D, device="cuda", generator=g).half()
            self.put(b, rows)
            if weights:
                self.put_weights(b, torch.rand(layers, hkv, m, device="cuda", generator=g))
        self.g = g

    def where(self, b, m):
        t = torch.arange(m, device="cuda")
        return self.table[b].long()[t // self.page], t % self.page

    def put(self, b, rows):
        ids, at = self.where(b, rows.shape[3])
        self.kv[ids, :, :, :, at] = rows.permute(3, 0, 1, 2, 4)

    def put_weights(self, b, w):
        ids, at = self.where(b, w.shape[2])
        self.w[ids, :, :, at] = w.permute(2, 0, 1)

    def rows(self, b, m=None):
        ids, at = self.where(b, self.lengths[b] if m is None else m)
        return self.kv[ids, :, :, :, at].permute(1, 2, 3, 0, 4)          # [layers][2][hkv][m][128]

    def weights(self, b, m=None):
        ids, at = self.where(b, self.lengths[b] if m is None else m)
        return self.w[ids, :, :, at].permute(1, 2, 0)

    @property
    def pages(self):
        return qattn.Pages(self.kv.data_ptr(), self.w.data_ptr() if self.w is not None else 0, self.n_pages, self.page)

    def query(self, layers=None, scale=1.5):
        return scale * torch.randn(layers or self.layers, len(self.lengths), 2 * self.hkv, D, device="cuda", generator=self.g)


def attend(ctx, c, q, layer=0, add=False, lengths=None, out=None):
    nl, n = q.shape[:2]
    out = torch.full_like(q, float("nan")) if out is None else out
    size = ctx.paged_workspace(n, nl, c.cols * c.page, add)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    lens = i32(c.lengths) if lengths is None else lengths
    ctx.paged_attn(c.pages, c.table.data_ptr(), c.cols, lens.data_ptr(), n, layer, nl, q.data_ptr(), out.data_ptr(), add,
                   ws.data_ptr(), size)
    return out


def reference(c, q, layer=0):
    """(out, tolerance of out, {b: (weights, relative error)}) in 64 bits."""
    nl, n = q.shape[:2]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    probs = {}
    for b in range(n):
        m = c.lengths[b]
        if not m:
            continue
        k, v = c.rows(b)[layer:layer + nl].double().unbind(1)
        qb = q[:, b].double().view(nl, c.hkv, 2, D)
        s = torch.einsum("lhgd,lhtd->lhgt", qb, k) / math.sqrt(D)
        part = torch.einsum("lhgd,lhtd->lhgt", qb ** 2, k ** 2).sqrt() / math.sqrt(D)
        rel = (U * (math.sqrt(D) * part + 2 * s.abs())).amax(-1) + U * (16 + math.sqrt(m / 16) + 2 * math.sqrt(m))
        p = torch.softmax(s, -1)
        out[:, b] = torch.einsum("lhgt,lhtd->lhgd", p, v).reshape(nl, -1, D)
        tol[:, b] = 8 * (rel[..., None] * torch.einsum("lhgt,lhtd->lhgd", p, v.abs())).reshape(nl, -1, D)
        probs[b] = (p.sum(2), 8 * (rel[..., None] * p).sum(2))
    return out, tol, probs


def check_attend(ctx, c, q, layer=0, add=False):
    nl = q.shape[0]
    before = [c.weights(b).clone() for b in range(len(c.lengths))] if add else None
    kv = c.kv.clone()
    w_all = c.w.clone() if add else None
    out = attend(ctx, c, q, layer, add)
    ctx.sync()
    want, tol, probs = reference(c, q, layer)
    off = (out.double() - want).abs()
    assert bool((off <= tol).all()), (float((off / tol.clamp(min=1e-30)).max()), float(off.max()))
    assert torch.equal(c.kv.view(torch.int16), kv.view(torch.int16))
    for b, m in enumerate(c.lengths):
        if m == 0:
            assert not out[:, b].any()
    if add:
        for b, (p, p_tol) in probs.items():
            got, old = c.weights(b).double(), before[b].double()
            want_w = old.clone()
            want_w[layer:layer + nl] += p
            limit = torch.zeros_like(old)
            limit[layer:layer + nl] = p_tol + 2 * U * want_w[layer:layer + nl]
            assert bool(((got - want_w).abs() <= limit).all()), b
            c.put_weights(b, before[b])
        assert torch.equal(c.w.view(torch.int32), w_all.view(torch.int32))      # nothing else was touched
    return out


# ---- attention -----------------------------------------------------------------------------------
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 512])
def test_attention_lengths_around_blocks_and_pages(page, add):
    lengths = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 0, 127, 128, 129, 255, 257, 511, 512, 513, 1000, 0]
    ctx = make()
    c = Cache(lengths, page=page, seed=page)
    check_attend(ctx, c, c.query(), add=add)


@pytest.mark.parametrize("hkv", [1, 2, 4, 8])
@pytest.mark.parametrize("layers,lengths", [(1, [1]), (1, [4096]), (3, [700, 5]), (28, [300]), (28, [1]), (2, [0, 3000, 0, 77])])
def test_attention_heads_and_layers(hkv, layers, lengths):
    ctx = make(layers, hkv)
    c = Cache(lengths, layers, hkv, page=32, seed=hkv)
    check_attend(ctx, c, c.query(), add=True)
    check_attend(ctx, c, c.query(), add=False)


def test_attention_on_a_layer_range():
    ctx = make(5, 4)
    c = Cache([90, 333], 5, 4, seed=3)
    check_attend(ctx, c, c.query(2), layer=2, add=True)
    check_attend(ctx, c, c.query(1), layer=4)


@pytest.mark.parametrize("add", [False, True])
def test_attention_long_history(add):
    ctx = make(1, 2)
    c = Cache([200001, 3], 1, 2, page=64, seed=5)
    check_attend(ctx, c, c.query(), add=add)


def test_attention_batch_of_1024_with_empty_rows():
    ctx = make(2, 2)
    r = np.random.default_rng(0)
    lengths = [int(x) for x in r.integers(0, 90, 1024)]
    c = Cache(lengths, 2, 2, seed=6)
    check_attend(ctx, c, c.query(), add=True)


def test_attention_all_rows_empty():
    ctx = make(2, 8)
    c = Cache([0] * 5, 2, 8, seed=7)
    out = attend(ctx, c, c.query(), add=True)
    ctx.sync()
    assert not out.any()


def test_rows_that_share_pages():
    """Three queries over one sequence's pages (a row with a shorter length among them): weights add up."""
    ctx = make(2, 4)
    c = Cache([500], 2, 4, page=32, seed=8)
    c.table = c.table.expand(3, -1).contiguous()
    c.lengths = [500, 41, 500]
    before = c.weights(0).clone().double()
    q = c.query()
    out = attend(ctx, c, q, add=True)
    ctx.sync()
    want, tol, probs = reference(c, q)
    assert bool(((out.double() - want).abs() <= tol).all())
    total, limit = before.clone(), torch.zeros_like(before)
    for b, m in enumerate(c.lengths):
        total[:, :, :m] += probs[b][0]
        limit[:, :, :m] += probs[b][1]
    assert bool(((c.weights(0).double() - total).abs() <= limit + 4 * U * total).all())


def test_infinities_and_nan_in_rows_follow_ieee():
    """An infinite or NaN value or key shows in its own head's output, as in the formula, and nowhere else."""
    ctx = make(1, 8)
    c = Cache([700], 1, 8, seed=9)
    rows = c.rows(0).clone()
    rows[0, 1, 1, 5, 7] = float("inf")                  # a value: channel 7 of heads 2, 3 is +inf
    rows[0, 0, 2, 600] = float("nan")                   # a key: heads 4, 5 are NaN
    rows[0, 0, 3] = 0.0
    rows[0, 0, 3, :, 0] = float("-inf")                 # every logit of heads 6, 7: -inf (q channel 0 > 0), NaN
    rows[0, 0, 4, :650] = 0.0
    rows[0, 0, 4, :650, 0] = float("-inf")              # all but the last 50 rows of heads 8, 9 masked away
    c.put(0, rows)
    q = c.query()
    q[..., 0] = q[..., 0].abs() + 0.1
    out = attend(ctx, c, q)
    ctx.sync()
    k, v = c.rows(0)[0].double().unbind(0)
    s = torch.einsum("hgd,htd->hgt", q[0, 0].double().view(8, 2, D), k) / math.sqrt(D)
    p = torch.softmax(s, -1)
    want = torch.einsum("hgt,htd->hgd", p, v).reshape(16, D)
    got = out[0, 0].double()
    assert torch.equal(torch.isnan(want), torch.isnan(got)) and torch.equal(torch.isinf(want), torch.isinf(got))
    fine = torch.isfinite(want)
    # logits of at most 40 in size and sums over 700 rows: U * (sqrt(128) * 40 + 2 * sqrt(700) + ...) * 8 < 4e-4 of |v| <= 5
    assert float((want - got)[fine].abs().max()) < 2e-3
    assert bool(torch.isfinite(got[8:10]).all())


def test_extreme_logits():
    """Softmax weights of one row only (logits hundreds apart) and equal logits."""
    ctx = make(1, 8)
    c = Cache([900], 1, 8, seed=10)
    check_attend(ctx, c, c.query(scale=200.0), add=True)
    check_attend(ctx, c, torch.zeros_like(c.query()), add=True)


def test_attention_equals_the_slot_decode():
    """The same rows in a slot and in pages: qa_paged_append's bits are qa_append's, outputs agree."""
    L, n = 3, 700
    ctx = make(L, 8, context=1024)
    qw, kw = H.norms(21, L)
    H.set_norms(ctx, qw, kw)
    q, k, v = H.inputs(21, L, 0, n)
    qn = torch.empty_like(q)
    ctx.append(0, 0, L, 0, n, q.data_ptr(), k.data_ptr(), v.data_ptr(), qn.data_ptr())
    c = Cache([0], L, 8, page=64, seed=11, room=n)
    pn = torch.empty_like(q)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    seq, held = torch.zeros_like(pos), pos + 1
    ctx.paged_append(c.pages, c.table.data_ptr(), 1, c.cols, seq.data_ptr(), held.data_ptr(), pos.data_ptr(), n, 0, L,
                     q.data_ptr(), k.data_ptr(), v.data_ptr(), pn.data_ptr())
    assert torch.equal(qn, pn)
    c.lengths = [n]
    got = c.rows(0).cpu().numpy().view(np.uint16)
    for layer in range(L):
        for h in range(8):
            for kv in (0, 1):
                assert np.array_equal(got[layer, kv, h], H.read_plane(ctx, 0, layer, kv, h, 0, n))
    assert not c.weights(0).any()                       # new rows start without weight
    last = qn[:, n - 1:].contiguous()
    slot_out = torch.empty_like(last)
    ctx.commit(0, n - 1)
    ctx.attn_decode(0, 0, L, n - 1, 1, last.data_ptr(), slot_out.data_ptr())
    out = attend(ctx, c, last)
    want, tol, _ = reference(c, last)
    ctx.sync()
    assert bool(((out.double() - want).abs() <= tol).all()) and bool(((slot_out.double() - want).abs() <= tol).all())


def test_attention_is_reproducible_and_graph_replays_with_new_lengths():
    ctx = make(4, 8)
    c = Cache([300, 0, 2000], 4, 8, seed=12)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ctx.set_stream(stream.cuda_stream)
    with torch.cuda.stream(stream):
        q, lens = c.query(), i32(c.lengths)
        first, out = torch.empty_like(q), torch.empty_like(q)
        size = ctx.paged_workspace(3, 4, c.cols * c.page, True)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        w0 = c.w.clone()

        def call(to):
            ctx.paged_attn(c.pages, c.table.data_ptr(), c.cols, lens.data_ptr(), 3, 0, 4, q.data_ptr(), to.data_ptr(),
                           True, ws.data_ptr(), size)
        call(first)
        w1 = c.w.clone()
        c.w.copy_(w0)
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            call(out)
        graph.replay()
        stream.synchronize()
        assert torch.equal(out, first) and torch.equal(c.w.view(torch.int32), w1.view(torch.int32))
        for lengths in ([1, 0, 17], [0, 0, 0], [299, 0, 1]):
            lens.copy_(i32(lengths))
            c.w.copy_(w0)
            graph.replay()
            stream.synchronize()
            c.lengths = lengths
            want, tol, _ = reference(c, q)
            assert bool(((out.double() - want).abs() <= tol).all()), lengths
    ctx.sync()


@pytest.mark.parametrize("lengths,layers", [([200, 300], 1), ([1000, 900], 1), ([300, 0, 2000], 4)])    # one CTA a unit, clusters, even split
def test_captured_calls_between_forked_streams(lengths, layers):
    """Inputs written by two streams that join before the calls, results read by two that fork behind them,
    all in one graph: every replay sees its own inputs, and its readers all its results."""
    ctx = make(layers, 8)
    n, keep = len(lengths), 64
    c = Cache(lengths, layers, 8, seed=61)
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    main.wait_stream(torch.cuda.current_stream())
    ctx.set_stream(main.cuda_stream)
    size = ctx.paged_workspace(n, layers, c.cols * c.page, True)
    with torch.cuda.stream(main):
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        q_new, lens_new, kv_new, w_new = c.query(), i32(lengths), c.kv.clone(), c.w.clone()
        q, lens, out = torch.zeros_like(q_new), i32([0] * n), torch.empty_like(q_new)
        out_seen, w_seen, kv_seen = torch.empty_like(out), torch.empty_like(c.w), torch.empty_like(c.kv)
        new, kept = i32([0] * n), torch.empty(n, layers, 8, keep, dtype=torch.int32, device="cuda")
        kept_seen, new_seen = torch.empty_like(kept), torch.empty_like(new)

        def calls():
            side.wait_stream(main)
            with torch.cuda.stream(side):
                c.kv.copy_(kv_new)
                lens.copy_(lens_new)
            q.copy_(q_new)
            c.w.copy_(w_new)
            main.wait_stream(side)
            ctx.paged_attn(c.pages, c.table.data_ptr(), c.cols, lens.data_ptr(), n, 0, layers, q.data_ptr(), out.data_ptr(),
                           True, ws.data_ptr(), size)
            side.wait_stream(main)
            with torch.cuda.stream(side):
                out_seen.copy_(out)
            w_seen.copy_(c.w)
            ctx.paged_evict(c.pages, c.table.data_ptr(), c.cols, c.table.data_ptr(), c.cols, lens.data_ptr(), new.data_ptr(),
                            n, keep, 16, kept.data_ptr())
            main.wait_stream(side)
            side.wait_stream(main)
            with torch.cuda.stream(side):
                kept_seen.copy_(kept)
                new_seen.copy_(new)
            kv_seen.copy_(c.kv)
            main.wait_stream(side)
        main.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=main):
            calls()
        seen = (out_seen, w_seen, kv_seen, kept_seen, new_seen)
        for i in range(12):
            q_new.copy_(c.query())
            lens_new.copy_(i32([max(m - 37 * i, 0) for m in lengths]))
            for t in seen:
                t.zero_()
            graph.replay()
            got = [t.clone() for t in seen]
            calls()
            main.synchronize()
            for x, y in zip(got, seen):
                assert torch.equal(x.view(torch.int16), y.view(torch.int16))
            assert bool(out_seen[:, 0].any()) == (lens_new[0] > 0) and new_seen.tolist() == [min(m, keep) for m in lens_new.tolist()]
    ctx.sync()


def test_calls_on_two_streams_with_their_own_workspaces():
    ctx = make(2, 8)
    c = Cache([3000, 1500], 2, 8, page=64, seed=13)
    q = c.query()
    want = attend(ctx, c, q)
    size = ctx.paged_workspace(2, 2, c.cols * c.page, False)
    lens = i32(c.lengths)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(q) for _ in range(8)] for _ in streams]
    spaces = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in streams]
    for i in range(8):
        for s, out, ws in zip(streams, outs, spaces):
            ctx.set_stream(s.cuda_stream)
            ctx.paged_attn(c.pages, c.table.data_ptr(), c.cols, lens.data_ptr(), 2, 0, 2, q.data_ptr(), out[i].data_ptr(),
                           False, ws.data_ptr(), size)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for out in outs for o in out)


def test_offsets_past_32_bits():
    """Pages at the end of a pool of more than 2^32 elements (8.6 GB)."""
    layers, hkv, page = 7, 8, 512
    per = layers * 2 * hkv * page * D
    n_pages = (1 << 32) // per + 9
    kv = torch.empty(n_pages, layers, 2, hkv, page, D, dtype=torch.float16, device="cuda")
    small = Cache([1200], layers, hkv, page=page, seed=14, extra_cols=0, spare=0)
    ids = i32([[n_pages - 1, n_pages - 5, n_pages - 2]])
    kv[ids[0].long()] = small.kv[small.table[0].long()]
    ctx = make(layers, hkv)
    q = small.query()
    want = attend(ctx, small, q)
    small.kv, small.table, small.n_pages, small.w = kv, ids, n_pages, None
    assert torch.equal(attend(ctx, small, q), want)
    ctx.sync()


def test_weights_gathered_by_two_streams_into_one_pool():
    """Calls that accumulate into the same pages from two streams, each with its own workspace: every
    call's weights arrive (their additions come in any order)."""
    ctx = make(1, 4)
    c = Cache([900, 400], 1, 4, page=32, seed=16)
    q = [c.query() for _ in range(2)]
    before = [c.weights(b).double().clone() for b in range(2)]
    size = ctx.paged_workspace(2, 1, c.cols * c.page, True)
    lens = i32(c.lengths)
    spaces = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    outs = [torch.empty_like(x) for x in q]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, x, out, ws in zip(streams, q, outs, spaces):
            ctx.set_stream(s.cuda_stream)
            ctx.paged_attn(c.pages, c.table.data_ptr(), c.cols, lens.data_ptr(), 2, 0, 1, x.data_ptr(), out.data_ptr(), True,
                           ws.data_ptr(), size)
    torch.cuda.synchronize()
    for b in range(2):
        total, limit = before[b].clone(), torch.zeros_like(before[b])
        for x in q:
            _, _, probs = reference(c, x)
            total += 5 * probs[b][0]
            limit += 5 * probs[b][1]
        assert bool(((c.weights(b).double() - total).abs() <= limit + 20 * U * total).all())


def test_lengths_up_to_the_tables_capacity_and_pages_at_the_pools_ends():
    ctx = make(2, 2)
    for page in (16, 512):
        c = Cache([3 * page, 3 * page - 1, 1], 2, 2, page=page, seed=17, extra_cols=0, spare=0)
        assert sorted(c.table[c.table >= 0].tolist()) == list(range(c.n_pages))
        check_attend(ctx, c, c.query(), add=True)


@pytest.mark.parametrize("layers,hkv,n,cols_rows", [(1, 8, 18, 512), (1, 1, 148, 512), (1, 1, 149, 512), (28, 1, 5, 256), (2, 8, 3, 513),
    (1, 8, 1, 4096), (1, 8, 1, 4097), (1, 4, 2, 4000), (1, 2, 9, 4096), (1, 8, 2, 4096), (1, 8, 3, 2048), (1, 8, 4, 1024),
    (3, 1, 6, 300), (1, 1, 1, 128), (1, 1, 1, 129), (1, 1, 1, 16)])
def test_calls_of_few_units_around_the_rule_for_their_own_ctas(layers, hkv, n, cols_rows):
    """Calls on either side of the rule (units and rows that a table can hold), ragged with empty rows."""
    ctx = make(layers, hkv)
    r = np.random.default_rng(n)
    lengths = [int(x) for x in r.integers(0, cols_rows + 1, n)]
    lengths[0], lengths[-1] = cols_rows, 0 if n > 1 else cols_rows
    c = Cache(lengths, layers, hkv, page=16, seed=n, extra_cols=0)
    check_attend(ctx, c, c.query(), add=True)
    check_attend(ctx, c, c.query())
    # lengths outside the table: zeros for that row, reported
    q = c.query()
    want, tol, _ = reference(c, q)
    bad = i32(lengths)
    bad[0] = c.cols * 16 + 1
    out = attend(ctx, c, q, lengths=bad)
    with pytest.raises(qattn.QAttnError) as err:
        ctx.sync()
    assert "code 61" in str(err.value) and not out[:, 0].any()
    assert bool(((out.double() - want).abs() <= tol)[:, 1:].all())


@pytest.mark.parametrize("layers,hkv,rows", [(28, 8, 3970), (28, 8, 1), (28, 8, 63), (28, 8, 65), (37, 8, 500), (38, 8, 40), (19, 8, 1000), (64, 4, 17),
    (40, 4, 1024), (40, 4, 1600), (28, 4, 2049), (28, 4, 15), (28, 2, 1500), (28, 1, 3000), (2, 8, 1537), (37, 4, 4100)])
def test_one_sequence_of_many_layers(layers, hkv, rows):
    """One sequence: CTAs, half-size CTAs or clusters for every layer and KV head, whatever the rows; empty
    and too long lengths."""
    ctx = make(layers, hkv)
    c = Cache([rows], layers, hkv, page=16, seed=rows, extra_cols=0)
    q = c.query()
    check_attend(ctx, c, q, add=True)
    out = check_attend(ctx, c, q)
    assert torch.equal(out, attend(ctx, c, q))
    assert not attend(ctx, c, q, lengths=i32([0])).any()
    ctx.sync()
    assert not attend(ctx, c, q, lengths=i32([c.cols * 16 + 1])).any()
    with pytest.raises(qattn.QAttnError) as err:
        ctx.sync()
    assert "code 61" in str(err.value)


# ---- append --------------------------------------------------------------------------------------
@pytest.mark.parametrize("hkv,page,n", [(8, 16, 1), (8, 16, 5), (4, 32, 7), (2, 64, 33), (1, 512, 130), (8, 128, 40)])
def test_append_tokens_bit_exact_with_the_oracle(hkv, page, n):
    """One token for each of n sequences at any position up to 40000, padded rows among them."""
    L = 2
    ctx = make(L, hkv)
    ctx.rope_positions(40000)
    r = np.random.default_rng(n)
    qw = (1 + 0.1 * r.standard_normal((L, D))).astype(np.float32)
    kw = (1 + 0.1 * r.standard_normal((L, D))).astype(np.float32)
    H.set_norms(ctx, qw, kw)
    held = [int(x) for x in r.integers(1, 600, n)]
    pos = [int(x) for x in r.integers(0, 40000, n)]
    pos[0] = 39999
    for b in range(1, n, 3):
        held[b] = 0
    c = Cache(held, L, hkv, page=page, seed=n)
    g = torch.Generator("cuda").manual_seed(n)
    q, k, v = (torch.randn(L, n, h, D, device="cuda", generator=g) * 3 for h in (2 * hkv, hkv, hkv))
    v[0, 0, 0, :2] = torch.tensor([1e30, -1e30])        # becomes +-inf in FP16, as in qa_append
    out = torch.full_like(q, 7.0)
    kv0, w0 = c.kv.clone(), c.w.clone()
    held_d, pos_d = i32(held), i32(pos)
    ctx.paged_append(c.pages, c.table.data_ptr(), n, c.cols, 0, held_d.data_ptr(), pos_d.data_ptr(), n, 0, L, q.data_ptr(),
                     k.data_ptr(), v.data_ptr(), out.data_ptr())
    ctx.sync()
    cos, sin = O.rope_tables(40000)
    for b in range(n):
        if not held[b]:
            assert not out[:, b].any()
            continue
        tables = (np.ascontiguousarray(cos[pos[b]:pos[b] + 1]), np.ascontiguousarray(sin[pos[b]:pos[b] + 1]))
        for layer in range(L):
            kv = O.LayerKV(hkv, 1)
            qref = O.append(kv, 0, *(t[layer, b:b + 1].cpu().numpy() for t in (q, k, v)), qw[layer], kw[layer], tables)
            assert np.array_equal(out[layer, b:b + 1].cpu().numpy(), qref)
            got = c.rows(b)[layer, :, :, held[b] - 1].cpu().numpy().view(np.uint16)
            assert np.array_equal(got[0], kv.k[:, 0]) and np.array_equal(got[1], kv.v[:, 0])
        ids, at = c.where(b, held[b])
        kv0[ids[-1], :, :, :, at[-1]] = c.kv[ids[-1], :, :, :, at[-1]]
        w0[ids[-1], :, :, at[-1]] = 0
    assert torch.equal(c.kv.view(torch.int16), kv0.view(torch.int16))           # no other row was touched
    assert torch.equal(c.w.view(torch.int32), w0.view(torch.int32))


def test_append_of_mixed_prompts_in_any_order_and_without_q_out():
    L, hkv, page = 2, 8, 16
    ctx = make(L, hkv, context=512)
    counts = [1, 200, 16, 33]
    seq = [s for s, m in enumerate(counts) for _ in range(m)]
    held = [i + 1 for m in counts for i in range(m)]
    order = np.random.default_rng(3).permutation(len(seq))
    seq, held = [seq[i] for i in order], [held[i] for i in order]
    n = len(seq)
    g = torch.Generator("cuda").manual_seed(4)
    q, k, v = (torch.randn(L, n, h, D, device="cuda", generator=g) for h in (2 * hkv, hkv, hkv))
    c = Cache([0] * 4, L, hkv, page=page, seed=15, room=200, weights=False)
    args = [i32(seq), i32(held), i32([h - 1 for h in held])]
    ctx.paged_append(c.pages, c.table.data_ptr(), 4, c.cols, *(t.data_ptr() for t in args), n, 0, L, q.data_ptr(),
                     k.data_ptr(), v.data_ptr(), 0)
    one = Cache([0] * 4, L, hkv, page=page, seed=15, room=200, weights=False)
    out, alone = torch.empty_like(q), torch.empty(L, 1, 2 * hkv, D, device="cuda")
    ctx.paged_append(one.pages, one.table.data_ptr(), 4, one.cols, *(t.data_ptr() for t in args), n, 0, L, q.data_ptr(),
                     k.data_ptr(), v.data_ptr(), out.data_ptr())
    assert torch.equal(c.kv.view(torch.int16), one.kv.view(torch.int16))
    again = Cache([0] * 4, L, hkv, page=page, seed=15, room=200, weights=False)
    for r in range(n):                                  # row by row: the same bits
        part = [t[:, r:r + 1].contiguous() for t in (q, k, v)]
        ctx.paged_append(again.pages, again.table.data_ptr(), 4, again.cols, *(t[r:].data_ptr() for t in args), 1, 0, L,
                         *(t.data_ptr() for t in part), alone.data_ptr())
        assert torch.equal(alone[:, 0], out[:, r])
    ctx.sync()
    assert torch.equal(c.kv.view(torch.int16), again.kv.view(torch.int16))
    # a layer range leaves the other layers alone
    kv0 = c.kv.clone()
    ctx.paged_append(c.pages, c.table.data_ptr(), 4, c.cols, *(t.data_ptr() for t in args), n, 1, 1, q[0].data_ptr(),
                     k[0].contiguous().data_ptr(), v[0].contiguous().data_ptr(), 0)
    ctx.sync()
    assert torch.equal(c.kv[:, 0].view(torch.int16), kv0[:, 0].view(torch.int16))
    assert not torch.equal(c.kv[:, 1].view(torch.int16), kv0[:, 1].view(torch.int16))


# ---- eviction ------------------------------------------------------------------------------------
def kept_rows(w, keep, recent):
    """Old indices kept of one head's weights, by the definition (NaN last, ties to the lower row)."""
    m = len(w)
    if m <= keep:
        return list(range(m))
    rank = sorted(range(m - recent), key=lambda i: (math.inf if math.isnan(w[i]) else -w[i], math.isnan(w[i]), i))
    return sorted(rank[:keep - recent]) + list(range(m - recent, m))


def check_evict(ctx, c, keep, recent, dst=None, same_lengths=False):
    """dst None: in place; else a Cache whose pages lie in the same pool."""
    n = len(c.lengths)
    lens = i32(c.lengths)
    new = lens if same_lengths else torch.full((n,), -9, dtype=torch.int32, device="cuda")
    kept = torch.full((n, c.layers, c.hkv, keep), -9, dtype=torch.int32, device="cuda")
    to = c.table if dst is None else dst
    rows, weights = [c.rows(b).clone() for b in range(n)], [c.weights(b).clone() for b in range(n)]
    kv0, w0 = c.kv.clone(), c.w.clone()
    ctx.paged_evict(c.pages, c.table.data_ptr(), c.cols, to.data_ptr(), to.shape[1], lens.data_ptr(), new.data_ptr(), n,
                    keep, recent, kept.data_ptr())
    ctx.sync()
    assert new.tolist() == [min(m, keep) for m in c.lengths]
    host = kept.cpu().numpy()
    for b, m in enumerate(c.lengths):
        t = torch.arange(min(m, keep), device="cuda")
        ids, at = to[b].long()[t // c.page], t % c.page
        w = weights[b].cpu().numpy()
        for layer in range(c.layers):
            for h in range(c.hkv):
                mine = kept_rows(w[layer, h].tolist(), keep, recent)
                assert host[b, layer, h].tolist() == mine + [-1] * (keep - len(mine)), (b, layer, h)
                i = torch.tensor(mine, dtype=torch.int64, device="cuda")
                kv0[ids, layer, :, h, at] = rows[b][layer, :, h, i].transpose(0, 1)
                w0[ids, layer, h, at] = weights[b][layer, h, i]
    assert torch.equal(c.kv.view(torch.int16), kv0.view(torch.int16))           # the rest is left as it was
    assert torch.equal(c.w.view(torch.int32), w0.view(torch.int32))
    return kept


@pytest.mark.parametrize("lengths,layers,hkv,page,keep,recent", [
    ([1], 1, 8, 16, 1, 0), ([2], 1, 8, 16, 1, 0), ([2], 1, 8, 16, 1, 1), ([17], 2, 1, 16, 16, 3),
    ([0, 5, 33, 34, 700, 1025], 2, 4, 16, 33, 4), ([513, 1024, 2000], 1, 8, 128, 512, 0), ([600], 3, 2, 32, 599, 599),
    ([1500, 40], 1, 8, 512, 700, 64), ([4096], 2, 8, 64, 2048, 256), ([20000], 1, 1, 256, 9001, 17), ([777], 1, 2, 16, 1, 0)])
def test_evict_in_place(lengths, layers, hkv, page, keep, recent):
    ctx = make(layers, hkv)
    c = Cache(lengths, layers, hkv, page=page, seed=keep, extra_cols=-(-keep // page))
    need = max(max(lengths), keep)                      # the table has a page for every kept row
    for b in range(len(lengths)):
        assert c.cols * page >= need
    check_evict(ctx, c, keep, recent, same_lengths=bool(keep % 2))


@pytest.mark.parametrize("page,keep,recent", [(16, 100, 10), (64, 300, 0), (32, 1000, 1000)])
def test_evict_into_other_pages(page, keep, recent):
    lengths = [1200, 90, 0, 301]
    ctx = make(2, 4)
    cols = -(-keep // page)
    c = Cache(lengths, 2, 4, page=page, seed=page, spare=4 * cols)
    used = set(c.table.flatten().tolist())
    free = [p for p in range(c.n_pages) if p not in used][:4 * cols]
    check_evict(ctx, c, keep, recent, dst=i32(free).view(4, cols).contiguous())


@pytest.mark.parametrize("rows,hkv,layers,page,keep,recent", [
    (5000, 8, 1, 16, 3000, 100), (40000, 1, 1, 64, 20001, 0), (524288, 1, 1, 512, 300000, 4096), (70000, 2, 1, 128, 1, 1),
    (9000, 8, 3, 32, 8999, 17), (4097, 4, 28, 64, 100, 0)])
def test_evict_long_units_over_several_slices(rows, hkv, layers, page, keep, recent):
    """Units whose rows are spread over a cluster (more than 4096), against a sort."""
    ctx = make(layers, hkv)
    g = torch.Generator("cuda").manual_seed(rows)
    cols = -(-rows // page)
    table = torch.randperm(cols, device="cuda", generator=g).to(torch.int32)[None].contiguous()
    kv = torch.randint(-30000, 30000, (cols, layers, 2, hkv, page, D), dtype=torch.int16, device="cuda", generator=g)
    w = (torch.rand(cols, layers, hkv, page, device="cuda", generator=g) * 50).floor() / 50     # many ties
    t = torch.arange(rows, device="cuda")
    ids, at = table[0].long()[t // page], t % page
    flat_w = w[ids, :, :, at].permute(1, 2, 0)                                                   # [layers][hkv][rows]
    rank = flat_w.clone()
    rank[..., rows - recent:] = 2.0
    want = torch.sort(torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep], dim=-1).values
    old = kv.clone()
    lens, new = i32([rows]), i32([0])
    kept = torch.empty(1, layers, hkv, keep, dtype=torch.int32, device="cuda")
    ctx.paged_evict(qattn.Pages(kv.data_ptr(), w.data_ptr(), cols, page), table.data_ptr(), cols, table.data_ptr(), cols,
                    lens.data_ptr(), new.data_ptr(), 1, keep, recent, kept.data_ptr())
    ctx.sync()
    assert new.tolist() == [keep] and torch.equal(kept[0].long(), want)
    got_w = w[ids[:keep], :, :, at[:keep]].permute(1, 2, 0)
    assert torch.equal(got_w, torch.gather(flat_w, 2, want))
    for layer in range(layers):
        for h in range(hkv):
            i = want[layer, h]
            assert torch.equal(kv[ids[:keep], layer, :, h, at[:keep]], old[ids[i], layer, :, h, at[i]])
    assert torch.equal(kv[ids[keep:], :, :, :, at[keep:]], old[ids[keep:], :, :, :, at[keep:]])


def test_evict_refuses_tables_beyond_its_rows():
    ctx = make(1, 8)
    c = Cache([40], 1, 8, seed=33)
    lens, new = i32([40]), i32([0])
    kept = torch.empty(8 * 20, dtype=torch.int32, device="cuda")
    with pytest.raises(qattn.QAttnError) as err:
        ctx.paged_evict(c.pages, c.table.data_ptr(), (1 << 19) // 16 + 1, c.table.data_ptr(), c.cols, lens.data_ptr(),
                        new.data_ptr(), 1, 20, 0, kept.data_ptr())
    assert err.value.status == qattn.QA_ERR_INVALID


def test_evict_ties_zeros_infinities_and_nan():
    ctx = make(1, 8)
    c = Cache([1000], 1, 8, seed=31)
    w = c.weights(0).clone()
    w[0, 0] = 0.0
    w[0, 1] = (w[0, 1] * 3).floor()                     # 0, 1, 2
    w[0, 2] = float("nan")
    w[0, 3, ::3] = float("nan")
    w[0, 4, ::5] = float("inf")
    w[0, 5] = -w[0, 5]
    w[0, 6, ::2] = -0.0
    w[0, 6, 1::2] = 0.0
    w[0, 7] = torch.where(w[0, 7] < 0.5, float("-inf"), 1e-42)      # subnormals above -inf
    c.put_weights(0, w)
    check_evict(ctx, c, 400, 30)


def test_evict_is_capturable_and_pairs_with_attention():
    """Append, attention with weights and eviction as a serving loop runs them, captured and replayed."""
    layers, hkv, page, steps, keep, recent = 2, 8, 16, 40, 48, 8
    ctx = make(layers, hkv)
    ctx.rope_positions(5000)
    n = 3
    start = [60, 33, 0]                                 # the last row is padding
    c = Cache(start, layers, hkv, page=page, seed=32, room=steps + 1)
    ref = Cache(start, layers, hkv, page=page, seed=32, room=steps + 1)
    assert torch.equal(c.table, ref.table)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ctx.set_stream(stream.cuda_stream)
    with torch.cuda.stream(stream):
        live = i32([1, 1, 0])
        lens, pos = i32(start), i32([4000, 33, 0])
        q, k, v = (torch.zeros(layers, n, h, D, device="cuda") for h in (2 * hkv, hkv, hkv))
        qn, out = torch.empty_like(q), torch.empty_like(q)
        size = ctx.paged_workspace(n, layers, c.cols * page, True)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        kept = torch.empty(n, layers, hkv, keep, dtype=torch.int32, device="cuda")

        def step(cache):
            lens.add_(live)
            ctx.paged_append(cache.pages, cache.table.data_ptr(), n, cache.cols, 0, lens.data_ptr(), pos.data_ptr(), n, 0,
                             layers, q.data_ptr(), k.data_ptr(), v.data_ptr(), qn.data_ptr())
            ctx.paged_attn(cache.pages, cache.table.data_ptr(), cache.cols, lens.data_ptr(), n, 0, layers, qn.data_ptr(),
                           out.data_ptr(), True, ws.data_ptr(), size)
            pos.add_(live)

        def evict(cache):
            ctx.paged_evict(cache.pages, cache.table.data_ptr(), cache.cols, cache.table.data_ptr(), cache.cols,
                            lens.data_ptr(), lens.data_ptr(), n, keep, recent, kept.data_ptr())
        stream.synchronize()
        g_step, g_evict = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g_step, stream=stream):
            step(c)
        with torch.cuda.graph(g_evict, stream=stream):
            evict(c)
        results = []
        for cache, do_step, do_evict in ((c, g_step.replay, g_evict.replay), (ref, lambda: step(ref), lambda: evict(ref))):
            lens.copy_(i32(start))
            pos.copy_(i32([4000, 33, 0]))
            g = torch.Generator("cuda").manual_seed(5)
            seen = []
            for i in range(steps):
                for t in (q, k, v):
                    t.copy_(torch.randn(t.shape, device="cuda", generator=g))
                do_step()
                seen.append(out.clone())
                if i % 10 == 9:
                    do_evict()
                    seen.append(kept.clone())
                    seen.append(lens.clone())
            stream.synchronize()
            results.append(seen)
    ctx.sync()
    for x, y in zip(*results):
        assert torch.equal(x, y)
    assert results[0][-1].tolist() == [48, 48, 0]
    assert torch.equal(c.kv.view(torch.int16), ref.kv.view(torch.int16))
    assert not any(r[:, 2].any() for r in results[0][:9])


def test_calls_in_a_row_equal_calls_one_by_one():
    """Paged calls between slot calls, each reading what the one before wrote, queued without a wait and
    with one after every call: the same bits. (Launches overlap; every kernel waits for the one before.)"""
    L, rows = 2, 130
    results = []
    for wait in (False, True):
        ctx = make(L, 8, context=512)
        ctx.rope_positions(600)
        c = Cache([rows, 40, 0], L, 8, seed=91, room=64)
        lens, live = i32(c.lengths), i32([1, 1, 0])
        pos, first = i32([300, 40, 0]), i32([0, 1, 2])
        g = torch.Generator("cuda").manual_seed(17)
        q, k, v = (torch.randn(L, 3, h, D, device="cuda", generator=g) for h in (16, 8, 8))
        pq, pk, pv = (torch.randn(L, rows, h, D, device="cuda", generator=g) for h in (16, 8, 8))
        qn, out, pqn, pout = (torch.zeros_like(t) for t in (q, q, pq, pq))
        sq, sk, sv = (torch.zeros(L, 1, h, D, device="cuda") for h in (16, 8, 8))
        sqn, sout = torch.zeros_like(sq), torch.zeros_like(sq)
        size = ctx.paged_workspace(3, L, c.cols * c.page, True)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        kept = torch.zeros(3, L, 8, 60, dtype=torch.int32, device="cuda")
        w = torch.randn(2048, 2048, device="cuda", generator=g).half()
        y = torch.zeros(L, 3, 2048, device="cuda")
        done = (lambda: ctx.sync()) if wait else (lambda: None)
        seen = []
        ctx.reset(0)
        # a prompt into a slot, its rows into the pages of the first sequence
        ctx.append(0, 0, L, 0, rows, pq.data_ptr(), pk.data_ptr(), pv.data_ptr(), pqn.data_ptr()); done()
        ctx.attn_prefill(0, 0, L, 0, rows, pqn.data_ptr(), pout.data_ptr()); done()
        ctx.commit(0, rows)
        held = torch.arange(1, rows + 1, dtype=torch.int32, device="cuda")
        at, seq0 = held - 1, torch.zeros_like(held)
        ctx.paged_append(c.pages, c.table.data_ptr(), 3, c.cols, seq0.data_ptr(), held.data_ptr(), at.data_ptr(), rows, 0, L,
                         pq.data_ptr(), pk.data_ptr(), pv.data_ptr(), pqn.data_ptr()); done()
        for i in range(12):
            lens.add_(live); done()
            for layer in range(L):
                ctx.paged_append(c.pages, c.table.data_ptr(), 3, c.cols, first.data_ptr(), lens.data_ptr(), pos.data_ptr(), 3, layer, 1,
                                 q[layer].data_ptr(), k[layer].data_ptr(), v[layer].data_ptr(), qn[layer].data_ptr()); done()
                ctx.paged_attn(c.pages, c.table.data_ptr(), c.cols, lens.data_ptr(), 3, layer, 1, qn[layer].data_ptr(),
                               out[layer].data_ptr(), True, ws.data_ptr(), size); done()
                # the next inputs come from this output: a projection, and a slot's decode step of its first row
                ctx.project_gemm(w.data_ptr(), 2048, 2048, out[layer].data_ptr(), 3, y[layer].data_ptr()); done()
            q.copy_(y.view(L, 3, 16, D)); done()
            sq.copy_(out[:, :1]); sk.copy_(out[:, :1, :8]); sv.copy_(out[:, :1, 8:]); done()
            ctx.decode_step(0, 0, L, rows + i, sq.data_ptr(), sk.data_ptr(), sv.data_ptr(), sqn.data_ptr(), sout.data_ptr()); done()
            ctx.commit(0, 1)
            # straight behind the step: attention of its queries, then an eviction
            ctx.paged_attn(c.pages, c.table[:1].data_ptr(), c.cols, lens.data_ptr(), 1, 0, L, sqn.data_ptr(), sout.data_ptr(),
                           True, ws.data_ptr(), size); done()
            if i % 5 == 4:
                ctx.paged_evict(c.pages, c.table.data_ptr(), c.cols, c.table.data_ptr(), c.cols, lens.data_ptr(), lens.data_ptr(), 3,
                                60, 7, kept.data_ptr()); done()
            pos.add_(live); done()
            seen += [out.clone(), sout.clone(), kept.clone(), lens.clone()]
        ctx.sync()
        results.append(seen + [pout, c.kv.clone(), c.w.clone()])
    for x, y in zip(*results):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))


# ---- host buffers, refusals, bad tables ----------------------------------------------------------
def test_host_buffer_context():
    L, hkv, n = 3, 8, 5
    lengths = [100, 1, 0, 517, 64]
    c = Cache(lengths, L, hkv, page=32, seed=41)
    dev, host = make(L, hkv), make(L, hkv, io_host=1)
    g = torch.Generator("cuda").manual_seed(42)
    q, k, v = (torch.randn(L, n, h, D, device="cuda", generator=g) for h in (2 * hkv, hkv, hkv))
    held, pos = i32(lengths), i32([0, 0, 0, 0, 0])
    qn, out = torch.empty_like(q), torch.empty_like(q)
    torch.cuda.synchronize()
    dev.paged_append(c.pages, c.table.data_ptr(), n, c.cols, 0, held.data_ptr(), pos.data_ptr(), n, 0, L, q.data_ptr(),
                     k.data_ptr(), v.data_ptr(), qn.data_ptr())
    out = attend(dev, c, qn, add=True)
    dev.sync()
    kv1, w1 = c.kv.clone(), c.w.clone()
    d = Cache(lengths, L, hkv, page=32, seed=41)
    hq, hk, hv = (t.cpu().numpy() for t in (q, k, v))
    hqn, hout = np.empty_like(hq), np.empty_like(hq)
    size = host.paged_workspace(n, L, d.cols * 32, True)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    host.paged_append(d.pages, d.table.data_ptr(), n, d.cols, 0, held.data_ptr(), pos.data_ptr(), n, 0, L, hq.ctypes.data,
                      hk.ctypes.data, hv.ctypes.data, hqn.ctypes.data)
    host.paged_append(d.pages, d.table.data_ptr(), n, d.cols, 0, held.data_ptr(), pos.data_ptr(), n, 0, L, hq.ctypes.data,
                      hk.ctypes.data, hv.ctypes.data, 0)
    host.paged_attn(d.pages, d.table.data_ptr(), d.cols, held.data_ptr(), n, 0, L, hqn.ctypes.data, hout.ctypes.data, True,
                    ws.data_ptr(), size)
    assert np.array_equal(hqn, qn.cpu().numpy()) and np.array_equal(hout, out.cpu().numpy())
    assert torch.equal(d.kv.view(torch.int16), kv1.view(torch.int16)) and torch.equal(d.w.view(torch.int32), w1.view(torch.int32))
    bad = i32([100, 1, 0, 10 ** 6, 64])
    torch.cuda.synchronize()
    with pytest.raises(qattn.QAttnError) as err:
        host.paged_attn(d.pages, d.table.data_ptr(), d.cols, bad.data_ptr(), n, 0, L, hqn.ctypes.data, hout.ctypes.data,
                        False, ws.data_ptr(), size)
    assert err.value.status == qattn.QA_ERR_INVALID and "code 61" in str(err.value)


def test_refusals_leave_everything_alone():
    L, hkv, n = 2, 8, 2
    ctx = make(L, hkv)
    c = Cache([40, 50], L, hkv, seed=51)
    q = c.query()
    k, v = (torch.zeros(L, n, hkv, D, device="cuda") for _ in range(2))
    out = torch.full_like(q, 3.0)
    lens, new = i32(c.lengths), torch.full((2,), 5, dtype=torch.int32, device="cuda")
    kept = torch.full((n, L, hkv, 60), 6, dtype=torch.int32, device="cuda")
    size = ctx.paged_workspace(n, L, c.cols * 16, True)
    ws = torch.empty(size + 16, dtype=torch.uint8, device="cuda")
    p, T, C, LN, W = c.pages, c.table.data_ptr(), c.cols, lens.data_ptr(), ws.data_ptr()
    Q, O_, K, V = q.data_ptr(), out.data_ptr(), k.data_ptr(), v.data_ptr()

    def pages(**kw):
        d = dict(kv=c.kv.data_ptr(), weights=c.w.data_ptr(), n_pages=c.n_pages, page_rows=16)
        d.update(kw)
        return qattn.Pages(d["kv"], d["weights"], d["n_pages"], d["page_rows"])
    attn = [p, T, C, LN, n, 0, L, Q, O_, True, W, size]
    app = [p, T, n, C, 0, LN, LN, n, 0, L, Q, K, V, O_]
    ev = [p, T, C, T, C, LN, new.data_ptr(), n, 30, 4, kept.data_ptr()]
    bad_pool = [pages(kv=0), pages(kv=c.kv.data_ptr() + 8), pages(n_pages=0), pages(page_rows=8), pages(page_rows=48),
                pages(page_rows=1024), pages(page_rows=0), pages(page_rows=-16), pages(weights=c.w.data_ptr() + 4)]
    cases = [(ctx.paged_attn, attn, i, x) for i, x in [(1, 0), (1, T + 2), (2, 0), (2, -1), (2, (1 << 16) + 1), (3, 0), (4, 0),
             (4, 1025), (5, -1), (6, 0), (6, 3), (7, 0), (7, Q + 4), (8, 0), (8, O_ + 8), (10, 0), (10, W + 8), (11, size - 1)]]
    cases += [(ctx.paged_attn, attn, 0, x) for x in bad_pool + [pages(weights=0)]]
    cases += [(ctx.paged_append, app, i, x) for i, x in [(1, 0), (2, 0), (2, 1), (3, 0), (4, T + 1), (5, 0), (6, 0), (7, 0),
              (7, -4), (7, (1 << 20) + 1), (8, 1), (9, 0), (10, 0), (10, Q + 4), (11, 0), (12, 0), (12, V + 4), (13, O_ + 4)]]
    cases += [(ctx.paged_append, app, 0, x) for x in bad_pool]
    cases += [(ctx.paged_evict, ev, i, x) for i, x in [(1, 0), (2, 0), (3, 0), (4, 0), (4, 1), (5, 0), (6, 0), (7, 0), (7, 2000),
              (8, 0), (8, C * 16 + 1), (9, -1), (9, 31), (10, 0), (10, kept.data_ptr() + 1)]]
    cases += [(ctx.paged_evict, ev, 0, x) for x in bad_pool + [pages(weights=0)]]
    kv0, w0 = c.kv.clone(), c.w.clone()
    for fn, args, i, x in cases:
        changed = list(args)
        changed[i] = x
        with pytest.raises(qattn.QAttnError) as err:
            fn(*changed)
        assert err.value.status == qattn.QA_ERR_INVALID, (fn.__name__, i, x)
    with pytest.raises(qattn.QAttnError):
        ctx.paged_workspace(0, 1, 16)
    with pytest.raises(qattn.QAttnError):
        ctx.paged_workspace(1, 3, 16)
    with pytest.raises(qattn.QAttnError):
        ctx.paged_workspace(1, 1, (1 << 20) + 1)
    for n_pos in (0, -1, (1 << 20) + 1):
        with pytest.raises(qattn.QAttnError):
            ctx.rope_positions(n_pos)
    ctx.sync()
    assert bool((out == 3).all()) and bool((new == 5).all()) and bool((kept == 6).all())
    assert torch.equal(c.kv.view(torch.int16), kv0.view(torch.int16)) and torch.equal(c.w.view(torch.int32), w0.view(torch.int32))


def test_bad_lengths_pages_and_positions_are_reported_and_skipped():
    """The kernels check every index they read (walked on the CPU in test_paged_index.py): the bad
    sequence's results are undefined, the others' are right, and nothing else is written."""
    L, hkv = 2, 4
    ctx = make(L, hkv)
    c = Cache([300, 200, 90], L, hkv, seed=61)
    q = c.query()
    want, tol, _ = reference(c, q)
    k, v = (torch.randn(L, 3, hkv, D, device="cuda") for _ in range(2))
    new, kept = torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, L, hkv, 50, dtype=torch.int32, device="cuda")
    good = c.table.clone()
    size = ctx.paged_workspace(3, L, c.cols * 16, True)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")

    def expect(code):
        with pytest.raises(qattn.QAttnError) as err:
            ctx.sync()
        assert err.value.status == qattn.QA_ERR_INVALID and f"code {code}" in str(err.value)
        ctx.sync()                                      # reported once

    def run(lengths, add=False):
        out, lens = torch.empty_like(q), i32(lengths)
        ctx.paged_attn(c.pages, c.table.data_ptr(), c.cols, lens.data_ptr(), 3, 0, L, q.data_ptr(), out.data_ptr(), add,
                       ws.data_ptr(), size)
        torch.cuda.synchronize()
        assert bool(((out.double() - want).abs() <= tol)[:, [0, 2]].all())
    for length in (-1, c.cols * 16 + 1, 2 ** 31 - 1, -2 ** 31):
        run([300, length, 90])
        expect(61)
    for page in (-1, c.n_pages, 2 ** 31 - 1, -2 ** 31):
        c.table[1, 3] = page
        run([300, 200, 90])
        expect(62)
        w0 = c.w.clone()
        run([300, 200, 90], add=True)
        expect(62)
        for b in (0, 1, 2):                             # only rows of the call's own pages change
            ids, _ = (good[b, :-(-c.lengths[b] // 16)].long(), None)
            w0[ids] = c.w[ids]
        assert torch.equal(c.w.view(torch.int32), w0.view(torch.int32))
        c.table.copy_(good)
    held, pos = [300, 200, 90], [5, 0, 0]
    for i, (h, p, s, code) in enumerate([(-3, 0, 1, 61), (c.cols * 16 + 1, 0, 1, 61), (200, -1, 1, 63), (200, 1, 1, 63),
                                         (200, 0, 3, 64), (200, 0, -1, 64)]):
        kv0, out = c.kv.clone(), torch.empty_like(q)
        a, b, d = i32([0, s, 2]), i32([300, h, 90]), i32([0, p, 0])
        ctx.paged_append(c.pages, c.table.data_ptr(), 3, c.cols, a.data_ptr(), b.data_ptr(), d.data_ptr(), 3, 0, L,
                         q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr())
        expect(code)
        assert not out[:, 1].any()
        for r in (0, 2):
            ids, at = c.where(r, held[r])
            assert not torch.equal(c.kv[ids[-1], :, :, :, at[-1]], kv0[ids[-1], :, :, :, at[-1]]) or i > 0
            kv0[ids[-1], :, :, :, at[-1]] = c.kv[ids[-1], :, :, :, at[-1]]
        assert torch.equal(c.kv.view(torch.int16), kv0.view(torch.int16))
    e = Cache([300, 200, 90], L, hkv, seed=61)
    for where, value, code in (("src", -1, 62), ("src", e.n_pages, 62), ("dst", -1, 62), ("len", 10 ** 9, 61), ("len", -2, 61)):
        c = Cache([300, 200, 90], L, hkv, seed=61)
        src, dst, lens = c.table.clone(), c.table.clone(), i32(c.lengths)
        if where == "len":
            lens[1] = value
        else:
            (src if where == "src" else dst)[1, 2] = value
        rows = [c.rows(b).clone() for b in range(3)]
        spare = sorted(set(range(c.n_pages)) - set(c.table.flatten().tolist()))
        ctx.paged_evict(c.pages, src.data_ptr(), c.cols, dst.data_ptr(), c.cols, lens.data_ptr(), new.data_ptr(), 3, 50, 5,
                        kept.data_ptr())
        expect(code)
        for b in (0, 2):
            i = kept[b, 1, 1].long()
            assert torch.equal(c.rows(b, 50)[1, :, 1].view(torch.int16), rows[b][1, :, 1, i].view(torch.int16))
        assert torch.equal(c.kv[spare].view(torch.int16), e.kv[spare].view(torch.int16))


# ---- sequences over the cache ----------------------------------------------------------------------
def test_sequences_follow_the_slot_model():
    """Prompts, steps, closing and opening through PagedSequences against AttentionModel over slots."""
    from fpga_qwen_b200.engine import AttentionModel
    from fpga_qwen_b200.paged import PagedSequences
    L, steps = 2, 20
    ctx = make(L, 8, context=1024)
    qw, kw = H.norms(71, L)
    H.set_norms(ctx, qw, kw)
    ref = make(L, 8, context=1024, max_seqs=3)
    H.set_norms(ref, qw, kw)
    s = PagedSequences(ctx, n_pages=120, page_rows=16, max_seqs=4, max_rows=700)
    prompts = {0: 600, 1: 33, 2: 1}
    models = {}
    for slot, n in prompts.items():
        seq = s.open()
        assert seq == slot
        q, k, v = H.inputs(100 + slot, L, 0, n)
        models[slot] = AttentionModel(ref, slot)
        want, got = models[slot].prefill(q, k, v), s.prefill(seq, q, k, v)
        # the slot model decodes one-row prompts; both lie within the tolerance of the oracle
        assert float((want - got).abs().max()) < 2 * H.MAX_ABS
    for i in range(steps):
        if i == 10:
            s.close(1)
        s.begin_step()
        q, k, v = (torch.randn(L, 4, h, D, device="cuda") for h in (16, 8, 8))
        qn, out = torch.empty_like(q), torch.empty_like(q)
        for layer in range(L):                          # the engine's order: layer by layer
            one = slice(layer, layer + 1)
            s.append(q[one], k[one], v[one], layer, q_out=qn[one])
            s.attend(qn[one], layer, out=out[one])
        for slot in s.host.live():
            want = models[slot].step(*(t[:, slot:slot + 1].contiguous() for t in (q, k, v)))
            assert s.position(slot) == models[slot].position == s.rows(slot)
            # two FP32 evaluations of the same rows: each within U * (sqrt(128) * |logit| + 2 sqrt(rows)) * 8 < 2e-4 of |v| <= 5
            assert float((want - out[:, slot:slot + 1]).abs().max()) < 2e-3
        assert not out[:, 3].any() and (i < 10 or not out[:, 1].any())
    assert len(s.host.free) == 120 - -(-620 // 16) - -(-21 // 16)
    ctx.sync()
    seq = s.open()                                      # a closed sequence's place and pages are used again
    assert seq == 1
    q, k, v = H.inputs(200, L, 0, 50)
    models[1].reset()
    want, got = models[1].prefill(q, k, v), s.prefill(1, q, k, v)
    assert float((want - got).abs().max()) < 2 * H.MAX_ABS
    with pytest.raises(qattn.QAttnError):
        s.prefill(1, q, k, v)
    with pytest.raises(qattn.QAttnError):
        s.prefill(3, q, k, v)
    with pytest.raises(qattn.QAttnError):
        s.append(q, k, v)
    ctx.sync()


def test_sequences_keep_a_budget_by_eviction():
    """A sequence decodes far past its cache: rows stay under the budget, positions go on, and the
    outputs are those of attention over the kept rows."""
    from fpga_qwen_b200.paged import PagedSequences
    L, budget, recent = 2, 64, 16
    ctx = make(L, 4, context=256)
    s = PagedSequences(ctx, n_pages=14, page_rows=16, max_seqs=2, max_rows=96, max_position=5000)
    seq = s.open()
    g = torch.Generator("cuda").manual_seed(1)
    q, k, v = (torch.randn(L, 40, h, D, device="cuda", generator=g) for h in (8, 4, 4))
    s.prefill(seq, q, k, v)
    keys, values = [], []                               # per step: the cached rows, as FP16
    for i in range(150):
        s.begin_step()
        q, k, v = (torch.randn(L, 2, h, D, device="cuda", generator=g) for h in (8, 4, 4))
        qn = s.append(q, k, v)
        out = s.attend(qn)
        n = s.rows(seq)
        t = torch.arange(n, device="cuda")
        ids, at = s.table[seq].long()[t // 16], t % 16
        rows = s.kv[ids, :, :, :, at].permute(1, 2, 3, 0, 4).double()
        p = torch.softmax(torch.einsum("lhgd,lhtd->lhgt", qn[:, 0].double().view(L, 4, 2, D), rows[:, 0]) / math.sqrt(D), -1)
        want = torch.einsum("lhgt,lhtd->lhgd", p, rows[:, 1]).reshape(L, 8, D)
        # U * (sqrt(128) * 40 + 2 * sqrt(96)) * 8 < 3e-4 of |v| <= 5
        assert float((out[:, 0].double() - want).abs().max()) < 1.5e-3
        assert not out[:, 1].any()
        if n >= 90:
            held = s.weights[ids, :, :, at].permute(1, 2, 0).cpu().numpy()
            kept = s.evict(budget, recent)
            assert s.rows(seq) == budget and s.position(seq) == 41 + i
            for layer in range(L):
                for h in range(4):
                    assert kept[seq, layer, h].tolist() == kept_rows(held[layer, h].tolist(), budget, recent)
    assert s.position(seq) == 190 and len(s.host.free) == 14 - -(-s.rows(seq) // 16)
    assert s.lengths.tolist() == [s.rows(seq), 0]
    with pytest.raises(qattn.QAttnError):
        s.evict(0)
    ctx.sync()


def test_sequences_captured_steps_stay_valid_and_shapes_are_checked():
    """One captured step (append and attention of every layer) replayed while sequences grow, close and
    are evicted gives the same as the calls; wrong shapes are refused."""
    from fpga_qwen_b200.paged import PagedSequences
    L, hkv = 2, 2

    def build():
        ctx = make(L, hkv, context=128)
        s = PagedSequences(ctx, n_pages=40, page_rows=16, max_seqs=3, max_rows=128, max_position=1000)
        g = torch.Generator("cuda").manual_seed(9)
        for n in (50, 17, 1):
            q, k, v = (torch.randn(L, n, h, D, device="cuda", generator=g) for h in (4, 2, 2))
            s.prefill(s.open(), q, k, v)
        return ctx, s
    results = []
    for captured in (True, False):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            ctx, s = build()
            q, k, v = (torch.zeros(L, 3, h, D, device="cuda") for h in (4, 2, 2))
            qn, out = torch.empty_like(q), torch.empty_like(q)

            def step():
                s.append(q, k, v, q_out=qn)
                s.attend(qn, out=out)
            run = step
            if captured:
                stream.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    step()
                run = graph.replay
            seen = []
            g = torch.Generator("cuda").manual_seed(10)
            for i in range(40):
                if i == 15:
                    s.close(1)
                if i == 20:
                    s.evict(32, 8)
                s.begin_step()
                for t in (q, k, v):
                    t.copy_(torch.randn(t.shape, device="cuda", generator=g))
                run()
                seen.append(out.clone())
            stream.synchronize()
            ctx.sync()
            results.append(seen)
            for bad in (lambda: s.attend(qn[:, :2]), lambda: s.attend(qn.half()), lambda: s.append(q, k, v, q_out=qn[:1]),
                        lambda: s.attend(qn, out=out[:1]), lambda: s.append(q, k[..., :64], v)):
                with pytest.raises(qattn.QAttnError) as err:
                    bad()
                assert err.value.status == qattn.QA_ERR_INVALID
    for x, y in zip(*results):
        assert torch.equal(x, y)
    ctx = make(L, hkv, context=128)
    one = PagedSequences(ctx, n_pages=4, max_seqs=1, max_rows=32, step_layers=1)
    one.open()
    one.begin_step()
    q, k, v = (torch.randn(L, 1, h, D, device="cuda") for h in (4, 2, 2))
    qn = one.append(q, k, v)
    one.attend(qn[1:], 1)
    with pytest.raises(qattn.QAttnError):
        one.attend(qn)                                  # its workspace holds one layer
    ctx.sync()


def test_sequences_prefilled_within_a_step_join_at_the_next():
    """A prompt that arrives between begin_step and append is no part of the step: the step writes no row of
    it and gives zeros; an eviction sees all its rows, and the next step appends behind them."""
    from fpga_qwen_b200.paged import PagedSequences
    L, hkv = 2, 2
    ctx = make(L, hkv, context=128)
    s = PagedSequences(ctx, n_pages=40, page_rows=16, max_seqs=3, max_rows=128)
    g = torch.Generator("cuda").manual_seed(11)

    def draw(n):
        return [torch.randn(L, n, h, D, device="cuda", generator=g) for h in (4, 2, 2)]

    def cached(seq):
        t = torch.arange(s.rows(seq), device="cuda")
        return s.kv[s.table[seq].long()[t // 16], :, :, :, t % 16].clone()
    s.prefill(s.open(), *draw(20))
    s.begin_step()
    late = s.open()
    s.prefill(late, *draw(50))
    before = cached(late)
    out = s.attend(s.append(*draw(3)))
    assert torch.equal(before.view(torch.int16), cached(late).view(torch.int16))
    assert out[:, 0].all() and not out[:, 1:].any()
    third = s.open()
    s.prefill(third, *draw(40))
    kept = s.evict(32, 8)
    # the prompt's rows weigh nothing yet: the lowest 24 and the last 8
    assert kept[late].tolist() == [[list(range(24)) + list(range(42, 50))] * hkv] * L
    assert kept[third].tolist() == [[list(range(24)) + list(range(32, 40))] * hkv] * L
    assert [s.rows(b) for b in range(3)] == [21, 32, 32] and s.lengths.tolist() == [21, 0, 0]
    s.begin_step()
    assert s.lengths.tolist() == [22, 33, 33] and s.positions.tolist() == [21, 50, 40]
    out = s.attend(s.append(*draw(3)))
    assert out.all()
    after = cached(late)
    assert torch.equal(after[:24].view(torch.int16), before[:24].view(torch.int16))
    assert torch.equal(after[24:32].view(torch.int16), before[42:].view(torch.int16))
    ctx.sync()
