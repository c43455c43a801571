"""GPU: the order of PagedSequences' calls within a step."""
import pytest
import torch

from fpga_qwen_b200 import qattn
from fpga_qwen_b200.paged import PagedSequences
from tests.test_gpu_paged import make

pytestmark = pytest.mark.gpu

L, HKV = 2, 2


def build(rows=(), **kw):
    ctx = make(L, HKV, context=128)
    s = PagedSequences(ctx, **{**dict(n_pages=40, page_rows=16, max_seqs=3, max_rows=128), **kw})
    g = torch.Generator("cuda").manual_seed(81)

    def draw(n, layers=L):
        return [torch.randn(layers, n, h, 128, device="cuda", generator=g) for h in (2 * HKV, HKV, HKV)]
    for n in rows:
        s.prefill(s.open(), *draw(n))
    return ctx, s, draw


def refused(call, status=qattn.QA_ERR_STATE):
    with pytest.raises(qattn.QAttnError) as err:
        call()
    assert err.value.status == status


def state(s):
    return ([list(p) if p else p for p in s.host.pages], list(s.host.rows), list(s.host.position), list(s.host.free),
            s.lengths.tolist(), s.positions.tolist(), s.table.clone(), s.kv.clone(), s.weights.clone())


def same(a, b):
    return all(torch.equal(x, y) if isinstance(x, torch.Tensor) else x == y for x, y in zip(a, b))


def test_a_step_whose_rows_are_not_written_lets_nothing_read_or_count_them():
    """On pages whose former owner left heavy weights: between begin_step and the last layer's append neither an
    eviction nor another begin_step nor attention of an unwritten layer runs; each is refused and changes nothing."""
    ctx, s, draw = build((60,))
    s.weights.fill_(100.0)                              # of a former owner
    s.weights[s.table[0, :4].long()] = 0.25
    s.begin_step()
    q, k, v = draw(3)
    one, two = ([t[i:i + 1] for t in (q, k, v)] for i in range(2))
    calls = [lambda: s.evict(16), lambda: s.evict(16, 4), s.begin_step, lambda: s.attend(torch.zeros_like(q))]
    before = state(s)
    for call in calls:
        refused(call)
    assert same(before, state(s))
    qn = s.append(*one, layer=0)
    s.attend(qn, layer=0)
    before = state(s)
    for call in calls + [lambda: s.attend(torch.zeros_like(qn), layer=1)]:
        refused(call)
    assert same(before, state(s))
    refused(lambda: s.append(q[:1, :2], k[:1], v[:1], layer=1), qattn.QA_ERR_INVALID)    # a refused append writes nothing
    refused(lambda: s.evict(16))
    qn = s.append(*two, layer=1)
    # every layer is written: rows of a weight of 0.25, less the new row, whose weight starts at zero
    kept = s.evict(16)
    assert kept[0, 1].tolist() == [list(range(16))] * HKV
    assert s.rows(0) == 16 and s.position(0) == 61 and s.lengths.tolist() == [16, 0, 0]
    s.attend(qn, layer=1)
    s.begin_step()
    s.append(*draw(3))
    assert s.lengths.tolist() == [17, 0, 0] and s.positions.tolist() == [61, 0, 0]
    ctx.sync()


def test_closing_the_sequences_of_a_step_ends_it():
    ctx, s, draw = build((20, 33))
    s.begin_step()
    s.close(0)
    refused(lambda: s.evict(16))
    refused(s.begin_step)
    late = s.open()                                     # takes no part in the step
    s.prefill(late, *draw(30))
    s.close(1)
    kept = s.evict(16)
    assert s.rows(late) == 16 and kept[late, 0, 0].tolist() == list(range(16))
    s.begin_step()
    out = s.attend(s.append(*draw(3)))
    assert out[:, late].all() and not out[:, 1:].any()
    ctx.sync()


def test_a_step_that_does_not_fit_is_no_step():
    ctx, s, draw = build((32, 32), n_pages=4)
    refused(s.begin_step, qattn.QA_ERR_CAPACITY)
    assert s.lengths.tolist() == [0, 0, 0]
    s.evict(16)
    s.begin_step()
    s.append(*draw(3))
    s.evict(16)
    ctx.sync()


def test_replayed_steps_are_the_callers_to_order():
    """Once an append was captured, replays cannot be seen: begin_step and evict take the step as made."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx, s, draw = build((20, 33))
        s.begin_step()                                  # the first step is made by the graph's first replay
        q, k, v = draw(3)
        qn, out = torch.empty_like(q), torch.zeros_like(q)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            s.append(q, k, v, q_out=qn)
            s.attend(qn, out=out)
        graph.replay()
        s.begin_step()
        graph.replay()
        s.evict(16, 2)
        s.begin_step()
        graph.replay()
        stream.synchronize()
        assert s.lengths.tolist() == [17, 17, 0] and s.positions.tolist() == [22, 35, 0] and out[:, :2].all()
        ctx.sync()


def test_host_bookkeeping_is_refused_under_capture():
    """A replay repeats the device's part alone: calls that also keep the host's books run outside a graph, and one made
    inside changes neither side and leaves the capture valid."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx, s, draw = build((32, 33))
        s.begin_step()
        s.append(*draw(3))
        q, k, v = draw(3)
        qn, out = torch.empty_like(q), torch.zeros_like(q)
        late, prompt = s.open(), draw(5)
        before = state(s)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            refused(s.begin_step)
            refused(lambda: s.evict(16))
            refused(lambda: s.close(0))
            refused(lambda: s.prefill(late, *prompt))
            s.append(q, k, v, q_out=qn)
            s.attend(qn, out=out)
        assert same(before, state(s))
        s.begin_step()
        graph.replay()
        stream.synchronize()
        assert s.lengths.tolist() == [34, 35, 1] and out.all()
        s.close(0)
        s.evict(16)
        assert [s.rows(b) for b in (1, late)] == [16, 1]
        ctx.sync()
