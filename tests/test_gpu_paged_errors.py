"""GPU: errors of paged calls and calls on slots do not touch one another.

Bad lengths and page ids are checked by the kernels before they are used (walked on the CPU in test_paged_index.py), so
none of these calls leaves the pool or the tables.
"""
import numpy as np
import pytest
import torch

from fpga_qwen_b200 import qattn
from tests.test_gpu_paged import Cache, i32, make

pytestmark = pytest.mark.gpu

LIMIT_US = 20000          # of a wait made to run out


def bad_evict(ctx, c, what="page"):
    """An eviction whose second sequence has a page id or a length outside its range."""
    table, lens = c.table.clone(), i32(c.lengths)
    if what == "page":
        table[1, 0] = c.n_pages
    else:
        lens[1] = c.cols * c.page + 1
    n = len(c.lengths)
    new, kept = i32([0] * n), torch.empty(n, c.layers, c.hkv, 8, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ctx.paged_evict(c.pages, table.data_ptr(), c.cols, table.data_ptr(), c.cols, lens.data_ptr(), new.data_ptr(), n, 8, 2,
                    kept.data_ptr())
    torch.cuda.synchronize()


@pytest.mark.parametrize("what,code", [("page", 62), ("length", 61)])
def test_a_bad_eviction_leaves_the_slots_of_a_host_buffer_context_alone(what, code):
    L, hkv, n = 2, 8, 40
    ctx, plain = (make(L, hkv, context=64, max_seqs=2, io_host=1) for _ in range(2))
    c = Cache([30, 20], L, hkv, seed=71)
    r = np.random.default_rng(72)
    q, k, v = (r.standard_normal((L, n, h, 128), dtype=np.float32) for h in (2 * hkv, hkv, hkv))
    row = [np.ascontiguousarray(t[:, :1]) for t in (q, k, v)]
    w = r.standard_normal((64, 128)).astype(np.float16)
    results = []
    for x in (ctx, plain):
        qn, out, qr, step, y = np.empty_like(q), np.empty_like(q), np.empty_like(row[0]), np.empty_like(row[0]), np.empty((1, 64), np.float32)
        x.append(0, 0, L, 0, n, q.ctypes.data, k.ctypes.data, v.ctypes.data, qn.ctypes.data)
        if x is ctx:
            bad_evict(x, c, what)
        x.attn_prefill(0, 0, L, 0, n, qn.ctypes.data, out.ctypes.data)
        x.commit(0, n)
        if x is ctx:
            bad_evict(x, c, what)
        x.decode_step(0, 0, L, n, *(t.ctypes.data for t in row), qr.ctypes.data, step.ctypes.data)
        assert x.position(0) == n
        x.commit(0, 1)
        wd = torch.from_numpy(w).cuda()
        torch.cuda.synchronize()
        x.project(wd.data_ptr(), 64, 128, q.ctypes.data, 1, y.ctypes.data)
        assert x.position(0) == n + 1
        results.append((qn, out, qr, step, y))
    for a, b in zip(*results):
        assert np.array_equal(a, b)
    plain.sync()
    with pytest.raises(qattn.QAttnError) as err:        # still there for the program to see, once
        ctx.sync()
    assert err.value.status == qattn.QA_ERR_INVALID and f"code {code}" in str(err.value)
    assert ctx.position(0) == n + 1
    ctx.sync()


def test_a_paged_host_buffer_call_reports_the_eviction_before_it():
    L, hkv = 2, 8
    ctx = make(L, hkv, io_host=1)
    c = Cache([30, 20], L, hkv, seed=73)
    q = np.zeros((L, 2, 2 * hkv, 128), np.float32)
    out = np.empty_like(q)
    lens = i32(c.lengths)
    size = ctx.paged_workspace(2, L, c.cols * c.page, False)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    args = (c.pages, c.table.data_ptr(), c.cols, lens.data_ptr(), 2, 0, L, q.ctypes.data, out.ctypes.data, False, ws.data_ptr(), size)
    bad_evict(ctx, c)
    with pytest.raises(qattn.QAttnError) as err:
        ctx.paged_attn(*args)
    assert err.value.status == qattn.QA_ERR_INVALID and "code 62" in str(err.value)
    ctx.paged_attn(*args)
    ctx.sync()


def test_bad_data_does_not_hide_an_expired_wait():
    ctx = make(1, 8)
    c = Cache([30, 20], 1, 8, seed=74)
    bad_evict(ctx, c)
    ctx.set_wait_limit(LIMIT_US)
    ctx.selftest_timeout()
    with pytest.raises(qattn.QAttnError) as err:
        ctx.sync()
    assert err.value.status == qattn.QA_ERR_TIMEOUT and "code 51" in str(err.value)
    with pytest.raises(qattn.QAttnError) as err:
        ctx.sync()
    assert err.value.status == qattn.QA_ERR_INVALID and "code 62" in str(err.value)
    ctx.sync()
    # the other way round, in a host-buffer context: the slot's call reports the wait and resets its sequence
    L, n = 1, 5
    ctx = make(L, 8, context=64, io_host=1)
    r = np.random.default_rng(75)
    q, k, v = (r.standard_normal((L, n, h, 128), dtype=np.float32) for h in (16, 8, 8))
    qn, step = np.empty_like(q), np.empty((L, 1, 16, 128), np.float32)
    ctx.append(0, 0, L, 0, n, q.ctypes.data, k.ctypes.data, v.ctypes.data, qn.ctypes.data)
    ctx.commit(0, n)
    ctx.set_wait_limit(LIMIT_US)
    ctx.selftest_timeout()
    bad_evict(ctx, c, "length")
    with pytest.raises(qattn.QAttnError) as err:
        ctx.decode_step(0, 0, L, n, *(t[:, :1].copy().ctypes.data for t in (q, k, v)), 0, step.ctypes.data)
    assert err.value.status == qattn.QA_ERR_TIMEOUT and ctx.position(0) == 0
    with pytest.raises(qattn.QAttnError) as err:
        ctx.sync()
    assert err.value.status == qattn.QA_ERR_INVALID and "code 61" in str(err.value)
    ctx.sync()
