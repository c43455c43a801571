"""GPU: paged calls of several contexts, each on its own host thread."""
import threading

import pytest
import torch

from fpga_qwen_b200 import qattn
from tests.test_gpu_paged import Cache, i32, make

pytestmark = pytest.mark.gpu


def test_evictions_of_contexts_on_their_own_host_threads():
    """Contexts on one GPU, each with its own thread and stream, whose selections take unlike amounts of shared memory
    (36 to 64 KB: as many rows as their tables can hold): every call is accepted and right."""
    L, hkv, rounds, calls = 28, 8, 120, 50
    tables, errors, jobs = (16384, 9216, 14336, 10240), [], []
    for i, rows in enumerate(tables):
        c = Cache([40], L, hkv, seed=76 + i, extra_cols=rows // 16 - 3)
        assert c.cols * 16 == rows
        s = torch.cuda.Stream()
        ctx = make(L, hkv)
        ctx.set_stream(s.cuda_stream)
        jobs.append((ctx, c, i32([40]), i32([0]), torch.zeros(1, L, hkv, 40, dtype=torch.int32, device="cuda"), s))
    torch.cuda.synchronize()
    start = threading.Barrier(len(jobs))

    def work(ctx, c, lens, new, out, _):
        args = (c.pages, c.table.data_ptr(), c.cols, c.table.data_ptr(), c.cols, lens.data_ptr(), new.data_ptr(), 1, 40, 4, out.data_ptr())
        start.wait()
        try:
            for _ in range(rounds):
                for _ in range(calls):                  # all rows stay: every call gives the same
                    ctx.paged_evict(*args)
                ctx.sync()
        except qattn.QAttnError as e:
            errors.append(str(e))
    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for j in jobs:
        assert j[3].tolist() == [40] and bool((j[4] == torch.arange(40, device="cuda")).all())
