"""GPU: where the weights of a row, or the operands of a product, lie far apart.

Bounds of qa_paged_attn that the tolerances count (csrc/attn_paged.cu): queries and softmax weights are sums of two
FP16 halves, 2^-22 of the value or 2^-36 of the largest query channel, 2^-37 of the largest weight of the row's
16-row block; sums are FP32.
"""
import math

import pytest
import torch

from tests.test_gpu_paged import Cache, attend, i32, make

pytestmark = pytest.mark.gpu

D = 128
BLOCK = 16


def weights_and_limits(q, k, v):
    """(out, limit) in 64 bits of queries q [heads][128] over k, v [rows][128]: each weight may be off by
    * its logit's error: operands of 22 bits, a scale, sums of at most two product steps and of eight terms, and the
      differences to the block's and the running maximum: below 2^-20 of the logit (the largest product is the logit
      itself in these tests);
    * exp2f of both differences (2 ulp each), the 22 bits of the weight and the roundings of the sums, at most 200 in a
      chain (blocks of a warp, warps, ranges) for numerator and denominator: below 2^-15;
    * 2^-37 of the largest weight in its block."""
    s = q.double() @ k.double().T / math.sqrt(D)
    p = torch.softmax(s, -1)
    rows = p.shape[1]
    pad = torch.nn.functional.pad(p, (0, -rows % BLOCK))
    top = pad.view(p.shape[0], -1, BLOCK).amax(-1, keepdim=True).expand(-1, -1, BLOCK).reshape(p.shape[0], -1)[:, :rows]
    off = p * (2.0 ** -15 + 2.0 ** -20 * s.abs()) + 2.0 ** -37 * top
    return p @ v.double(), off @ v.double().abs()


def far_apart(rows, hkv, page, every, seed, queries=1):
    """One sequence (`queries` table rows share its pages): one row in `every` weighs most, all others lie 25, 28, 40 or 80
    nats below, by KV head. The heavy rows' values are 0.01, the light ones' 1000 and more, all of one sign."""
    c = Cache([rows], 1, hkv, page=page, seed=seed)
    data = torch.zeros(1, 2, hkv, rows, D, device="cuda", dtype=torch.float16)
    data[0, 0, :, :, 0] = 0.25 * torch.rand(hkv, rows, device="cuda", generator=c.g)     # light: logits of 0 to 2
    data[0, 1] = 1000 + 500 * torch.rand(hkv, rows, D, device="cuda", generator=c.g)
    for h in range(hkv):
        data[0, 0, h, ::every, 0] = (2 + (25, 28, 40, 80)[h % 4]) / 8
    data[0, 1, :, ::every] = 0.01
    c.put(0, data)
    q = torch.zeros(1, queries, 2 * hkv, D, device="cuda")
    q[..., 0] = 8 * math.sqrt(D)
    c.table = c.table.expand(queries, -1).contiguous()
    c.lengths = [rows] * queries
    return c, q


@pytest.mark.parametrize("rows,queries,every", [(131071, 1, 1 << 30), (131071, 1, 997), (131071, 48, 1 << 30), (131071, 3, 500),
                                                (5000, 100, 1 << 30), (700, 1, 1 << 30), (40, 300, 1 << 30), (17, 1, 16)])
@pytest.mark.parametrize("add", [False, True])
def test_light_rows_next_to_heavy_ones(rows, queries, every, add):
    hkv = 4
    c, q = far_apart(rows, hkv, 64, every, rows + queries, queries)
    ctx = make(1, hkv)
    out = attend(ctx, c, q, add=add)
    ctx.sync()
    k, v = c.rows(0)[0].unbind(0)
    for h in range(hkv):
        want, limit = weights_and_limits(q[0, 0, 2 * h:2 * h + 2], k[h], v[h])
        off = (out[0, :, 2 * h:2 * h + 2].double() - want).abs()
        assert bool((off <= limit).all()), (h, float((off / limit).max()), float((off / want.abs()).max()))
