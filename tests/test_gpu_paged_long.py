"""GPU: attention over long histories, so that a single row that is lost, doubled or misplaced shows."""
import numpy as np
import pytest
import torch

from tests.paged_codes import EXACT, codes
from tests.test_gpu_paged import Cache, attend, make, reference

pytestmark = pytest.mark.gpu

# (lengths, layers, KV heads, page): clusters, CTAs and half-size CTAs for a unit, even splits with units over many ranges
SHAPES = [([200001, 3], 1, 2, 64), ([131071, 77777], 1, 8, 64), ([40000], 1, 1, 16), ([100003], 3, 8, 512), ([30011], 7, 8, 32),
          ([20011], 28, 8, 64), ([4096, 0, 1, 3001, 17, 2500, 4095, 777], 1, 8, 16), ([1024, 1000, 3], 1, 8, 16), ([2049], 28, 8, 16),
          ([int(x) for x in np.random.default_rng(7).integers(0, 2000, 200)], 1, 2, 128)]


def test_exp2_of_whole_numbers_is_exact():
    x = torch.arange(-126, 128, device="cuda", dtype=torch.float32)
    assert torch.equal(torch.exp2(x), torch.ldexp(torch.ones_like(x), x.int()))


@pytest.mark.parametrize("lengths,layers,hkv,page", SHAPES)
@pytest.mark.parametrize("add", [False, True])
def test_every_row_counts_once(lengths, layers, hkv, page, add):
    """Equal weights over coded values (paged_codes.py): each channel of each head is exact."""
    c = Cache(lengths, layers, hkv, page=page, seed=91)
    for b, m in enumerate(lengths):
        rows = c.rows(b).clone()
        for layer in range(layers):
            for h in range(hkv):
                rows[layer, 1, h] = codes(m, "cuda", salt=b + 3 * layer + 17 * h)
        c.put(b, rows)
        c.put_weights(b, torch.zeros(layers, hkv, m, device="cuda"))
    ctx = make(layers, hkv)
    out = attend(ctx, c, torch.zeros_like(c.query()), add=add)
    ctx.sync()
    for b, m in enumerate(lengths):
        got = out[:, b].double().view(layers, hkv, 2, 128)
        if not m:
            assert not got.any()
            continue
        want = c.rows(b)[:, 1].double().sum(2) / m                       # [layers][hkv][128]
        for head in range(2):
            off = (got[:, :, head] - want).abs()
            assert bool((off <= EXACT * want).all()), (b, head, float(off.max()))
        if add:
            w = c.weights(b).double() * m / 2
            assert bool(((w - 1).abs() <= EXACT).all()), (b, float(w.min()), float(w.max()))


@pytest.mark.parametrize("lengths,layers,hkv,page", SHAPES)
def test_error_in_two_norm(lengths, layers, hkv, page):
    """Random rows: a head's output within 4e-6 of its 2-norm (a 16-row block missing from 200001 rows is 9e-3, one row
    2e-3). A weight's own error is at most some 2e-6: operands and weights of 22 bits (2^-22 each, the logits' over products
    of a 2-norm of about 2), two exp2f of 2 ulp each, roundings of sums; those of different rows are unlike, and so is
    what they add to the output; as much again for what is common to all rows."""
    c = Cache(lengths, layers, hkv, page=page, seed=92, weights=False)
    ctx = make(layers, hkv)
    q = c.query()
    out = attend(ctx, c, q)
    ctx.sync()
    want, _, _ = reference(c, q)
    off = (out.double() - want).norm(dim=-1)
    assert bool((off <= 4e-6 * want.norm(dim=-1)).all()), float((off / want.norm(dim=-1).clamp(min=1e-30)).max())
