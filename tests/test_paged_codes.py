"""CPU: the codes of paged_codes.py show every mistake with a row, under the tolerance that the GPU tests use."""
import random

import pytest
import torch

from tests.paged_codes import BLOCK, D, EXACT, codes


def seen(want, got):
    return bool(((got - want).abs() > EXACT * want.abs()).any())


@pytest.mark.parametrize("rows", [1, 17, 2049, 40000, 200001])
def test_a_row_lost_doubled_or_replaced_is_seen(rows):
    v = codes(rows).double()
    assert torch.equal(v, v.half().double()) and bool((v.amax(1) >= 1).all()) and bool(((v > 0).sum(1) == 1).all())
    total = v.sum(0)
    want = total / rows
    assert not seen(want, (total / rows).float().double())
    r = random.Random(rows)
    blocks = -(-rows // BLOCK)
    at = {0, rows - 1} | {r.randrange(rows) for _ in range(300)}
    for t in at:
        if rows > 1:
            assert seen(want, (total - v[t]) / rows)                # missing from the numerator
            assert seen(want, (total - v[t]) / (rows - 1))          # missing altogether
            assert seen(want, total / (rows - 1))                   # missing from the sum
        assert seen(want, (total + v[t]) / rows)
        assert rows == 1 or seen(want, (total + v[t]) / (rows + 1))
        for other in (t + 1, t + BLOCK, t + BLOCK * D):             # its neighbour's place, block's or channel's
            if other < rows:
                assert seen(want, (total - v[t] + v[other]) / rows), (t, other)
    for b in {0, blocks - 1} | {r.randrange(blocks) for _ in range(100)}:
        part = v[b * BLOCK:(b + 1) * BLOCK]
        n = part.shape[0]
        if rows > n:
            assert seen(want, (total + part.sum(0)) / (rows + n)) and seen(want, (total - part.sum(0)) / (rows - n))
