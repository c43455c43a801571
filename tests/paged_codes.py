"""Values under which every row of an attention call shows by itself.

With zero queries every row weighs 1 / rows. Row t's value is one code, of 64 levels, in channel (t / 16) % 128 and zero in
the others, so a channel sums the codes of the 16-row blocks that fall to it, all exactly representable. A row left out,
taken twice or taken in another's place moves its channel by at least 128 / 64 / 2 of its share, and a row missing from
the softmax sum alone moves every channel by 1 / rows.
"""
import torch

D, BLOCK = 128, 16
# exp2f of a whole number is exact (the GPU test looks), so all weights are one power of two; every sum is then a whole
# number, below 2^24, of a code's smallest step, and exact in any order. What is left is a division, or a reciprocal and
# a product: at most 2^-22, and a factor of four on top.
EXACT = 2.0 ** -20


def codes(rows, device="cpu", salt=0):
    """[rows][128] FP16."""
    t = torch.arange(rows, device=device)
    v = torch.zeros(rows, D, dtype=torch.float16, device=device)
    v[t, t // BLOCK % D] = (1 + ((t * 7919 + (t // (BLOCK * D)) * 31 + salt) % 64).double() / 64).half()
    return v
