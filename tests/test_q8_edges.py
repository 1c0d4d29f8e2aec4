"""8-bit rows and products at the edges of their definition, without a GPU."""

import pytest
import torch

from nanokv_amd.q8 import quantize_q8


# -- the code of every bf16 value under every bf16 peak ------------------------------
def every_value_and_peak(device="cpu"):
    """(x [rows, 16] bf16, codes): rows of one peak and 15 values below it, of every pair of
    mantissas 2^0 to 2^-8 apart, and rne(127 y / a) of them in integers."""
    mant = torch.arange(128, 256)
    xs, codes = [], []
    for e in range(9):
        a, y = torch.meshgrid(mant, mant, indexing="ij")
        below = y <= (a << e)
        n, d = 127 * y, a << e
        up = (2 * n + d) // (2 * d)                                  # floor(n / d + 1/2)
        up -= (((2 * n + d) % (2 * d) == 0) & (up % 2 == 1)).long()  # a tie goes to the even code
        # (128 values a peak, in rows of 15 behind it; values above the peak and the filling are 0)
        val = torch.where(below, y.float() * 2.0 ** -e, torch.zeros(()))
        up = torch.where(below, up, torch.zeros((), dtype=torch.long))
        val, up = (torch.nn.functional.pad(t, (0, 7)).view(128, 9, 15) for t in (val, up))
        sign = torch.where((torch.arange(15) % 2).bool(), -1, 1)
        xs.append(torch.cat([a[:, :1, None].float().expand(128, 9, 1), val * sign], -1).view(-1, 16))
        codes.append(torch.cat([torch.full((128, 9, 1), 127), up * sign], -1).view(-1, 16))
    return (torch.cat(xs) * 2.0 ** -9).bfloat16().to(device), torch.cat(codes).to(device)


def test_codes_are_the_nearest_with_ties_to_even():
    """q = rne(127 y / a), exactly: 254 of the 139328 pairs lie half way between two codes."""
    x, codes = every_value_and_peak()
    assert torch.equal(quantize_q8(x).q.long(), codes)
    big = quantize_q8(x * 2.0 ** 100)
    assert torch.equal(big.q.long(), codes)
