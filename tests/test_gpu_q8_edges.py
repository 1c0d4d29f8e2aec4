"""8-bit rows and products at the edges of their definition, on the GPU."""

import pytest
import torch

from tests.test_q8_edges import (check_a_norm_past_the_range, check_codes_behind_a_norm, check_gradients_are_refused,
                                 check_nothing_is_broadcast, every_value_and_peak)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 8, 100, None])
def test_codes_are_the_definition_and_the_cpu_forms(rows):
    """Every kernel that writes codes: rne(127 y / a) exactly, so the bits of the CPU's form too.
    The product's own quantisation (1 and 8 rows) shows through a weight that copies its column."""
    from nanokv_amd.q8 import Q8, linear_q8, quantize_q8
    x, codes = every_value_and_peak("cuda")
    assert torch.equal(quantize_q8(x).q.long(), codes)
    eye = Q8(torch.eye(16, dtype=torch.int8, device="cuda"), torch.ones(16, device="cuda"))
    if rows is None:
        wide = x.view(-1, 16 * 128)                # other rows share a peak: against the CPU's form
        a, b = quantize_q8(wide), quantize_q8(wide.cpu())
        assert torch.equal(a.q.cpu(), b.q) and torch.equal(a.scale.cpu(), b.scale)
        return
    scale = quantize_q8(x).scale
    want = (codes.float() * scale[:, None]).bfloat16()
    ties = (x[:, 1:].double().abs() * 254 / x[:, :1].double() % 2 == 1).any(-1).nonzero()[:, 0]
    at = ties[:: max(1, len(ties) // 40)]          # rows that hold a value half way between two codes
    for i in at.tolist():
        i = min(i, x.shape[0] - rows)
        assert torch.equal(linear_q8(x[i:i + rows], eye), want[i:i + rows])


def test_codes_behind_a_norm_are_the_cpu_forms():
    """t * w is one fp32 rounding on both sides, and the codes do not depend on the sum of squares."""
    from nanokv_amd.q8 import rmsnorm_q8
    g = torch.Generator().manual_seed(3)
    for rows, n in ((1, 2560), (300, 528), (2, 9728), (1500, 1024)):
        x, r, w = (torch.randn(*s, generator=g).bfloat16() for s in ((rows, n), (rows, n), (n,)))
        for res in (None, r):
            a, _ = rmsnorm_q8(x.cuda(), w.cuda(), 1e-6, None if res is None else res.cuda())
            b, _ = rmsnorm_q8(x, w, 1e-6, res)
            assert torch.equal(a.q.cpu(), b.q)
            # a sum of n squares, 43 roundings at most here and a library's order there, under a root
            assert bool(((a.scale.cpu() - b.scale).abs() <= 2.0 ** -17 * b.scale).all())


def test_operands_that_ask_for_a_gradient_are_refused():
    check_gradients_are_refused("cuda")


def test_nothing_is_broadcast():
    check_nothing_is_broadcast("cuda")


def test_codes_behind_a_norm():
    check_codes_behind_a_norm("cuda")


def test_a_norm_past_the_range():
    check_a_norm_past_the_range("cuda")
