"""Every kernel of the 8-bit products against the definition in 64 bits, at sizes that are
ragged on all sides; tolerances as in test_gpu_q8."""

import pytest
import torch

from tests.test_gpu_q8 import _check_codes, _check_gated, _check_product, _codes, _gen, _hidden
from tests.test_q8_edges import CUT_TILES, TILES, tile_of

pytestmark = pytest.mark.gpu


def _check(m, n, k, gated):
    """The product of m rows, and the same bits from 16 of its rows at a time (the kernel of
    few rows: sums are exact and every kernel rounds alike)."""
    from nanokv_amd.q8 import Q8, linear_q8, linear_silu_mul_q8
    x, w = _codes(m, k, seed=m + k, lo=-128), _codes(n * (1 + gated), k, seed=n, lo=-128)
    x = Q8(x.q, x.scale * (20 / k ** 0.5))
    bias = torch.randn(n, generator=_gen(n), device="cuda").bfloat16()
    run = linear_silu_mul_q8 if gated else (lambda x, w: linear_q8(x, w, bias))
    y = run(x, w)
    if gated:
        _check_gated(y, x, w)
    else:
        _check_product(y, x, w, bias)
        _check_product(linear_q8(x, w), x, w)
    for at in sorted({0, *range(0, m, max(16, m // 20)), max(0, m - 16)}):
        part = slice(at, at + 16)
        assert tile_of(min(16, m - at), n, k, gated)[0] == (0, 0)
        assert torch.equal(y[part], run(Q8(x.q[part], x.scale[part]), w)), at


@pytest.mark.parametrize("k,wide", [(144, False), (1040, False), (1040, True)])
@pytest.mark.parametrize("m,n,gated,tile", TILES)
def test_every_tile(m, n, gated, tile, k, wide):
    if wide:                                       # rows of y that are stored 4 channels at a time
        n = (n + 3) // 4 * 4
    assert tile_of(m, n, k, gated) == (tile, 1)
    _check(m, n, k, gated)


@pytest.mark.parametrize("m,n,k,gated,tile", CUT_TILES)
def test_every_tile_of_a_cut_k(m, n, k, gated, tile):
    assert tile_of(m, n, k, gated)[0] == tile and tile_of(m, n, k, gated)[1] > 1
    _check(m, n, k, gated)


@pytest.mark.parametrize("m,n,k,gated,tile", [(4095, 2553, 4096, 0, (160, 256)), (2777, 2555, 9728, 0, (128, 256)),
                                              (2777, 9725, 2560, 1, (256, 256))])
def test_a_prompt_chunks_products(m, n, k, gated, tile):
    """o, down and gate|up of a chunk, with a row and a few channels cut off."""
    assert tile_of(m, n, k, gated) == (tile, 1)
    _check(m, n, k, gated)


@pytest.mark.parametrize("n", [33, 4097])
@pytest.mark.parametrize("k", [16, 1040, 2064, 4096, 4112, 6160, 8192, 9728, 12288])
def test_one_row_of_every_length(n, k):
    """A token's products: k of every number of 1024-code chunks that the kernel is built for."""
    from nanokv_amd.q8 import (linear_q8, linear_silu_mul_q8, norm_linear_q8, norm_linear_silu_mul_q8, quantize_q8,
                               rmsnorm_q8)
    x, res, w = _hidden(1, k, k), _hidden(1, k, 9 * k), _codes(2 * n, k, seed=n)
    w = type(w)(w.q, w.scale * (10 / k ** 0.5))
    half = type(w)(w.q[:n], w.scale[:n])
    bias = torch.randn(n, generator=_gen(n), device="cuda").bfloat16()
    t = quantize_q8(x)
    assert torch.equal(linear_q8(x, half, bias), linear_q8(t, half, bias))
    assert torch.equal(linear_silu_mul_q8(x, w), linear_silu_mul_q8(t, w))
    _check_product(linear_q8(x, half, bias), t, half, bias)
    _check_gated(linear_silu_mul_q8(x, w), t, w)
    wn = (1 + 0.2 * torch.randn(k, generator=_gen(k), device="cuda")).bfloat16()
    for r in (None, res):
        t, want = rmsnorm_q8(x, wn, 1e-6, r)
        y, got = norm_linear_q8(x, wn, 1e-6, half, r, bias)
        assert torch.equal(got, want)
        _check_product(y, t, half, bias, 2.0 ** -18)
        y, got = norm_linear_silu_mul_q8(x, wn, 1e-6, w, r)
        assert torch.equal(got, want)
        _check_gated(y, t, w, 2.0 ** -9)


@pytest.mark.parametrize("rows", [3, 1030])
@pytest.mark.parametrize("n", [16, 512, 528, 1024, 1040, 2048, 2064, 2560, 2576, 4096, 4112, 8192, 8208, 12288, 12304, 16384, 16400,
                               32768])
def test_rows_of_every_length(rows, n):
    """Both ends of every range of row lengths that has a kernel of its own."""
    from nanokv_amd.q8 import quantize_q8, rmsnorm_q8
    x, res = _hidden(rows, n, rows + n), _hidden(rows, n, 9 * n, 2.0)
    w = (1 + 0.2 * torch.randn(n, generator=_gen(n), device="cuda")).bfloat16()
    t, cpu = quantize_q8(x), quantize_q8(x.cpu())
    assert torch.equal(t.q.cpu(), cpu.q) and torch.equal(t.scale.cpu(), cpu.scale)
    _check_codes(t, x.double(), 2.0 ** -16)
    for r in (None, res):
        t, out = rmsnorm_q8(x, w, 1e-6, r)
        s = x.double() if r is None else x.double() + r.double()
        assert out is x if r is None else torch.equal(out, (x.float() + r.float()).bfloat16())
        _check_codes(t, s * torch.rsqrt(s.square().mean(-1, keepdim=True) + 1e-6) * w.double(), 2.0 ** -14)
