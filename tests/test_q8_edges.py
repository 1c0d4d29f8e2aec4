"""8-bit rows and products at the edges of their definition, without a GPU."""

import pytest
import torch

from nanokv_amd import _lib
from nanokv_amd.q8 import (Q8, dequantize_q8, linear_q8, linear_silu_mul_q8, norm_linear_q8, norm_linear_silu_mul_q8,
                           quantize_q8, rmsnorm_q8)


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


def check_codes_behind_a_norm(device):
    """A code is the nearest integer up to the roundings in front of it, relative to the value:
    t * w, its peak's, 127 / a and the product with it, u = 2^-24 each; with a residual t and its
    peak's t too.  (Not 2^-16 absolute, which moves ten times as many small values.)"""
    g = torch.Generator(device=device).manual_seed(7)
    x, r = (torch.randn(400, 2560, generator=g, device=device).bfloat16() for _ in range(2))
    w = (1 + 0.2 * torch.randn(2560, generator=g, device=device)).bfloat16()
    for res, roundings in ((None, 4), (r, 6)):
        t, _ = rmsnorm_q8(x, w, 1e-6, res)
        y = (x.double() if res is None else x.double() + r.double()) * w.double()
        y *= 127 / y.abs().amax(-1, keepdim=True)
        assert bool(((t.q.double() - y).abs() <= 0.5 + y.abs() * roundings * 2.0 ** -24 * (1 + 2.0 ** -20)).all())


def test_codes_behind_a_norm():
    check_codes_behind_a_norm("cpu")


def check_a_norm_past_the_range(device):
    """|t * weight| is held in fp32 before the root's division: past its range the row is NaN."""
    x = torch.full((2, 32), 100.0).bfloat16().to(device)
    x[1] = 1
    w = torch.full((32,), 2.0 ** 127).bfloat16().to(device)
    t, _ = rmsnorm_q8(x, w, 1e-6)
    assert bool(t.scale[0].isnan()) and not bool(t.q[0].any())
    assert abs(float(t.scale[1]) * 127 / 2.0 ** 127 - 1) < 1e-5 and bool((t.q[1] == 127).all())


def test_a_norm_past_the_range():
    check_a_norm_past_the_range("cpu")


# -- gradients -----------------------------------------------------------------------
def gradient_calls(device="cpu"):
    """(name, call, the operands it takes) with every operand that a gradient could be asked of."""
    g = torch.Generator().manual_seed(1)
    x, r = (torch.randn(3, 32, generator=g).bfloat16().to(device) for _ in range(2))
    wn, b = torch.ones(32, device=device).bfloat16(), torch.zeros(8, device=device).bfloat16()
    w, t = quantize_q8(torch.randn(8, 32, generator=g).bfloat16().to(device)), quantize_q8(x)
    return [("quantize", lambda x: quantize_q8(x), (x,)),
            ("dequantize", lambda s: dequantize_q8(Q8(t.q, s)), (t.scale,)),
            ("rmsnorm", lambda x, wn, r: rmsnorm_q8(x, wn, 1e-6, r), (x, wn, r)),
            ("linear", lambda x, s, b: linear_q8(x, Q8(w.q, s), b), (x, w.scale, b)),
            ("linear of codes", lambda xs, s, b: linear_q8(Q8(t.q, xs), Q8(w.q, s), b), (t.scale, w.scale, b)),
            ("gated", lambda x, s: linear_silu_mul_q8(x, Q8(w.q, s)), (x, w.scale)),
            ("norm, linear", lambda x, wn, s, r, b: norm_linear_q8(x, wn, 1e-6, Q8(w.q, s), r, b), (x, wn, w.scale, r, b)),
            ("norm, gated", lambda x, wn, s, r: norm_linear_silu_mul_q8(x, wn, 1e-6, Q8(w.q, s), r), (x, wn, w.scale, r))]


def check_gradients_are_refused(device):
    from torch.autograd import forward_ad
    for name, call, operands in gradient_calls(device):
        call(*operands)
        for i, t in enumerate(operands):
            asks = t.clone().requires_grad_()
            args = [asks if j == i else o for j, o in enumerate(operands)]
            with pytest.raises(ValueError, match="gradient"):
                call(*args)
                pytest.fail(f"{name}: operand {i}")
            for off in (torch.no_grad, torch.inference_mode):      # (nothing is asked there)
                with off():
                    call(*args)
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(t, torch.ones_like(t))
                with pytest.raises(ValueError, match="gradient"):
                    call(*[dual if j == i else o for j, o in enumerate(operands)])
                call(*operands)


def test_operands_that_ask_for_a_gradient_are_refused():
    check_gradients_are_refused("cpu")
    w = quantize_q8(torch.randn(8, 32))
    for transform in (torch.func.grad, lambda f: lambda x: torch.func.jvp(f, (x,), (x,))):
        with pytest.raises(ValueError, match="gradient"):
            transform(lambda x: linear_q8(x, w).sum())(torch.randn(3, 32))


# -- operands ------------------------------------------------------------------------
def check_nothing_is_broadcast(device):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(3, 32, generator=g).bfloat16().to(device)
    w = quantize_q8(torch.randn(8, 32, generator=g).bfloat16().to(device))
    one, wn = torch.ones(1, device=device).bfloat16(), torch.ones(32, device=device).bfloat16()
    for rows in (x, x[:1], quantize_q8(x)):
        for bias in (one, one[0], one.expand(3, 1), torch.zeros(3, 8, device=device).bfloat16(), one.expand(4)):
            with pytest.raises(ValueError, match="bias"):
                linear_q8(rows, w, bias)
            if not isinstance(rows, Q8):
                with pytest.raises(ValueError, match="bias"):
                    norm_linear_q8(rows, wn, 1e-6, w, None, bias)
    for norm in (lambda wn, r: rmsnorm_q8(x, wn, 1e-6, r), lambda wn, r: norm_linear_q8(x, wn, 1e-6, w, r),
                 lambda wn, r: norm_linear_silu_mul_q8(x, wn, 1e-6, w, r)):
        norm(wn, x)
        for bad in (one, one[0], wn.expand(3, 32), wn[:16]):
            with pytest.raises(ValueError, match="weight"):
                norm(bad, None)
        for bad in (x[:1], x[0], x[:, :1], x.view(3, 1, 32), x.view(1, 3, 32)):
            with pytest.raises(ValueError, match="residual"):
                norm(wn, bad)


def test_nothing_is_broadcast():
    check_nothing_is_broadcast("cpu")


def test_sizes_that_no_c_int_holds_are_refused():
    """ctypes would hand the low 32 bits on: 2^32 + 1 rows would be one."""
    def empty(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="meta")

    def codes(n, k):
        return Q8(empty(n, k, dtype=torch.int8), empty(n, dtype=torch.float32))

    wn = empty(16)
    for rows in (2 ** 31, 2 ** 32 + 1):
        for call in (lambda: quantize_q8(empty(rows, 16)), lambda: dequantize_q8(codes(rows, 16)),
                     lambda: rmsnorm_q8(empty(rows, 16), wn, 1e-6), lambda: linear_q8(empty(rows, 16), codes(4, 16)),
                     lambda: linear_q8(codes(rows, 16), codes(4, 16)),
                     lambda: norm_linear_q8(empty(rows, 16), wn, 1e-6, codes(4, 16)),
                     lambda: linear_q8(empty(2, 16), codes(rows, 16)),
                     lambda: norm_linear_silu_mul_q8(empty(2, 16), wn, 1e-6, codes(rows, 16))):
            with pytest.raises(ValueError, match="at most 2147483647"):
                call()
    k = 2 ** 32 + 16
    for call in (lambda: quantize_q8(empty(1, k)), lambda: linear_q8(empty(2, k), codes(4, k)),
                 lambda: rmsnorm_q8(empty(1, k), empty(k), 1e-6)):
        with pytest.raises(ValueError, match="at most 2147483647"):
            call()


def test_products_that_no_launch_holds_are_refused():
    """2^32 threads: 256 for 16 channels of few rows, 256 or 512 for a tile (addresses are never dereferenced)."""
    lib, gap = _lib.load(), 1 << 44
    w, sw, x, sx, y, ws = (gap * i for i in range(1, 7))
    # (the largest sizes that fit are not called here: without a device the launch itself would fail)
    for m, n in ((2, 2 ** 28), (32, 2 ** 28), (2 ** 29 + 2 ** 28, 8), (6 * 10 ** 8, 8), (2 ** 20, 2 ** 20)):
        for rc in (lib.nkv_linear_q8(w, sw, x, sx, None, y, m, n, 16, ws, None),
                   lib.nkv_linear_silu_mul_q8(w, sw, x, sx, y, m, n, 16, ws, None)):
            assert rc == _lib.NKV_ERR_ARG and b"too large for a launch" in lib.nkv_last_error(), (m, n)
    for m, n in ((2, 2 ** 28), (8, 2 ** 29)):
        for rc in (lib.nkv_gemv_q8(w, sw, x, None, y, m, n, 16, None),
                   lib.nkv_gemv_silu_mul_q8(w, sw, x, y, m, n, 16, None),
                   lib.nkv_norm_gemv_q8(w, sw, x, None, sx, 1e-6, None, y, None, m, n, 16, None),
                   lib.nkv_norm_gemv_silu_mul_q8(w, sw, x, None, sx, 1e-6, y, None, m, n, 16, None)):
            assert rc == _lib.NKV_ERR_ARG and b"too large for a launch" in lib.nkv_last_error(), (m, n)
    # what is refused for its size is refused before anything else is: a call that fits gets further
    assert lib.nkv_linear_q8(w + 8, sw, x, sx, None, y, 32, 2 ** 28 - 16, 16, ws, None) == _lib.NKV_ERR_ARG
    assert b"aligned" in lib.nkv_last_error()
    assert lib.nkv_gemv_q8(w + 8, sw, x, None, y, 8, 2 ** 28 - 16, 16, None) == _lib.NKV_ERR_ARG
    assert b"aligned" in lib.nkv_last_error()
    assert lib.nkv_linear_q8(w + 8, sw, x, sx, None, y, 2 ** 28, 8, 16, ws, None) == _lib.NKV_ERR_ARG
    assert b"aligned" in lib.nkv_last_error()
    assert lib.nkv_gemv_q8(w + 8, sw, x, None, y, 1, 2 ** 29, 16, None) == _lib.NKV_ERR_ARG    # resident workgroups
    assert b"aligned" in lib.nkv_last_error()


# -- the tiles of products -----------------------------------------------------------
# (m, n, gated) -> (weight rows, rows of x) of a tile: each of them, ragged on both sides
TILES = [(2079, 5395, 0, (256, 256)), (1549, 5819, 0, (192, 256)), (1287, 5409, 0, (160, 256)), (5003, 777, 0, (128, 256)),
         (327, 5517, 0, (128, 128)), (301, 6143, 0, (128, 64)), (5657, 133, 0, (128, 64)), (4495, 65, 0, (64, 64)),
         (173, 1, 0, (64, 32)), (1073, 4915, 1, (256, 256)), (649, 5513, 1, (192, 256)), (323, 5511, 1, (128, 256)),
         (143, 5453, 1, (128, 128)), (5657, 65, 1, (128, 64)), (33, 4687, 1, (64, 64)), (209, 5, 1, (64, 32))]
# the same with a k that is cut over workgroups
CUT_TILES = [(65, 3225, 11200, 0, (128, 128)), (87, 3, 11200, 0, (64, 64)), (65, 1365, 11200, 1, (128, 128)),
             (163, 5, 11200, 1, (64, 64))]


def tile_of(m, n, k, gated):
    """(weight rows, rows of x), and the workgroups that k is cut over; (0, 0), 0: the kernel of few rows."""
    t = _lib.load().nkv_linear_q8_tile(m, n, k, gated)
    return (t & 1023, t >> 10 & 1023), t >> 20


def test_every_tile_has_its_sizes():
    """What the GPU tests go over is every tile that a product takes (a table that is tuned
    anew says so here)."""
    for m, n, gated, tile in TILES:
        for k in (144, 1040):
            assert tile_of(m, n, k, gated) == tile_of(m, (n + 3) // 4 * 4, k, gated) == (tile, 1), (m, n, k, gated)
    for m, n, k, gated, tile in CUT_TILES:
        assert tile_of(m, n, k, gated)[0] == tile and tile_of(m, n, k, gated)[1] > 1, (m, n, k, gated)
    listed = ({(g, t, False) for _, _, g, t in TILES} | {(g, t, True) for _, _, _, g, t in CUT_TILES}
              | {(g, (0, 0), False) for g in (0, 1)})
    import random
    rng = random.Random(5)
    for _ in range(20000):
        m, n = round(2 ** rng.uniform(0, 13)), round(2 ** rng.uniform(0, 15))
        k, g = 16 * round(2 ** rng.uniform(0, 11)), rng.randint(0, 1)
        tile, parts = tile_of(m, n, k, g)
        assert (g, tile, parts > 1) in listed, (m, n, k, g)
    assert tile_of(0, 8, 16, 0) == tile_of(8, 0, 16, 0) == tile_of(8, 8, 0, 1) == tile_of(100, 8, 131072, 0) == ((0, 0), 0)
