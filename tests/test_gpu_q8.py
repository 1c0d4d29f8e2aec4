"""8-bit rows and products (nanokv_amd.q8) against their definition in 64 bits.

Tolerances, with u = 2^-24 the half step of fp32:
* a row's scale is one division: off by u relative; its codes are the nearest
  integer of y * inv, inv and the product off by u relative each, so within 1/2 + 2 * 127 u < 1/2 + 2^-16
  of y * 127 / a.
* behind a norm, t = x + r and t * w are rounded once each: codes within
  1/2 + 127 * 4 u + ... < 1/2 + 2^-14; the sum of n <= 32768 squares is a chain of
  at most 32 adds a thread and 11 levels of joining, so the scale is off by
  less than (32 + 11) u / 2 + 6 u < 2^-18 relative.
* a product's integers are exact; it is scaled in fp32 (conversion and two
  products: 3 u) and rounded to bf16 (2^-8): 2^-8 |ref| + 2^-21 (|product| + |bias|).
* SiLU's exponent argument is off by at most 4 u |g|, so its relative error is
  below 8 u |g| + 2^-20: for |g| < 500, below 2^-11.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _hidden(m, k, seed, scale=1.0):
    g = _gen(seed)
    ch = torch.randn(k, generator=g, device="cuda").mul(0.7).exp()
    return (torch.randn(m, k, generator=g, device="cuda") * ch * scale).bfloat16()


def _codes(*shape, seed, lo=-127, hi=128):
    from nanokv_amd.q8 import Q8
    g = _gen(seed)
    q = torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int8)
    return Q8(q, torch.rand(shape[:-1], generator=g, device="cuda") * 1e-2 + 1e-4)


def _check_codes(t, y, slack):
    """codes and scales of rows y (64 bits)."""
    top = y.abs().amax(-1)
    assert bool(((t.scale.double() - top / 127).abs() <= 2.0 ** -18 * top / 127).all())
    live = top > 0
    err = (t.q.double()[live] - y[live] * (127 / top[live]).unsqueeze(-1)).abs()
    assert err.numel() == 0 or float(err.max()) <= 0.5 + slack
    assert int(t.q.int().abs().max()) <= 127
    assert bool((t.q[~live] == 0).all()) and bool((t.scale[~live] == 0).all())


def _ref_product(x, w, bias=None):
    """(ref, magnitude of its terms) in 64 bits; integers below 2^53 are exact."""
    p = (x.q.double() @ w.q.double().T) * x.scale.double().unsqueeze(-1) * w.scale.double()
    if bias is None:
        return p, p.abs()
    return p + bias.double(), p.abs() + bias.double().abs()


def _check_product(y, x, w, bias=None, extra=0.0):
    ref, mag = _ref_product(x, w, bias)
    assert y.dtype == torch.bfloat16 and y.shape == ref.shape
    err = (y.double() - ref).abs()
    assert bool((err <= 2.0 ** -8 * ref.abs() + (2.0 ** -21 + extra) * mag + 1e-37).all()), \
        f"worst {float((err / (mag + 1e-37)).max()):.3e}"


def _check_gated(y, x, w, extra=0.0):
    gate, up = _ref_product(x, w)[0].chunk(2, dim=-1)
    assert float(gate.abs().max()) < 500
    ref = gate * torch.sigmoid(gate) * up
    assert y.dtype == torch.bfloat16 and y.shape == ref.shape
    err = (y.double() - ref).abs()
    assert bool((err <= (2.0 ** -8 + 2.0 ** -11 + extra) * ref.abs() + 1e-36).all())


# -- rows ------------------------------------------------------------------------
@pytest.mark.parametrize("rows,n", [(1, 16), (3, 32), (2, 512), (5, 528), (1, 2560), (257, 2560), (7, 8192), (3, 8208),
                                    (1, 9728), (1030, 9728), (2, 32768), (4099, 128), (1025, 1008), (1024, 2048),
                                    (1500, 2544), (1100, 4096), (2, 12288), (2, 16384), (3, 1024), (3, 4080)])
def test_quantize_and_read_back(rows, n):
    from nanokv_amd.q8 import dequantize_q8, quantize_q8
    x = _hidden(rows, n, rows + n)
    x[rows // 2, : n // 2] = 0
    t = quantize_q8(x)
    assert t.q.dtype == torch.int8 and t.q.shape == x.shape and t.scale.shape == (rows,)
    _check_codes(t, x.double(), 2.0 ** -16)
    back = dequantize_q8(t)
    assert back.dtype == torch.bfloat16
    ref = t.q.double() * t.scale.double().unsqueeze(-1)
    assert bool(((back.double() - ref).abs() <= (2.0 ** -8 + 2.0 ** -22) * ref.abs()).all())


@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("rows,n", [(1, 16), (3, 48), (2, 512), (5, 528), (1, 2560), (300, 2560), (7, 8192), (3, 8208),
                                    (2, 32768), (4099, 128), (1025, 1008), (1024, 2048), (1500, 2544), (1100, 4096),
                                    (2, 12288), (2, 16384), (3, 1024), (3, 4080)])
def test_rmsnorm(rows, n, with_residual):
    from nanokv_amd.q8 import rmsnorm_q8
    x, w = _hidden(rows, n, rows + n), (1 + 0.2 * torch.randn(n, generator=_gen(n), device="cuda")).bfloat16()
    res = _hidden(rows, n, 9 * n, 2.0) if with_residual else None
    t, out = rmsnorm_q8(x, w, 1e-6, res)
    s = x.double() if res is None else x.double() + res.double()
    if res is None:
        assert out is x
    else:
        assert torch.equal(out, (x.float() + res.float()).bfloat16())
    _check_codes(t, s * torch.rsqrt(s.square().mean(-1, keepdim=True) + 1e-6) * w.double(), 2.0 ** -14)


def _odd_rows(n):
    """(rows, which are NaN, which are zero)"""
    x = _hidden(9, n, n)
    x[0] = 0
    x[1, n // 2] = float("nan")
    x[2, n - 1] = float("inf")
    x[3, 0] = -float("inf")
    x[4] = 1e-38                                  # below the smallest row that is kept
    x[5] = torch.where(x[5] > 0, 2.0, -2.0).bfloat16()   # every code at its largest
    x[6] = 0
    x[6, n - 1] = -3.0
    x[7] = x[7] * 1e30
    x[8, 1], x[8, 2] = float("nan"), float("inf")
    return x, [1, 2, 3, 8], [0, 4]


@pytest.mark.parametrize("n", [16, 2560, 9728])
def test_rows_without_a_finite_peak(n):
    from nanokv_amd.q8 import dequantize_q8, linear_q8, quantize_q8
    x, nan, zero = _odd_rows(n)
    t = quantize_q8(x)
    fine = [i for i in range(9) if i not in nan + zero]
    assert bool(t.scale[nan].isnan().all()) and bool((t.q[nan] == 0).all())
    assert bool((t.scale[zero] == 0).all()) and bool((t.q[zero] == 0).all())
    _check_codes(type(t)(t.q[fine], t.scale[fine]), x[fine].double(), 2.0 ** -16)
    assert bool((t.q[5].abs() == 127).all()) and int(t.q[6, n - 1]) == -127
    assert bool(dequantize_q8(t)[nan].isnan().all())
    w = _codes(5, n, seed=1)
    for rows in (x, t):                           # 9 rows, and the rows one by one below
        y = linear_q8(rows, w)
        assert bool(y[nan].isnan().all()) and bool((y[zero] == 0).all()) and bool(y[fine].isfinite().all())
    for i in range(9):
        y = linear_q8(x[i:i + 1], w)
        assert bool(y.isnan().all()) if i in nan else bool(y.isfinite().all())
        assert i not in zero or bool((y == 0).all())
    for i in (0, 1, 5):                           # drafts of 8 and of 4
        part = x[i:i + 8] if i < 2 else x[i:]
        assert torch.equal(linear_q8(part, w).nan_to_num(7.0), linear_q8(t, w)[i:i + part.shape[0]].nan_to_num(7.0))


@pytest.mark.parametrize("rows", [1, 4, 8, 9])
def test_norm_of_rows_without_a_finite_peak(rows):
    from nanokv_amd.q8 import norm_linear_q8, rmsnorm_q8
    x, nan, zero = _odd_rows(2560)
    nan = nan + [7]                               # its squares pass fp32's range
    wn = torch.ones(2560, device="cuda", dtype=torch.bfloat16)
    w = _codes(5, 2560, seed=1)
    for i in range(0, 9, rows):
        part = list(range(i, min(9, i + rows)))
        t, _ = rmsnorm_q8(x[part], wn, 1e-6)
        y, _ = norm_linear_q8(x[part], wn, 1e-6, w)
        for j, row in enumerate(part):
            assert bool(t.scale[j].isnan()) == (row in nan) and bool((t.scale[j] == 0)) == (row in zero)
            assert bool(y[j].isnan().all()) if row in nan else bool(y[j].isfinite().all())
            assert row not in nan + zero or bool((t.q[j] == 0).all())


@pytest.mark.parametrize("rows,n", [(5, 256), (3, 2560), (2, 9728)])
def test_residual_out_may_be_an_input(rows, n):
    import ctypes

    from nanokv_amd import _lib
    from nanokv_amd.q8 import rmsnorm_q8
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    wn = (1 + 0.2 * torch.randn(n, generator=_gen(n), device="cuda")).bfloat16()
    x, res = _hidden(rows, n, 1), _hidden(rows, n, 2)
    want, out = rmsnorm_q8(x, wn, 1e-6, res)
    for into in (0, 1):
        ins = [x.clone(), res.clone()]
        q, s = torch.empty_like(want.q), torch.empty_like(want.scale)
        _lib.check(_lib.load().nkv_rmsnorm_q8(p(ins[0]), p(ins[1]), p(wn), 1e-6, p(q), p(s), p(ins[into]), rows, n,
                                              torch.cuda.current_stream().cuda_stream), "rmsnorm_q8")
        assert torch.equal(q, want.q) and torch.equal(s, want.scale) and torch.equal(ins[into], out)


def test_an_output_off_its_eight_bytes():
    """y two bytes into an allocation: the wide stores are not taken."""
    import ctypes

    from nanokv_amd import _lib
    lib = _lib.load()
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    for m, n, k in ((1, 64, 64), (20, 64, 64), (300, 640, 128), (70, 256, 9728)):
        x, w = _codes(m, k, seed=m), _codes(n, k, seed=n)
        ws = torch.empty(max(4, lib.nkv_linear_q8_workspace(m, n, k, 0)), dtype=torch.int32, device="cuda")
        y = torch.empty(m * n + 1, dtype=torch.bfloat16, device="cuda")[1:]
        assert lib.nkv_linear_q8(p(w.q), p(w.scale), p(x.q), p(x.scale), None, p(y), m, n, k, p(ws),
                                 torch.cuda.current_stream().cuda_stream) == 0
        _check_product(y.view(m, n), x, w)


def test_strided_and_unaligned_rows():
    from nanokv_amd.q8 import linear_q8, quantize_q8, rmsnorm_q8
    wide = _hidden(33, 1024, 3)
    w = _codes(40, 256, seed=2)
    wn = torch.ones(256, device="cuda", dtype=torch.bfloat16)
    for lo in (0, 8, 16, 3):                      # 16-byte boundaries and not
        x = wide[:, lo:lo + 256]
        want = quantize_q8(x.contiguous())
        for got in (quantize_q8(x), quantize_q8(x.reshape(3, 11, 256))):
            assert torch.equal(got.q.view(33, 256), want.q) and torch.equal(got.scale.view(33), want.scale)
        assert torch.equal(linear_q8(x, w), linear_q8(x.contiguous(), w))
        assert torch.equal(linear_q8(x[:3], w), linear_q8(x[:3].contiguous(), w))
        assert torch.equal(rmsnorm_q8(x, wn, 1e-6)[0].q, rmsnorm_q8(x.contiguous(), wn, 1e-6)[0].q)
    x = wide[:, :256].t().contiguous().t()        # columns first
    assert torch.equal(quantize_q8(x).q, quantize_q8(wide[:, :256].contiguous()).q)
    x = wide[:1, :256].expand(5, 256)             # the same row five times
    assert torch.equal(quantize_q8(x).q, quantize_q8(x.contiguous()).q)
    vec = wide[0, :256]
    assert quantize_q8(vec).scale.shape == () and linear_q8(vec, w).shape == (40,)
    codes = type(w)(w.q.repeat(1, 2)[:, 256:], w.scale)      # a weight that is a column range
    assert torch.equal(linear_q8(wide[:, :256], codes), linear_q8(wide[:, :256], w))


# -- products ----------------------------------------------------------------------
SHAPES = [(1, 1, 16), (1, 7, 48), (2, 33, 64), (3, 1000, 2560), (5, 17, 80), (6, 2560, 9728), (15, 100, 144),
          (16, 64, 128), (17, 65, 1040), (31, 129, 2576), (33, 96, 208), (48, 200, 512), (49, 2560, 1024), (63, 255, 272),
          (64, 256, 256), (65, 257, 4096), (100, 1, 2560), (128, 128, 128), (129, 130, 16), (200, 384, 32), (255, 511, 112),
          (257, 300, 640), (513, 6144, 384), (1000, 77, 1000 // 16 * 16), (1025, 1283, 336), (70, 130, 9728), (99, 257, 12304), (300, 101, 2064), (130, 640, 16400)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(m, n, k):
    from nanokv_amd.q8 import linear_q8
    x, w = _codes(m, k, seed=m + k, lo=-128), _codes(n, k, seed=n, lo=-128)
    y = linear_q8(x, w)
    _check_product(y, x, w)
    bias = torch.randn(n, generator=_gen(n), device="cuda").bfloat16()
    _check_product(linear_q8(x, w, bias), x, w, bias)


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gated_product(m, n, k):
    from nanokv_amd.q8 import linear_silu_mul_q8
    x, w = _codes(m, k, seed=m + k), _codes(2 * n, k, seed=n)
    x = type(x)(x.q, x.scale * (20 / k ** 0.5))      # |gate| of a few units
    y = linear_silu_mul_q8(x, w)
    _check_gated(y, x, w)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 6, 7, 8, 9, 40])
@pytest.mark.parametrize("n,k", [(1, 16), (31, 496), (17, 1024), (514, 1040), (100, 2560), (31, 2576), (2560, 4096), (7, 4112),
                                 (130, 9728), (5, 12288), (8200, 144)])
def test_bf16_rows_are_quantised_then_multiplied(m, n, k):
    """One launch or two: the same bits."""
    from nanokv_amd.q8 import linear_q8, linear_silu_mul_q8, quantize_q8
    x, w = _hidden(m, k, m + n + k), _codes(2 * n, k, seed=n)
    w = type(w)(w.q, w.scale * (10 / k ** 0.5))
    half = type(w)(w.q[:n], w.scale[:n])
    bias = torch.randn(n, generator=_gen(n), device="cuda").bfloat16()
    t = quantize_q8(x)
    assert torch.equal(linear_q8(x, half, bias), linear_q8(t, half, bias))
    assert torch.equal(linear_silu_mul_q8(x, w), linear_silu_mul_q8(t, w))
    _check_product(linear_q8(x, half), t, half)
    _check_gated(linear_silu_mul_q8(x, w), t, w)


@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 3000, 2560), (2, 31, 496), (3, 514, 1040), (4, 77, 4096),
                                   (1, 10, 12288), (5, 60, 2560), (70, 60, 528), (8, 40, 16), (2, 9728, 2560), (6, 9728, 2560),
                                   (7, 33, 2576), (8, 12300, 144), (8, 1000, 1024), (2, 16, 4112), (9, 16, 2560)])
def test_norm_then_product(m, n, k, with_residual):
    from nanokv_amd.q8 import norm_linear_q8, norm_linear_silu_mul_q8, rmsnorm_q8
    x, w = _hidden(m, k, m + n + k), _codes(2 * n, k, seed=n)
    w = type(w)(w.q, w.scale * (10 / k ** 0.5))
    half = type(w)(w.q[:n], w.scale[:n])
    wn = (1 + 0.2 * torch.randn(k, generator=_gen(k), device="cuda")).bfloat16()
    res = _hidden(m, k, 9 * k) if with_residual else None
    bias = torch.randn(n, generator=_gen(n), device="cuda").bfloat16()
    t, want = rmsnorm_q8(x, wn, 1e-6, res)
    # the codes do not depend on the sum of squares, and the scale by 2^-18
    y, got = norm_linear_q8(x, wn, 1e-6, half, res, bias)
    assert torch.equal(got, want)
    _check_product(y, t, half, bias, 2.0 ** -18)
    y, got = norm_linear_silu_mul_q8(x, wn, 1e-6, w, res)
    assert torch.equal(got, want)
    _check_gated(y, t, w, 2.0 ** -9)              # |gate| < 500 times the scale's 2^-18


def test_a_cut_k_gives_the_same_bits():
    """Sums joined from several workgroups are the sums: rows of a call that is cut
    against the same rows in calls that are not."""
    from nanokv_amd import _lib
    from nanokv_amd.q8 import Q8, linear_q8, linear_silu_mul_q8
    need = _lib.load().nkv_linear_q8_workspace
    for m, n, k in ((70, 130, 9728), (99, 257, 12304), (130, 640, 16400), (47, 2560, 12304), (64, 301, 16400), (400, 640, 9744)):
        assert need(m, n, k, 0) and need(m, n, k, 1) and not need(16, n, k, 0)
        x, w = _codes(m, k, seed=m), _codes(2 * n, k, seed=n)
        x = Q8(x.q, x.scale * (20 / k ** 0.5))
        half = Q8(w.q[:n], w.scale[:n])
        bias = torch.randn(n, generator=_gen(n), device="cuda").bfloat16()
        whole, gated = linear_q8(x, half, bias), linear_silu_mul_q8(x, w)
        for i in range(0, m, 16):
            part = Q8(x.q[i:i + 16], x.scale[i:i + 16])
            assert torch.equal(whole[i:i + 16], linear_q8(part, half, bias))
            assert torch.equal(gated[i:i + 16], linear_silu_mul_q8(part, w))


def test_longest_sums_are_exact():
    from nanokv_amd.q8 import Q8, linear_q8
    for m in (1, 5, 70, 300):
        k = 131056
        x = Q8(torch.full((m, k), 127, dtype=torch.int8, device="cuda"), torch.ones(m, device="cuda"))
        w = Q8(torch.full((3, k), -128, dtype=torch.int8, device="cuda"), torch.full((3,), 2.0 ** -10, device="cuda"))
        x.q[:, 5] = 1
        w.q[1] = 1
        w.q[2, ::2] = 127
        _check_product(linear_q8(x, w), x, w)


def test_offsets_past_32_bits():
    """Weights, rows and outputs of more than 2^31 elements: the last rows count."""
    from nanokv_amd.q8 import Q8, dequantize_q8, linear_q8, linear_silu_mul_q8, quantize_q8
    k, n = 32768, 66000                            # 2.16e9 codes
    w = Q8(torch.zeros(n, k, dtype=torch.int8, device="cuda"), torch.full((n,), 1e-3, device="cuda"))
    w.q[-9:] = _codes(9, k, seed=1).q
    w.q[n // 2 - 9:n // 2] = _codes(9, k, seed=2).q
    x = _hidden(1, k, 4, 0.05)
    for rows in (x, x.expand(7, k), x.expand(70, k)):
        t = quantize_q8(rows)
        last = Q8(w.q[-9:], w.scale[-9:])
        _check_product(linear_q8(rows, w)[:, -9:], t, last)
        both = Q8(torch.cat([w.q[n // 2 - 9:n // 2], w.q[-9:]]), w.scale[:18])
        _check_gated(linear_silu_mul_q8(rows, w)[:, -9:], t, both)
    t = quantize_q8(dequantize_q8(w))              # 66000 rows of 32768
    assert torch.equal(t.q[-9:], quantize_q8(dequantize_q8(Q8(w.q[-9:], w.scale[-9:]))).q)
    small = _codes(33000, 16, seed=3)              # 66000 x 33000 outputs
    tall = Q8(w.q[:, :16].contiguous(), w.scale)
    y = linear_q8(tall, small)
    _check_product(y[-9:], Q8(tall.q[-9:], tall.scale[-9:]), small)
    x = Q8(w.q, w.scale)                           # 66000 x 32768 rows
    _check_product(linear_q8(x, Q8(w.q[-3:], w.scale[-3:]))[-9:], Q8(w.q[-9:], w.scale[-9:]), Q8(w.q[-3:], w.scale[-3:]))


def test_more_rows_than_one_launch_takes():
    from nanokv_amd.q8 import dequantize_q8, quantize_q8, rmsnorm_q8
    rows = 2**21 + 5
    x = _hidden(rows, 32, 6)
    wn = torch.ones(32, dtype=torch.bfloat16, device="cuda")
    t, (h, res) = quantize_q8(x), rmsnorm_q8(x, wn, 1e-6, x)
    wide = quantize_q8(x[:, :16])                  # rows that lie apart
    for at in (slice(0, 9), slice(2**21 - 4, rows)):
        a, (b, r) = quantize_q8(x[at].contiguous()), rmsnorm_q8(x[at].contiguous(), wn, 1e-6, x[at].contiguous())
        assert torch.equal(t.q[at], a.q) and torch.equal(t.scale[at], a.scale) and torch.equal(res[at], r)
        assert torch.equal(h.q[at], b.q) and torch.equal(h.scale[at], b.scale)
        c = quantize_q8(x[at, :16].contiguous())
        assert torch.equal(wide.q[at], c.q) and torch.equal(wide.scale[at], c.scale)
        assert torch.equal(dequantize_q8(t)[at], dequantize_q8(a))


def test_no_rows_and_no_channels():
    from nanokv_amd.q8 import (dequantize_q8, linear_q8, linear_silu_mul_q8, norm_linear_q8, quantize_q8, rmsnorm_q8)
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    wn = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    w = _codes(8, 64, seed=1)
    t = quantize_q8(x)
    assert t.q.shape == (0, 64) and t.scale.shape == (0,) and dequantize_q8(t).shape == (0, 64)
    assert rmsnorm_q8(x, wn, 1e-6, x)[1].shape == (0, 64)
    assert linear_q8(x, w).shape == (0, 8) and linear_q8(t, w).shape == (0, 8)
    assert linear_silu_mul_q8(x, w).shape == (0, 4) and norm_linear_q8(x, wn, 1e-6, w)[0].shape == (0, 8)
    none = type(w)(w.q[:0], w.scale[:0])
    assert linear_q8(_hidden(3, 64, 1), none).shape == (3, 0)
    assert norm_linear_q8(_hidden(3, 64, 1), wn, 1e-6, none)[0].shape == (3, 0)


def test_rows_behind_the_last_are_left_as_they_were():
    """Outputs of ragged sizes inside a larger buffer: nothing around them is written."""
    import ctypes

    from nanokv_amd import _lib
    lib = _lib.load()
    stream = torch.cuda.current_stream().cuda_stream
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    sums = []

    def ws(*size):
        sums.append(torch.full((lib.nkv_linear_q8_workspace(*size) + 64,), 5, dtype=torch.int32, device="cuda"))
        return p(sums[-1])

    for m, n, k in ((1, 3, 64), (5, 33, 48), (3, 17, 2560), (8, 100, 4096), (37, 129, 256), (70, 65, 128), (300, 300, 144), (70, 130, 9728)):
        x, w = _codes(m, k, seed=m), _codes(2 * n, k, seed=n)
        y = torch.full((m * n + 512,), 7.0, dtype=torch.bfloat16, device="cuda")
        assert lib.nkv_linear_q8(p(w.q), p(w.scale), p(x.q), p(x.scale), None, p(y), m, n, k, ws(m, n, k, 0), stream) == 0
        assert bool((y[m * n:] == 7).all())
        y.fill_(7.0)
        assert lib.nkv_linear_silu_mul_q8(p(w.q), p(w.scale), p(x.q), p(x.scale), p(y), m, n, k, ws(m, n, k, 1), stream) == 0
        assert bool((y[m * n:] == 7).all())
        assert all(bool((t[-64:] == 5).all()) for t in sums)
        q = torch.full((m * k + 512,), 9, dtype=torch.int8, device="cuda")
        s = torch.full((m + 64,), 9.0, device="cuda")
        assert lib.nkv_quantize_q8(p(_hidden(m, k, 1)), k, p(q), p(s), m, k, stream) == 0
        assert bool((q[m * k:] == 9).all()) and bool((s[m:] == 9).all())
        if m <= 8:
            y.fill_(7.0)
            assert lib.nkv_gemv_q8(p(w.q), p(w.scale), p(_hidden(m, k, 1)), None, p(y), m, n, k, stream) == 0
            assert bool((y[m * n:] == 7).all()) and bool((y[:m * n] != 7).any())
            y.fill_(7.0)
            ro = torch.full((m * k + 512,), 9.0, dtype=torch.bfloat16, device="cuda")
            rows, wn = _hidden(m, k, 1), torch.ones(k, dtype=torch.bfloat16, device="cuda")
            assert lib.nkv_norm_gemv_silu_mul_q8(p(w.q), p(w.scale), p(rows), None, p(wn), 1e-6, p(y), p(ro), m, n, k, stream) == 0
            assert bool((y[m * n:] == 7).all()) and bool((ro[m * k:] == 9).all())
            assert torch.equal(ro[:m * k].view(m, k), rows)    # without a residual: x


# -- together -----------------------------------------------------------------------
def _mlp(x, res, wn, gate_up, down):
    from nanokv_amd.q8 import linear_q8, linear_silu_mul_q8, rmsnorm_q8
    t, res = rmsnorm_q8(x, wn, 1e-6, res)
    return linear_q8(linear_silu_mul_q8(t, gate_up), down), res


# (3000 rows: tiles of more than 64 KiB of LDS; 70 rows of 9728: sums in a workspace)
@pytest.mark.parametrize("m,k,inter", [(1, 512, 1040), (6, 512, 1040), (77, 512, 1040), (300, 512, 1040), (3000, 512, 1040),
                                       (70, 512, 9728)])
def test_a_captured_mlp_replays_with_new_rows(m, k, inter):
    from nanokv_amd.q8 import norm_linear_silu_mul_q8, linear_q8
    wn = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    gate_up, down = _codes(2 * inter, k, seed=1), _codes(k, inter, seed=2)
    gate_up = type(gate_up)(gate_up.q, gate_up.scale * 0.01)
    x, res = _hidden(m, k, 1), _hidden(m, k, 2)

    def step():
        a = _mlp(x, res, wn, gate_up, down)
        h, r = norm_linear_silu_mul_q8(x, wn, 1e-6, gate_up, res)
        return a + (linear_q8(h, down), r)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        x.copy_(_hidden(m, k, 10 + i))
        res.copy_(_hidden(m, k, 20 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_on_another_stream():
    k = 512
    wn = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    gate_up, down = _codes(256, k, seed=1), _codes(k, 128, seed=2)
    want = [_mlp(_hidden(m, k, m), _hidden(m, k, 2), wn, gate_up, down) for m in (1, 9, 100)]
    side = torch.cuda.Stream()
    ins = [(_hidden(m, k, m), _hidden(m, k, 2)) for m in (1, 9, 100)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [_mlp(x, r, wn, gate_up, down) for x, r in ins]
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_refusals():
    from nanokv_amd.q8 import Q8, linear_q8, linear_silu_mul_q8, norm_linear_q8, quantize_q8, rmsnorm_q8
    x, w = _hidden(3, 64, 1), _codes(8, 64, seed=1)
    wn = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    for bad in (x.float(), x.half(), x[:, :8], x.clone().requires_grad_()):
        with pytest.raises(ValueError):
            quantize_q8(bad)
        with pytest.raises(ValueError):
            rmsnorm_q8(bad, wn[: bad.shape[1]], 1e-6)
        with pytest.raises(ValueError):
            linear_q8(bad, w)
    with pytest.raises(ValueError, match="at most|32768"):
        quantize_q8(torch.zeros(1, 32784, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError, match="131056"):
        long = _codes(2, 131072, seed=1)
        linear_q8(long, long)
    for bad in (Q8(w.q[:, :32], w.scale), Q8(w.q, w.scale[:4]), Q8(w.q.cpu(), w.scale.cpu()), Q8(w.q.int(), w.scale),
                Q8(w.q, w.scale.half())):
        for rows in (x, quantize_q8(x), x.repeat(3, 1)):
            with pytest.raises(ValueError):
                linear_q8(rows, bad)
    with pytest.raises(ValueError, match="even"):
        linear_silu_mul_q8(x, Q8(w.q[:7], w.scale[:7]))
    for bias in (torch.zeros(7, dtype=torch.bfloat16, device="cuda"), torch.zeros(8, device="cuda"), torch.zeros(8)):
        for rows in (x, x.repeat(3, 1)):
            with pytest.raises(ValueError, match="bias"):
                linear_q8(rows, w, bias)
            with pytest.raises(ValueError, match="bias"):
                norm_linear_q8(rows, wn, 1e-6, w, None, bias)
    for res in (x[:2], x.float(), x.cpu()):
        with pytest.raises(ValueError, match="residual"):
            rmsnorm_q8(x, wn, 1e-6, res)
        with pytest.raises(ValueError, match="residual"):
            norm_linear_q8(x, wn, 1e-6, w, res)
    with pytest.raises(ValueError, match="weight"):
        rmsnorm_q8(x, wn[:32], 1e-6)
