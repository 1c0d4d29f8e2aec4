"""8-bit rows and products without a GPU: the formulas on CPU tensors against
their definition, and what the C entry points refuse before any device work."""

import ctypes

import pytest
import torch

from nanokv_amd import _lib
from nanokv_amd.q8 import (Q8, dequantize_q8, linear_q8, linear_silu_mul_q8, norm_linear_q8, norm_linear_silu_mul_q8,
                           quantize_q8, rmsnorm_q8)


def _rows(m, k, seed):
    return torch.randn(m, k, generator=torch.Generator().manual_seed(seed)).bfloat16()


def test_quantize_by_hand():
    x = torch.zeros(5, 16)
    x[0, :4] = torch.tensor([127.0, -127.0, 0.5, 1.5])      # ties go to the even code
    x[1, 3] = -2.0
    x[2, 0] = 2.0 ** -120
    x[3, 5] = float("inf")
    x[4, 5], x[4, 6] = float("nan"), float("inf")
    t = quantize_q8(x)
    assert t.q[0, :4].tolist() == [127, -127, 0, 2] and float(t.scale[0]) == 1.0
    assert int(t.q[1, 3]) == -127 and float(t.scale[1]) == torch.tensor(2.0).div(127).item()
    assert t.scale[2] == 0 and not t.q[2].any()
    assert bool(t.scale[3:].isnan().all()) and not t.q[3:].any()
    back = dequantize_q8(t)
    assert bool(back[3:].isnan().all()) and not back[2].any() and float(back[1, 3]) == -2.0


def test_products_by_their_definition():
    x, wide = _rows(3, 32, 1), _rows(10, 32, 2)
    w = quantize_q8(wide)
    t = quantize_q8(x)
    ref = (t.q.double() * t.scale.double()[:, None]) @ (w.q.double() * w.scale.double()[:, None]).T
    bias = _rows(1, 10, 3)[0]
    for rows in (x, t):
        for got, want in ((linear_q8(rows, w), ref), (linear_q8(rows, w, bias), ref + bias.double())):
            assert got.dtype == torch.bfloat16
            assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * (1 + want.abs())).all())
        gate, up = ref.chunk(2, dim=-1)
        want = gate * torch.sigmoid(gate) * up
        got = linear_silu_mul_q8(rows, w)
        assert bool(((got.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -14) * want.abs() + 1e-30).all())


def test_norm_by_its_definition():
    x, r, wn = _rows(4, 48, 1), _rows(4, 48, 2), _rows(1, 48, 3)[0]
    w = quantize_q8(_rows(6, 48, 4))
    for res in (None, r):
        t, out = rmsnorm_q8(x, wn, 1e-6, res)
        s = x.double() if res is None else x.double() + r.double()
        y = s / (s.square().mean(-1, keepdim=True) + 1e-6).sqrt() * wn.double()
        assert float((t.q.double() * t.scale.double()[:, None] - y).abs().div(t.scale.double()[:, None]).max()) <= 0.5 + 2.0 ** -12
        assert out is x if res is None else torch.equal(out, (x.float() + r.float()).bfloat16())
        got = norm_linear_q8(x, wn, 1e-6, w, res)
        assert torch.equal(got[0], linear_q8(t, w)) and torch.equal(got[1], out)
        assert torch.equal(norm_linear_silu_mul_q8(x, wn, 1e-6, w, res)[0], linear_silu_mul_q8(t, w))


def test_norm_of_rows_without_a_finite_peak():
    x = torch.ones(5, 32)
    x[0] = 0
    x[1, 3] = float("nan")
    x[2, 4] = -float("inf")
    x[3] = 2.0 ** 70                  # its squares pass fp32's range
    x[4] = 2.0 ** -121
    t, _ = rmsnorm_q8(x, torch.ones(32), 1e-6)
    assert (t.scale[[0, 4]] == 0).all() and t.scale[1:4].isnan().all() and not t.q.any()


def test_shapes_and_refusals():
    x, w = _rows(6, 32, 1), quantize_q8(_rows(8, 32, 2))
    assert linear_q8(x.view(2, 3, 32), w).shape == (2, 3, 8) and linear_q8(x[0], w).shape == (8,)
    assert quantize_q8(x.view(2, 3, 32)).scale.shape == (2, 3)
    assert linear_q8(x[:0], w).shape == (0, 8)
    for bad in (x[:, :8], x[:, :0], torch.tensor(1.0)):
        with pytest.raises(ValueError):
            quantize_q8(bad)
    for bad in (Q8(w.q, w.scale[:3]), Q8(w.q.float(), w.scale), Q8(w.q, w.scale.double()), Q8(w.q[:, :16], w.scale)):
        with pytest.raises(ValueError):
            linear_q8(x, bad)
    with pytest.raises(ValueError, match="even"):
        linear_silu_mul_q8(x, Q8(w.q[:3], w.scale[:3]))
    with pytest.raises(ValueError):
        dequantize_q8(Q8(w.q, w.scale[:2]))


# -- the C entry points (addresses are never dereferenced) ------------------------
AT = {"w": 1 << 24, "sw": 1 << 25, "x": 4096, "sx": 1 << 26, "res": 1 << 16, "nw": 1 << 17, "b": 1 << 18, "y": 1 << 27,
      "ro": 1 << 28, "q": 1 << 29, "s": 1 << 30, "ws": 1 << 34}


def _p(**moved):
    return {k: ctypes.c_void_p(v) for k, v in {**AT, **moved}.items()}


def _product(name, m=8, n=64, k=128, **moved):
    p, lib = _p(**moved), _lib.load()
    if name == "nkv_linear_q8":
        return lib.nkv_linear_q8(p["w"], p["sw"], p["x"], p["sx"], p["b"], p["y"], m, n, k, p["ws"], None)
    return lib.nkv_linear_silu_mul_q8(p["w"], p["sw"], p["x"], p["sx"], p["y"], m, n, k, p["ws"], None)


def _token(name, m=1, n=64, k=128, **moved):
    p, lib = _p(**moved), _lib.load()
    if name == "nkv_gemv_q8":
        return lib.nkv_gemv_q8(p["w"], p["sw"], p["x"], p["b"], p["y"], m, n, k, None)
    if name == "nkv_gemv_silu_mul_q8":
        return lib.nkv_gemv_silu_mul_q8(p["w"], p["sw"], p["x"], p["y"], m, n, k, None)
    if name == "nkv_norm_gemv_q8":
        return lib.nkv_norm_gemv_q8(p["w"], p["sw"], p["x"], p["res"], p["nw"], 1e-6, p["b"], p["y"], p["ro"], m, n, k, None)
    return lib.nkv_norm_gemv_silu_mul_q8(p["w"], p["sw"], p["x"], p["res"], p["nw"], 1e-6, p["y"], p["ro"], m, n, k, None)


@pytest.mark.parametrize("name", ["nkv_linear_q8", "nkv_linear_silu_mul_q8"])
def test_products_refuse_bad_arguments(name):
    for bad in (dict(m=0), dict(n=0), dict(k=0), dict(k=8), dict(k=24), dict(k=131072), dict(n=2 ** 31 - 1), dict(w=8),
                dict(x=4100), dict(w=0), dict(sw=0), dict(x=0), dict(sx=0), dict(y=0)):
        assert _product(name, **bad) == _lib.NKV_ERR_ARG, bad
    out = 2 * 8 * 64
    lib = _lib.load()
    for bad in (dict(ws=0), dict(ws=AT["ws"] + 4), dict(ws=AT["y"] - 64), dict(ws=AT["w"]), dict(ws=AT["x"] + 512)):
        size = dict(m=70, n=256, k=9728)
        if lib.nkv_linear_q8_workspace(70, 256, 9728, name != "nkv_linear_q8"):
            assert _product(name, **size, **bad) == _lib.NKV_ERR_ARG, bad
            assert b"workspace" in lib.nkv_last_error()
    for what, size in (("w", 64 * 128), ("sw", 4 * 64), ("x", 8 * 128), ("sx", 4 * 8)):
        for where in (AT[what], AT[what] + size - 2, AT[what] - out + 2):
            assert _product(name, y=where) == _lib.NKV_ERR_ARG and b"overlap" in _lib.load().nkv_last_error()


@pytest.mark.parametrize("name", ["nkv_gemv_q8", "nkv_gemv_silu_mul_q8", "nkv_norm_gemv_q8", "nkv_norm_gemv_silu_mul_q8"])
def test_token_products_refuse_bad_arguments(name):
    norm = "norm" in name
    for bad in [dict(n=0), dict(k=0), dict(k=24), dict(k=12304), dict(n=2 ** 31 - 1), dict(w=8),
                dict(x=4104), dict(w=0), dict(sw=0), dict(x=0), dict(y=0)] + norm * [dict(nw=0), dict(nw=8), dict(res=24),
                                                                                     dict(ro=8)]:
        assert _token(name, **bad) == _lib.NKV_ERR_ARG, bad
    for bad in (dict(m=0), dict(m=-1), dict(m=9), dict(m=2, k=4112), dict(m=8, k=12288)):
        assert _token(name, **bad) == _lib.NKV_ERR_ARG, bad
    for out, where in [("y", AT["x"] + 2 * 8 * 128 - 16)] + norm * [("ro", AT["res"] - 2 * 8 * 128 + 16), ("y", AT["ro"] + 2 * 7 * 128)]:
        assert _token(name, m=8, **{out: where}) == _lib.NKV_ERR_ARG and b"overlap" in _lib.load().nkv_last_error()
    row = 2 * 128
    for out, size in [("y", 2 * 64)] + norm * [("ro", row)]:
        for what, length in [("w", 64 * 128), ("sw", 4 * 64), ("x", row)] + norm * [("res", row), ("nw", 256)]:
            for where in (AT[what], AT[what] + length - 16, AT[what] - size + 16):
                assert _token(name, **{out: where}) == _lib.NKV_ERR_ARG and b"overlap" in _lib.load().nkv_last_error()
    if norm:
        assert _token(name, y=AT["ro"] + 16) == _lib.NKV_ERR_ARG


def test_workspace_sizes():
    need = _lib.load().nkv_linear_q8_workspace
    assert need(1, 2560, 9728, 0) == need(32, 2560, 9728, 1) == 0          # few rows: cut inside a workgroup
    assert need(4096, 2560, 4096, 0) == need(1000, 6144, 2560, 0) == 0     # tiles enough
    parts, rest = divmod(need(70, 130, 9728, 1), 70 * 2 * 130)
    assert parts >= 2 and rest == 0
    assert need(0, 8, 16, 0) == need(8, 0, 16, 0) == need(8, 8, 0, 0) == need(-1, -1, -1, 1) == 0
    top = 2**31 - 1                                                        # what the products refuse needs none
    assert need(top, 8, 16, 0) == need(8, top, 16, 1) == need(70, 130, top, 0) == need(top, top, top, 1) == 0


def test_rows_refuse_bad_arguments():
    lib = _lib.load()

    def quantize(rows=4, n=64, stride=64, **moved):
        p = _p(**moved)
        return lib.nkv_quantize_q8(p["x"], stride, p["q"], p["s"], rows, n, None)

    def norm(rows=4, n=64, **moved):
        p = _p(**moved)
        return lib.nkv_rmsnorm_q8(p["x"], p["res"], p["nw"], 1e-6, p["q"], p["s"], p["ro"], rows, n, None)

    def back(rows=4, n=64, **moved):
        p = _p(**moved)
        return lib.nkv_dequantize_q8(p["q"], p["s"], p["y"], rows, n, None)

    for fn in (quantize, norm, back):
        for bad in (dict(rows=0), dict(rows=-1), dict(n=0), dict(n=8), dict(n=72), dict(q=8), dict(q=0), dict(s=0)):
            assert fn(**bad) == _lib.NKV_ERR_ARG, (fn.__name__, bad)
    assert back(rows=2**31 - 1, n=64) == _lib.NKV_ERR_ARG
    for bad in (dict(n=32784, stride=32784), dict(x=0), dict(x=4104), dict(stride=56), dict(stride=68), dict(q=AT["x"] + 16),
                dict(s=AT["x"] + 16), dict(s=AT["q"] + 16), dict(q=AT["x"] + 2 * (3 * 128 + 64) - 16, stride=128)):
        assert quantize(**bad) == _lib.NKV_ERR_ARG, bad
    for bad in (dict(n=32784), dict(x=0), dict(x=8), dict(nw=0), dict(nw=8), dict(res=8), dict(ro=8), dict(q=AT["x"] + 16),
                dict(ro=AT["x"] + 16), dict(ro=AT["res"] - 16), dict(ro=AT["nw"]), dict(ro=AT["q"]), dict(s=AT["res"]),
                dict(s=AT["nw"])):
        assert norm(**bad) == _lib.NKV_ERR_ARG, bad
    for bad in (dict(y=0), dict(y=8), dict(y=AT["q"]), dict(y=AT["s"])):
        assert back(**bad) == _lib.NKV_ERR_ARG, bad
