"""8-bit projections: rows and weights held as int8 codes with fp32 scales.

A row y[n] is held as q = rne(y * 127 / a) with the scale s = a / 127,
a = max |y| (``quantize_q8``; ``dequantize_q8`` reads it back), a weight
[n, k] the same way with one scale an output channel.  Products are summed
exactly in 32-bit integers and scaled by token and channel in fp32
(``linear_q8``; ``linear_silu_mul_q8`` for a gate|up weight).  ``rmsnorm_q8`` is
the RMSNorm (+ residual add) whose output is held in 8 bits; the
``norm_linear_*`` pair puts it in front of a product.

A row whose largest magnitude is below 2^-119 is zero; one that holds a NaN or
an infinity has the scale NaN and the codes 0, so what is computed from it is
NaN.

On the GPU the operands are bf16 and the work is this library's kernels (no
fallback: the library must load); one row (a decode token) takes its norm and
quantisation inside the product's launch.  CPU tensors take the formulas,
which the tests of the modules' routing run on.  Inference only: nothing here
has a gradient, and inputs that ask for one are refused.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .store import current_stream_ptr

TINY = 2.0 ** -119       # rows whose largest magnitude is below are zero
TOKEN_ROW = 12288        # longest row that a product quantises in its own launch


class Q8(NamedTuple):
    """int8 codes [..., n] and their fp32 scales [...]."""
    q: torch.Tensor
    scale: torch.Tensor


# -- formulas (CPU tensors) ----------------------------------------------------
def _quantize_formula(y: torch.Tensor) -> Q8:
    top = y.abs().amax(dim=-1)      # (NaN where the row holds one)
    zero, odd = top < TINY, ~top.isfinite()
    none = torch.zeros_like(top)
    inv = torch.where(zero | odd, none, 127.0 / top)
    q = torch.where(odd.unsqueeze(-1), none.unsqueeze(-1), torch.round(y * inv.unsqueeze(-1))).to(torch.int8)
    return Q8(q, torch.where(odd, torch.full_like(top, float("nan")), torch.where(zero, none, top / 127.0)))


def _norm_formula(x, weight, eps, residual):
    t = x.float() if residual is None else x.float() + residual.float()
    y = t * torch.rsqrt(t.pow(2).mean(dim=-1, keepdim=True) + eps) * weight.float()
    return _quantize_formula(y), x if residual is None else t.to(x.dtype)


def _product_formula(x: Q8, weight: Q8, bias=None) -> torch.Tensor:
    """fp32 [..., n]."""
    y = (x.q.double() @ weight.q.double().transpose(0, 1)).float() * x.scale.unsqueeze(-1) * weight.scale
    return y if bias is None else y + bias.float()


def _silu_mul_formula(x: Q8, weight: Q8) -> torch.Tensor:
    gate, up = _product_formula(x, weight).chunk(2, dim=-1)
    return gate / (1.0 + torch.exp(-gate)) * up


# -- operands --------------------------------------------------------------------
def _call(name: str, device: int, *args) -> None:
    """nkv_<name>(*args, stream): the tensors' device is made current for the launch."""
    fn = getattr(_lib.load(), "nkv_" + name)
    if device == torch.cuda.current_device():
        rc = fn(*args, current_stream_ptr())
    else:
        with torch.cuda.device(device):
            rc = fn(*args, current_stream_ptr())
    if rc:
        _lib.check(rc, name)


def _rows(x: torch.Tensor, who: str, what: str = "x") -> torch.Tensor:
    """x as dense bf16 rows on a 16-byte boundary (copied if it is neither)."""
    if x.dtype != torch.bfloat16:
        raise ValueError(f"{who}: {what} must be bfloat16 on the GPU (got {x.dtype})")
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{who}: {what} asks for a gradient, and the 8-bit operators have none")
    if not x.is_contiguous():
        x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _vector(t: torch.Tensor, n: int, device: torch.device, who: str, what: str) -> torch.Tensor:
    if t.dim() != 1 or t.shape[0] != n or t.device != device:
        raise ValueError(f"{who}: {what} must be a [{n}] tensor on {device} (got {tuple(t.shape)} on {t.device})")
    return _rows(t, who, what)


def _like(t: torch.Tensor, x: torch.Tensor, who: str, what: str) -> torch.Tensor:
    if t.shape != x.shape or t.device != x.device:
        raise ValueError(f"{who}: {what} must be like x, {tuple(x.shape)} on {x.device} "
                         f"(got {tuple(t.shape)} on {t.device})")
    return _rows(t, who, what)


def _check_width(n: int, who: str) -> None:
    if n < 16 or n % 16:
        raise ValueError(f"{who}: the last dimension must be a positive multiple of 16 (got {n})")


def _check_q8(t: Q8, who: str, what: str) -> None:
    q, scale = t
    if q.dtype != torch.int8 or scale.dtype != torch.float32 or q.dim() < 1 or scale.shape != q.shape[:-1]:
        raise ValueError(f"{who}: {what} must hold int8 codes [..., n] and float32 scales [...] "
                         f"(got {q.dtype} {tuple(q.shape)}, {scale.dtype} {tuple(scale.shape)})")
    if q.device != scale.device:
        raise ValueError(f"{who}: {what}'s codes and scales must be on one device")


def _dense(t: Q8) -> Q8:
    q, scale = t
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    return Q8(q, scale if scale.is_contiguous() else scale.contiguous())


def _check_weight(weight: Q8, k: int, device: torch.device, who: str, halves: bool = False) -> None:
    _check_q8(weight, who, "weight")
    q = weight.q
    if q.dim() != 2 or q.shape[1] != k or q.device != device:
        raise ValueError(f"{who}: weight must be [n, {k}] on {device} (got {tuple(q.shape)} on {q.device})")
    if halves and q.shape[0] % 2:
        raise ValueError(f"{who}: the gate|up weight needs an even number of rows")
    _check_width(k, who)


# -- operators ---------------------------------------------------------------------
def quantize_q8(x: torch.Tensor) -> Q8:
    """x [..., n] (n a multiple of 16) as int8 codes and a scale a row.

    2-D rows may lie apart (a column range of a wider matrix, on 16-byte
    boundaries) and are read in place."""
    if x.dim() < 1:
        raise ValueError("quantize_q8: x needs at least one dimension")
    n = x.shape[-1]
    _check_width(n, "quantize_q8")
    if not x.is_cuda:
        return _quantize_formula(x.float())
    stride = n
    if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) > n and x.stride(0) % 8 == 0 and x.data_ptr() % 16 == 0 \
            and x.dtype == torch.bfloat16 and not x.requires_grad:
        stride = x.stride(0)
    else:
        x = _rows(x, "quantize_q8")
    out = Q8(torch.empty(x.shape, dtype=torch.int8, device=x.device),
             torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device))
    rows = out.scale.numel()
    if rows:
        _call("quantize_q8", x.get_device(), x.data_ptr(), stride, out.q.data_ptr(), out.scale.data_ptr(), rows, n)
    return out


def dequantize_q8(t: Q8) -> torch.Tensor:
    """bf16(q * scale)."""
    _check_q8(t, "dequantize_q8", "t")
    n = t.q.shape[-1]
    _check_width(n, "dequantize_q8")
    if not t.q.is_cuda:
        return (t.q.float() * t.scale.unsqueeze(-1)).to(torch.bfloat16)
    t = _dense(t)
    out = torch.empty(t.q.shape, dtype=torch.bfloat16, device=t.q.device)
    if out.numel():
        _call("dequantize_q8", out.get_device(), t.q.data_ptr(), t.scale.data_ptr(), out.data_ptr(), t.scale.numel(), n)
    return out


def rmsnorm_q8(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None = None):
    """RMSNorm of x (+ residual) over the last dim, held in 8 bits: (Q8, the new
    residual bf16(x + residual), or x itself without one)."""
    n = x.shape[-1] if x.dim() else 0
    _check_width(n, "rmsnorm_q8")
    if not x.is_cuda:
        return _norm_formula(x, weight, eps, residual)
    x = _rows(x, "rmsnorm_q8")
    weight = _vector(weight, n, x.device, "rmsnorm_q8", "weight")
    out = Q8(torch.empty(x.shape, dtype=torch.int8, device=x.device),
             torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device))
    res_out = x
    if residual is not None:
        residual = _like(residual, x, "rmsnorm_q8", "residual")
        res_out = torch.empty_like(x)
    rows = out.scale.numel()
    if rows:
        _call("rmsnorm_q8", x.get_device(), x.data_ptr(), residual.data_ptr() if residual is not None else None,
              weight.data_ptr(), float(eps), out.q.data_ptr(), out.scale.data_ptr(),
              res_out.data_ptr() if residual is not None else None, rows, n)
    return out, res_out


def _linear(x, weight: Q8, bias, silu_mul: bool, who: str) -> torch.Tensor:
    q = x.q if isinstance(x, Q8) else x
    if isinstance(x, Q8):
        _check_q8(x, who, "x")
    if q.dim() < 1:
        raise ValueError(f"{who}: x needs at least one dimension")
    k = q.shape[-1]
    _check_weight(weight, k, q.device, who, silu_mul)
    n = weight.q.shape[0] // (2 if silu_mul else 1)
    if not q.is_cuda:
        t = x if isinstance(x, Q8) else quantize_q8(x)
        y = _silu_mul_formula(t, weight) if silu_mul else _product_formula(t, weight, bias)
        return y.to(torch.bfloat16 if isinstance(x, Q8) else x.dtype)
    weight = _dense(weight)
    if bias is not None:
        bias = _vector(bias, n, q.device, who, "bias")
    b = () if silu_mul else (bias.data_ptr() if bias is not None else None,)
    name = "linear_silu_mul_q8" if silu_mul else "linear_q8"
    y = torch.empty(*q.shape[:-1], n, dtype=torch.bfloat16, device=q.device)
    m = q.numel() // k
    if m == 0 or n == 0:
        return y
    if not isinstance(x, Q8):
        if m == 1 and k <= TOKEN_ROW:
            x = _rows(x, who)
            _call("gemv_silu_mul_q8" if silu_mul else "gemv_q8", x.get_device(), weight.q.data_ptr(),
                  weight.scale.data_ptr(), x.data_ptr(), *b, y.data_ptr(), n, k)
            return y
        x = quantize_q8(x)
    x = _dense(x)
    _call(name, y.get_device(), weight.q.data_ptr(), weight.scale.data_ptr(), x.q.data_ptr(), x.scale.data_ptr(), *b,
          y.data_ptr(), m, n, k)
    return y


def linear_q8(x, weight: Q8, bias: torch.Tensor | None = None) -> torch.Tensor:
    """x [..., k] . weight [n, k]^T (+ bias [n]): x is a Q8 or is quantised first."""
    return _linear(x, weight, bias, False, "linear_q8")


def linear_silu_mul_q8(x, gate_up_weight: Q8) -> torch.Tensor:
    """SiLU(gate) * up of x's product with gate_up_weight [2 I, k] (gate rows, then
    up rows), in fp32 and rounded once: [..., I]."""
    return _linear(x, gate_up_weight, None, True, "linear_silu_mul_q8")


def _norm_linear(x, norm_weight, eps, weight: Q8, residual, bias, silu_mul: bool, who: str):
    k = x.shape[-1] if x.dim() else 0
    _check_weight(weight, k, x.device, who, silu_mul)
    m = x.numel() // k
    if not (x.is_cuda and m == 1 and k <= TOKEN_ROW and weight.q.shape[0]):
        t, res_out = rmsnorm_q8(x, norm_weight, eps, residual)
        return _linear(t, weight, bias, silu_mul, who), res_out
    weight = _dense(weight)
    x = _rows(x, who)
    norm_weight = _vector(norm_weight, k, x.device, who, "norm_weight")
    n = weight.q.shape[0] // (2 if silu_mul else 1)
    res_out = x
    if residual is not None:
        residual = _like(residual, x, who, "residual")
        res_out = torch.empty_like(x)
    if bias is not None:
        bias = _vector(bias, n, x.device, who, "bias")
    b = () if silu_mul else (bias.data_ptr() if bias is not None else None,)
    y = torch.empty(*x.shape[:-1], n, dtype=torch.bfloat16, device=x.device)
    has = residual is not None
    _call("norm_gemv_silu_mul_q8" if silu_mul else "norm_gemv_q8", x.get_device(), weight.q.data_ptr(),
          weight.scale.data_ptr(), x.data_ptr(), residual.data_ptr() if has else None, norm_weight.data_ptr(),
          float(eps), *b, y.data_ptr(), res_out.data_ptr() if has else None, n, k)
    return y, res_out


def norm_linear_q8(x: torch.Tensor, norm_weight: torch.Tensor, eps: float, weight: Q8,
                   residual: torch.Tensor | None = None, bias: torch.Tensor | None = None):
    """linear_q8 of rmsnorm_q8(x, residual): (y, the new residual)."""
    return _norm_linear(x, norm_weight, eps, weight, residual, bias, False, "norm_linear_q8")


def norm_linear_silu_mul_q8(x: torch.Tensor, norm_weight: torch.Tensor, eps: float, gate_up_weight: Q8,
                            residual: torch.Tensor | None = None):
    """linear_silu_mul_q8 of rmsnorm_q8(x, residual): (y, the new residual)."""
    return _norm_linear(x, norm_weight, eps, gate_up_weight, residual, None, True, "norm_linear_silu_mul_q8")


__all__ = ["Q8", "dequantize_q8", "linear_q8", "linear_silu_mul_q8", "norm_linear_q8", "norm_linear_silu_mul_q8",
           "quantize_q8", "rmsnorm_q8"]
