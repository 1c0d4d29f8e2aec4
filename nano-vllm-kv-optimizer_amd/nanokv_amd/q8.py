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
NaN.  (Behind a norm also one whose sum of squares or largest |t * weight|, before
the root's division, passes fp32's range.)

On the GPU the operands are bf16 and the work is this library's kernels (no
fallback: the library must load); one row (a decode token) and up to 8 (a draft,
not too many channels) take their norm and quantisation inside the product's
launch.  CPU tensors take the formulas,
which the tests of the modules' routing run on.  Inference only: nothing here
has a gradient, and operands that ask for one (``requires_grad`` with gradients
enabled, or a forward-mode tangent) are refused on either.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .store import current_stream_ptr

TINY = 2.0 ** -119       # rows whose largest magnitude is below are zero
SPLIT_ROWS = 32          # products of more rows may need a workspace
TOKEN_ROW = 12288        # longest row that a product quantises in its own launch: one,
DRAFT_ROWS, DRAFT_ROW = 8, 4096          # or each of several
INT_MAX = 2 ** 31 - 1    # the library's sizes are C ints


class Q8(NamedTuple):
    """int8 codes [..., n] and their fp32 scales [...]."""
    q: torch.Tensor
    scale: torch.Tensor


# -- formulas (CPU tensors) ----------------------------------------------------
SNAP, MAGIC = 1.5 * 2.0 ** 8, 1.5 * 2.0 ** 23    # sums with them are rounded to 2^-15, to whole numbers


def _quantize_formula(y: torch.Tensor, exact: bool = True) -> Q8:
    top = y.abs().amax(dim=-1)      # (NaN where the row holds one)
    zero, odd = top < TINY, ~top.isfinite()
    none = torch.zeros_like(top)
    # the kernels' roundings, so their bits: a true division (127.0 / top is a reciprocal and a
    # product), and with `exact` y * inv to 2^-15 before whole numbers, which makes ties of bf16 exact
    inv = torch.where(zero | odd, none, torch.full_like(top, 127.0) / top)
    code = y * inv.unsqueeze(-1)
    code = ((code + SNAP) + (MAGIC - SNAP)) - MAGIC if exact else torch.round(code)
    q = torch.where(odd.unsqueeze(-1), none.unsqueeze(-1), code).to(torch.int8)
    return Q8(q, torch.where(odd, torch.full_like(top, float("nan")), torch.where(zero, none, top / 127.0)))


def _norm_formula(x, weight, eps, residual):
    t = x.float() if residual is None else x.float() + residual.float()
    mean = t.pow(2).mean(dim=-1)
    r = torch.rsqrt(mean + eps)
    codes = _quantize_formula(t * weight.float(), exact=False)      # (they do not depend on r)
    top = (t * weight.float()).abs().amax(dim=-1) * r
    zero = (codes.scale == 0) | (top < TINY)
    odd = ~(mean.isfinite() & top.isfinite())           # NaN where the squares pass fp32's range too
    scale = torch.where(zero, torch.zeros_like(top), top / 127.0)
    q = torch.where((zero | odd).unsqueeze(-1), torch.zeros_like(codes.q), codes.q)
    return (Q8(q, torch.where(odd, torch.full_like(top, float("nan")), scale)),
            x if residual is None else t.to(x.dtype))


def _product_formula(x: Q8, weight: Q8, bias=None) -> torch.Tensor:
    """fp32 [..., n]."""
    y = (x.q.double() @ weight.q.double().transpose(0, 1)).float() * x.scale.unsqueeze(-1) * weight.scale
    return y if bias is None else y + bias.float()


def _silu_mul_formula(x: Q8, weight: Q8) -> torch.Tensor:
    gate, up = _product_formula(x, weight).chunk(2, dim=-1)
    return gate / (1.0 + torch.exp(-gate)) * up


# -- operands --------------------------------------------------------------------
# A token's call is bound by the host (3 us of launch, 1 us an allocation),
# so the checks ask each tensor for little, and devices are compared as numbers.
_I8, _F32, _BF16 = torch.int8, torch.float32, torch.bfloat16
_ENTRY: dict = {}        # the library's functions by name, once it is loaded
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or current_stream_ptr
_grad_enabled = torch.is_grad_enabled
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _empty(shape, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """torch.empty, of one or two dimensions by its strides (its arguments are read in 0.7 us less)."""
    if len(shape) == 2:
        return torch.empty_strided(shape, (shape[1], 1), dtype=dtype, device=device)
    if len(shape) == 1:
        return torch.empty_strided(shape, (1,), dtype=dtype, device=device)
    return torch.empty(shape, dtype=dtype, device=device)


def _call(name: str, device: int, *args) -> None:
    """nkv_<name>(*args, stream) on the tensors' device, which is made current for the launch."""
    fn = _ENTRY.get(name)
    if fn is None:
        fn = _ENTRY[name] = getattr(_lib.load(), "nkv_" + name)
    if device == _current_device():
        rc = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(device))
    if rc:
        _lib.check(rc, name)


def _no_gradients(who: str, *operands) -> None:
    asks = False
    if _grad_enabled():
        for t in operands:
            if t is not None and t.requires_grad:
                asks = True
    if forward_ad._current_level >= 0:       # inside a dual_level
        asks = asks or any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in operands)
    if asks:
        raise ValueError(f"{who}: an operand asks for a gradient, and the 8-bit operators have none")


def _rows(x: torch.Tensor, who: str, what: str = "x") -> torch.Tensor:
    """x as dense bf16 rows on a 16-byte boundary (copied if it is neither)."""
    if x.dtype is not _BF16:
        raise ValueError(f"{who}: {what} must be bfloat16 on the GPU (got {x.dtype})")
    if not x.is_contiguous():
        x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _fine(t: torch.Tensor) -> bool:
    """What _rows returns as it is."""
    return t.dtype is _BF16 and t.is_contiguous() and t.data_ptr() % 16 == 0


def _vector(t: torch.Tensor, n: int, device: int, who: str, what: str) -> torch.Tensor:
    if t.dim() != 1 or t.shape[0] != n or t.get_device() != device:
        raise ValueError(f"{who}: {what} must be a [{n}] tensor on x's device (got {tuple(t.shape)} on {t.device})")
    return _rows(t, who, what) if device >= 0 else t


def _like(t: torch.Tensor, x: torch.Tensor, who: str, what: str) -> torch.Tensor:
    if t.shape != x.shape or t.get_device() != x.get_device():
        raise ValueError(f"{who}: {what} must be like x, {tuple(x.shape)} on {x.device} "
                         f"(got {tuple(t.shape)} on {t.device})")
    return _rows(t, who, what) if t.is_cuda else t


def _norm_checked(x, weight, eps, residual, who: str, what: str):
    """_norm_formula of operands that the kernels would take (none is broadcast)."""
    _vector(weight, x.shape[-1], x.get_device(), who, what)
    if residual is not None:
        _like(residual, x, who, "residual")
    return _norm_formula(x, weight, eps, residual)


def _width(x: torch.Tensor, who: str) -> int:
    n = x.shape[-1] if x.dim() else 0
    if n < 16 or n % 16:
        raise ValueError(f"{who}: the last dimension must be a positive multiple of 16 (got {n})")
    if x.numel() > INT_MAX and max(n, x.numel() // n) > INT_MAX:       # (as C ints they would wrap)
        raise ValueError(f"{who}: at most {INT_MAX} rows and elements a row (got {x.numel() // n} rows of {n})")
    return n


def _check_q8(t: Q8, who: str, what: str) -> None:
    q, scale = t
    if q.dtype is not _I8 or scale.dtype is not _F32 or q.dim() < 1 or scale.shape != q.shape[:-1]:
        raise ValueError(f"{who}: {what} must hold int8 codes [..., n] and float32 scales [...] "
                         f"(got {q.dtype} {tuple(q.shape)}, {scale.dtype} {tuple(scale.shape)})")
    if q.get_device() != scale.get_device():
        raise ValueError(f"{who}: {what}'s codes and scales must be on one device")


def _dense(t: Q8) -> Q8:
    q, scale = t
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    return Q8(q, scale if scale.is_contiguous() else scale.contiguous())


def _weight(weight: Q8, k: int, device: int, who: str, halves: bool) -> tuple:
    """(codes [n, k], scales [n], channels of y) of a weight on `device` (a number, -1: CPU), dense on the GPU."""
    q, scale = weight
    if (q.dtype is not _I8 or scale.dtype is not _F32 or q.dim() != 2 or scale.dim() != 1 or q.size(1) != k
            or scale.size(0) != q.size(0) or q.get_device() != device or scale.get_device() != device):
        raise ValueError(f"{who}: weight must hold int8 codes [n, {k}] and float32 scales [n] on x's device "
                         f"(got {q.dtype} {tuple(q.shape)} on {q.device}, {scale.dtype} {tuple(scale.shape)} on "
                         f"{scale.device})")
    n = q.size(0)
    if n > INT_MAX:
        raise ValueError(f"{who}: the weight has at most {INT_MAX} rows (got {n})")
    if halves:
        if n % 2:
            raise ValueError(f"{who}: the gate|up weight needs an even number of rows")
        n //= 2
    if device >= 0 and not (q.is_contiguous() and scale.is_contiguous() and q.data_ptr() % 16 == 0):
        q, scale = _dense(Q8(q, scale))
    return q, scale, n


def _one_launch(m: int, n: int, k: int, norm: bool) -> bool:
    """Whether m rows take their norm and quantisation inside the product's launch.

    Several rows (one or two a wavefront) are quantised again by every workgroup,
    16 channels each, while its first weights are on their way: more of that, or a
    norm with its residual, takes longer than a launch of the rows' own (us over cold weights,
    two launches / one: 2 to 4 x 4096 -> 2560 8.2 / 6.5, gate|up of 9728 for 6 rows 16.0 / 15.5,
    6 x 2560 -> 24576 17.2 / 17.9; with a norm 4 x 2560 -> 6144 9.0 / 7.9, 6 rows 9.2 / 9.4, gate|up of
    9728 for 2 rows 16.0 / 14.2, 4 rows 16.2 / 15.7, 6 rows 16.4 / 17.4).  Eagerly a launch and its
    buffer are 5 us of host time too."""
    if m == 1:
        return k <= TOKEN_ROW and n > 0
    return 0 < m <= DRAFT_ROWS and k <= DRAFT_ROW and 0 < (m + 3) // 4 * n * k <= (1 << 25 if norm else 1 << 26)


# -- operators ---------------------------------------------------------------------
def quantize_q8(x: torch.Tensor) -> Q8:
    """x [..., n] (n a multiple of 16) as int8 codes and a scale a row.

    2-D rows may lie apart (a column range of a wider matrix, on 16-byte
    boundaries) and are read in place."""
    n = _width(x, "quantize_q8")
    _no_gradients("quantize_q8", x)
    if not x.is_cuda:
        return _quantize_formula(x.float())
    stride = n
    if not _fine(x):
        x, stride = _strided(x, n, "quantize_q8")
    shape, device = x.shape, x.device
    q, scale = _empty(shape, _I8, device), _empty(shape[:-1], _F32, device)
    rows = x.numel() // n
    if rows:
        _call("quantize_q8", x.get_device(), x.data_ptr(), stride, q.data_ptr(), scale.data_ptr(), rows, n)
    return Q8(q, scale)


def _strided(x: torch.Tensor, n: int, who: str) -> tuple:
    """(x, elements from row to row): 2-D bf16 rows that lie apart stay where they are."""
    if (x.dim() == 2 and x.stride(1) == 1 and x.stride(0) > n and x.stride(0) % 8 == 0 and x.data_ptr() % 16 == 0
            and x.dtype is _BF16):
        return x, x.stride(0)
    return _rows(x, who), n


def dequantize_q8(t: Q8) -> torch.Tensor:
    """bf16(q * scale)."""
    _check_q8(t, "dequantize_q8", "t")
    n = _width(t.q, "dequantize_q8")
    _no_gradients("dequantize_q8", t.scale)
    if not t.q.is_cuda:
        return (t.q.float() * t.scale.unsqueeze(-1)).to(_BF16)
    q, scale = t
    if not (q.is_contiguous() and scale.is_contiguous() and q.data_ptr() % 16 == 0):
        q, scale = _dense(t)
    out = _empty(q.shape, _BF16, q.device)
    rows = out.numel() // n
    if rows:
        _call("dequantize_q8", out.get_device(), q.data_ptr(), scale.data_ptr(), out.data_ptr(), rows, n)
    return out


def _norm(x, weight, eps, residual, q: int, scale: int, rows: int, n: int, who: str, what: str):
    """nkv_rmsnorm_q8 of checked dense rows x into the addresses q and scale; the new residual."""
    device = x.get_device()
    if weight.get_device() != device or weight.shape != (n,) or not _fine(weight):
        weight = _vector(weight, n, device, who, what)
    if residual is None:
        if rows:
            _call("rmsnorm_q8", device, x.data_ptr(), None, weight.data_ptr(), float(eps), q, scale, None, rows, n)
        return x
    if residual.get_device() != device or residual.shape != x.shape or not _fine(residual):
        residual = _like(residual, x, who, "residual")
    res_out = torch.empty_like(x)
    if rows:
        _call("rmsnorm_q8", device, x.data_ptr(), residual.data_ptr(), weight.data_ptr(), float(eps), q, scale,
              res_out.data_ptr(), rows, n)
    return res_out


def rmsnorm_q8(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None = None):
    """RMSNorm of x (+ residual) over the last dim, held in 8 bits: (Q8, the new
    residual bf16(x + residual), or x itself without one)."""
    n = _width(x, "rmsnorm_q8")
    _no_gradients("rmsnorm_q8", x, weight, residual)
    if not x.is_cuda:
        return _norm_checked(x, weight, eps, residual, "rmsnorm_q8", "weight")
    if not _fine(x):
        x = _rows(x, "rmsnorm_q8")
    shape, device = x.shape, x.device
    q, scale = _empty(shape, _I8, device), _empty(shape[:-1], _F32, device)
    res_out = _norm(x, weight, eps, residual, q.data_ptr(), scale.data_ptr(), x.numel() // n, n, "rmsnorm_q8", "weight")
    return Q8(q, scale), res_out


def _product(q: int, scale: int, shape, device: torch.device, m: int, k: int, weight: tuple, bias, silu_mul: bool):
    """The product of m > 0 rows of codes at the addresses q and scale; y [*shape[:-1], n]."""
    wq, ws, n = weight
    y = _empty((*shape[:-1], n), _BF16, device)
    if n:
        b = () if silu_mul else (bias.data_ptr() if bias is not None else None,)
        device = y.get_device()
        sums = None              # of a k that is cut over workgroups (dropped behind the launch: the stream orders its reuse)
        if m > SPLIT_ROWS:
            need = _workspace(device, m, n, k, silu_mul)
            if need:
                sums = torch.empty(need, dtype=torch.int32, device=y.device)
        _call("linear_silu_mul_q8" if silu_mul else "linear_q8", device, wq.data_ptr(), ws.data_ptr(), q, scale,
              *b, y.data_ptr(), m, n, k, sums.data_ptr() if sums is not None else None)
    return y


def _workspace(device: int, m: int, n: int, k: int, silu_mul: bool) -> int:
    fn = _ENTRY.get("workspace")
    if fn is None:
        fn = _ENTRY["workspace"] = _lib.load().nkv_linear_q8_workspace
    if device == _current_device():
        return fn(m, n, k, silu_mul)
    with torch.cuda.device(device):
        return fn(m, n, k, silu_mul)


def _linear(x, weight: Q8, bias, silu_mul: bool, who: str) -> torch.Tensor:
    held = isinstance(x, Q8)
    if held:
        _check_q8(x, who, "x")
    q = x.q if held else x
    k = _width(q, who)
    _no_gradients(who, x.scale if held else x, weight[1], bias)
    device = q.get_device()
    w = _weight(weight, k, device, who, silu_mul)
    n = w[2]
    if bias is not None:
        bias = _vector(bias, n, device, who, "bias")
    if device < 0:
        t = x if held else quantize_q8(x)
        y = _silu_mul_formula(t, weight) if silu_mul else _product_formula(t, weight, bias)
        return y.to(_BF16 if held else x.dtype)
    m = q.numel() // k
    if held:
        x = _dense(x)
        if m:
            return _product(x.q.data_ptr(), x.scale.data_ptr(), q.shape, q.device, m, k, w, bias, silu_mul)
    elif _one_launch(m, n, k, False):
        if not _fine(x):
            x = _rows(x, who)
        y = _empty((*x.shape[:-1], n), _BF16, x.device)
        if silu_mul:
            _call("gemv_silu_mul_q8", device, w[0].data_ptr(), w[1].data_ptr(), x.data_ptr(), y.data_ptr(), m, n, k)
        else:
            _call("gemv_q8", device, w[0].data_ptr(), w[1].data_ptr(), x.data_ptr(),
                  bias.data_ptr() if bias is not None else None, y.data_ptr(), m, n, k)
        return y
    else:
        stride = k
        if not _fine(x):
            x, stride = _strided(x, k, who)
        if m:
            codes = torch.empty(m * (k + 4), dtype=_I8, device=x.device)    # the codes, then their scales
            at = codes.data_ptr()
            _call("quantize_q8", device, x.data_ptr(), stride, at, at + m * k, m, k)
            return _product(at, at + m * k, x.shape, x.device, m, k, w, bias, silu_mul)
    return torch.empty((*q.shape[:-1], n), dtype=_BF16, device=q.device)


def linear_q8(x, weight: Q8, bias: torch.Tensor | None = None) -> torch.Tensor:
    """x [..., k] . weight [n, k]^T (+ bias [n]): x is a Q8 or is quantised first."""
    return _linear(x, weight, bias, False, "linear_q8")


def linear_silu_mul_q8(x, gate_up_weight: Q8) -> torch.Tensor:
    """SiLU(gate) * up of x's product with gate_up_weight [2 I, k] (gate rows, then
    up rows), in fp32 and rounded once: [..., I]."""
    return _linear(x, gate_up_weight, None, True, "linear_silu_mul_q8")


def _norm_linear(x, norm_weight, eps, weight: Q8, residual, bias, silu_mul: bool, who: str):
    k = _width(x, who)
    _no_gradients(who, x, norm_weight, weight[1], residual, bias)
    device = x.get_device()
    w = _weight(weight, k, device, who, silu_mul)
    n = w[2]
    if bias is not None:
        bias = _vector(bias, n, device, who, "bias")
    if device < 0:
        t, res_out = _norm_checked(x, norm_weight, eps, residual, who, "norm_weight")
        y = _silu_mul_formula(t, weight) if silu_mul else _product_formula(t, weight, bias)
        return y.to(x.dtype), res_out
    x = _rows(x, who)
    m = x.numel() // k
    if not _one_launch(m, n, k, True):
        codes = torch.empty(m * (k + 4), dtype=_I8, device=x.device)        # the codes, then their scales
        at = codes.data_ptr()
        res_out = _norm(x, norm_weight, eps, residual, at, at + m * k, m, k, who, "norm_weight")
        if m == 0:
            return torch.empty((*x.shape[:-1], n), dtype=_BF16, device=x.device), res_out
        return _product(at, at + m * k, x.shape, x.device, m, k, w, bias, silu_mul), res_out
    norm_weight = _vector(norm_weight, k, device, who, "norm_weight")
    res_out = x
    has = residual is not None
    if has:
        residual = _like(residual, x, who, "residual")
        res_out = torch.empty_like(x)
    y = _empty((*x.shape[:-1], n), _BF16, x.device)
    b = () if silu_mul else (bias.data_ptr() if bias is not None else None,)
    _call("norm_gemv_silu_mul_q8" if silu_mul else "norm_gemv_q8", device, w[0].data_ptr(), w[1].data_ptr(),
          x.data_ptr(), residual.data_ptr() if has else None, norm_weight.data_ptr(), float(eps), *b, y.data_ptr(),
          res_out.data_ptr() if has else None, m, n, k)
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
