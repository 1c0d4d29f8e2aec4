"""Dense attention over a paged cache: writing to it and reading it.

A layer's cache is a ``PagedKV``: keys and values [pages, Hkv, page, D] in bf16, or
int8 codes with an fp32 scale a row (``new_paged_kv`` makes one).  Slot s is token
s % page of page s // page; a sequence's pages are listed in its row of a page
table.

* ``qkv_append_paged``: the fused projection's rows: RMSNorm of each head of q and k
  (or none), the rotation of their positions, keys and values written to their slots,
  the queries returned, in one launch.  ``append_paged`` writes rows that are
  rotated already, ``read_paged`` reads slots back, ``move_paged`` moves rows from slots
  to slots.
* ``attend_paged``: attention of every sequence's new tokens over all of its keys:
  one token, several in order (a draft, a prompt or its next chunk), or a tree of
  drafted tokens (``tree_masks`` makes its masks from the parents).

A head's row y is held in 8 bits as rne(y * 127 / a) with the scale a / 127, a =
max |y|; one whose largest magnitude is below 2^-119 is zero, one with a NaN or an
infinity has the scale NaN.

On the GPU the operands are bf16 and the work is this library's kernels (no
fallback: the library must load), on the current stream of their device, with nothing
read back: a step of fixed sizes can be captured in a graph.  CPU tensors take the formulas.  Inference
only: operands that ask for a gradient are refused.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .q8 import _asks_gradient, _call, _current_device, _fine, _quantize_formula

_BF16, _I8, _I32, _I64, _F32 = torch.bfloat16, torch.int8, torch.int32, torch.int64, torch.float32
MAX_TREE = 64          # drafted tokens of a tree: bits of a mask


class PagedKV(NamedTuple):
    """Keys and values [pages, Hkv, page, D] (bf16, or int8 codes) and the codes' fp32
    scales [pages, Hkv, page] (finite, or NaN: as they are written here).  Other orders in memory (views) are read in place as
    long as a row's D values lie together and k and v lie alike."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor | None = None
    v_scale: torch.Tensor | None = None


def new_paged_kv(pages: int, num_kv_heads: int, page_size: int = 64, head_dim: int = 128,
                 dtype: torch.dtype = torch.bfloat16, device="cuda") -> PagedKV:
    """An empty cache of bf16 values or int8 codes."""
    if dtype not in (_BF16, _I8):
        raise ValueError(f"new_paged_kv: dtype must be torch.bfloat16 or torch.int8 (got {dtype})")
    shape = (pages, num_kv_heads, page_size, head_dim)
    cache = PagedKV(*(torch.zeros(shape, dtype=dtype, device=device) for _ in range(2)))
    if dtype is _I8:
        cache = PagedKV(cache.k, cache.v, *(torch.zeros(shape[:3], device=device) for _ in range(2)))
    _cache_args(cache, "new_paged_kv")
    return cache


def _cache_args(cache: PagedKV, who: str) -> tuple:
    """(k, v, their scales, three strides, pages, Hkv, page, D): the cache as the library takes it."""
    k, v, ks, vs = cache
    shape, strides, dtype = k.shape, k.stride(), k.dtype
    if (dtype is not _BF16 and dtype is not _I8) or v.dtype is not dtype or len(shape) != 4 or v.shape != shape:
        raise ValueError(f"{who}: the cache holds bfloat16 or int8 keys and values [pages, Hkv, page, D] "
                         f"(got {dtype} {tuple(shape)}, {v.dtype} {tuple(v.shape)})")
    device = k.get_device()
    if v.get_device() != device or v.stride() != strides or strides[3] != 1:
        raise ValueError(f"{who}: the cache's keys and values must lie alike on one device, a row's values together")
    pages, hkv, page, d = shape
    if d not in (64, 128) or not 16 <= page <= 4096 or page & (page - 1) or pages < 1 or hkv < 1:
        raise ValueError(f"{who}: heads have 64 or 128 dims and pages a power of two from 16 to 4096 tokens "
                         f"(got {tuple(shape)})")
    if dtype is _I8:
        for s in (ks, vs):
            if s is None or s.dtype is not _F32 or s.shape != shape[:3] or s.get_device() != device or not s.is_contiguous():
                raise ValueError(f"{who}: an int8 cache needs dense float32 scales {tuple(shape[:3])} on its device")
        return (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), *strides[:3], pages, hkv, page, d)
    if ks is not None or vs is not None:
        raise ValueError(f"{who}: a bfloat16 cache has no scales")
    return (k.data_ptr(), v.data_ptr(), None, None, *strides[:3], pages, hkv, page, d)


def _to_i32(t: torch.Tensor) -> torch.Tensor:
    """An int64 tensor as int32, what does not fit as the type's ends: they too lie outside every cache and table."""
    return t.clamp(-2 ** 31, 2 ** 31 - 1).to(_I32)


def _ints(t: torch.Tensor, dtype: torch.dtype, n: int | None, device: int, who: str, what: str) -> torch.Tensor:
    """t as a dense vector of dtype (converted from the other integer type)."""
    if t.dtype not in (_I32, _I64) or t.dim() != 1 or (n is not None and t.shape[0] != n) or t.get_device() != device:
        raise ValueError(f"{who}: {what} must be int32 or int64 [{'n' if n is None else n}] on the cache's device "
                         f"(got {t.dtype} {tuple(t.shape)} on {t.device})")
    if t.dtype is not dtype:
        t = _to_i32(t) if dtype is _I32 else t.to(dtype)
    return t if t.is_contiguous() else t.contiguous()


def _no_gradients(who: str, *operands) -> None:
    if _asks_gradient(*operands):
        raise ValueError(f"{who}: an operand asks for a gradient, and the paged operators have none")


def _head_rows(t: torch.Tensor, hkv: int, d: int, device: int, who: str, what: str) -> tuple:
    """(t, elements from row to row) of [T, Hkv, D] rows, read in place if each lies together."""
    if t.dim() != 3 or t.shape[1] != hkv or t.shape[2] != d or t.get_device() != device:
        raise ValueError(f"{who}: {what} must be [T, {hkv}, {d}] on the cache's device "
                         f"(got {tuple(t.shape)} on {t.device})")
    if device < 0:
        return t, t.stride(0)
    if t.dtype is not _BF16:
        raise ValueError(f"{who}: {what} must be bfloat16 on the GPU (got {t.dtype})")
    s = t.stride()
    if s[2] == 1 and (hkv == 1 or s[1] == d) and s[0] % 8 == 0 and t.data_ptr() % 16 == 0:
        return t, s[0]
    t = t.contiguous()
    return (t if t.data_ptr() % 16 == 0 else t.clone()), hkv * d


# -- formulas (CPU tensors) ----------------------------------------------------
def _store_formula(cache: PagedKV, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    """k, v [T, Hkv, D] fp32 to the slots that lie inside the cache."""
    pages, _, page, _ = cache.k.shape
    live = (slots >= 0) & (slots < pages * page)
    at = slots[live].long()
    p, o = at // page, at % page
    for held, scale, y in ((cache.k, cache.k_scale, k[live]), (cache.v, cache.v_scale, v[live])):
        if scale is None:
            held[p, :, o] = y.to(held.dtype)
        else:
            t = _quantize_formula(y, exact=False)
            ties = _quantize_formula(y)
            bf16s = (y == y.bfloat16().float()) & (y.abs().amax(-1) == y.abs().amax(-1).bfloat16().float()).unsqueeze(-1)
            held[p, :, o] = torch.where(bf16s, ties.q, t.q)
            scale[p, :, o] = t.scale


def _head_formula(x: torch.Tensor, weight, eps: float, cos, sin, interleaved: bool) -> torch.Tensor:
    """x [T, heads, D] fp32, normed and rotated."""
    if weight is not None:
        x = x * torch.rsqrt(x.pow(2).mean(dim=-1, keepdim=True) + eps) * weight.float()
    if cos is None:
        return x
    r = 2 * cos.shape[-1]
    cos, sin = cos.unsqueeze(1), sin.unsqueeze(1)
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., r:]), dim=-1)


# -- writing -------------------------------------------------------------------
def append_paged(cache: PagedKV, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Keys and values [T, Hkv, D] (rotated already) to their slots [T].

    Slots outside the cache (-1: a row of padding) store nothing; the others are
    distinct."""
    who = "append_paged"
    args = _cache_args(cache, who)
    hkv, d = args[8], args[10]
    _no_gradients(who, k, v)
    device = cache.k.get_device()
    k, k_stride = _head_rows(k, hkv, d, device, who, "k")
    v, v_stride = _head_rows(v, hkv, d, device, who, "v")
    rows = k.shape[0]
    if v.shape[0] != rows:
        raise ValueError(f"{who}: k and v must be alike (got {tuple(k.shape)}, {tuple(v.shape)})")
    slots = _ints(slots, _I32, rows, device, who, "slots")
    if device < 0:
        _store_formula(cache, slots, k.float(), v.float())
    elif rows:
        _call("paged_append", device, *args, None, 0, k.data_ptr(), k_stride, v.data_ptr(), v_stride, rows, 0,
              slots.data_ptr(), None, None, None, 0, 0, 0, None, None, 0.0, None)


def _rope_tables(cos, sin, d: int, device: int, who: str) -> tuple:
    """(cos, sin, positions of the table, rotated dims)."""
    if cos is None or sin is None:
        if cos is not None or sin is not None:
            raise ValueError(f"{who}: cos and sin come together")
        return None, None, 0, 0
    if (cos.dim() != 2 or sin.shape != cos.shape or cos.dtype is not _F32 or sin.dtype is not _F32
            or cos.get_device() != device or sin.get_device() != device or cos.shape[0] < 1
            or cos.shape[1] < 8 or cos.shape[1] % 8 or 2 * cos.shape[1] > d):
        raise ValueError(f"{who}: cos and sin must be float32 [positions, R / 2] on the cache's device, R a multiple of "
                         f"16 up to {d} (got {tuple(cos.shape)}, {tuple(sin.shape)})")
    if device >= 0:
        cos, sin = (t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
                    for t in (cos, sin))
    return cos, sin, cos.shape[0], 2 * cos.shape[1]


def _norm_weight(w, d: int, device: int, who: str, what: str):
    if w is None:
        return None
    if w.dim() != 1 or w.shape[0] != d or w.get_device() != device or (device >= 0 and w.dtype is not _BF16):
        raise ValueError(f"{who}: {what} must be a bfloat16 [{d}] tensor on the cache's device "
                         f"(got {w.dtype} {tuple(w.shape)} on {w.device})")
    return w if device < 0 or _fine(w) else w.clone(memory_format=torch.contiguous_format)


def qkv_append_paged(cache: PagedKV, qkv: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor | None,
                     cos: torch.Tensor | None, sin: torch.Tensor | None, num_heads: int, *,
                     q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6,
                     interleaved: bool = False) -> torch.Tensor:
    """The fused projection's rows qkv [T, (Hq + 2 Hkv) D]: q [T, Hq, D], normed and
    rotated; k, normed and rotated, and v go to their slots [T] of the cache.

    cos, sin: fp32 [max position, R / 2], the rotation of the first R dims of a head
    (R a multiple of 16; None: no rotation) at positions [T] (clamped to the table):
    the pairs (i, i + R / 2), or (2 i, 2 i + 1) if interleaved.  Scalings for long
    contexts are in the tables.  Everything is computed in fp32 and rounded once."""
    who = "qkv_append_paged"
    args = _cache_args(cache, who)
    hkv, d = args[8], args[10]
    device = cache.k.get_device()
    if num_heads < 1 or qkv.dim() != 2 or qkv.shape[1] != (num_heads + 2 * hkv) * d or qkv.get_device() != device:
        raise ValueError(f"{who}: qkv must be [T, {(num_heads + 2 * hkv) * d}] on the cache's device "
                         f"(got {tuple(qkv.shape)} on {qkv.device})")
    _no_gradients(who, qkv, q_norm, k_norm, cos, sin)
    rows = qkv.shape[0]
    cos, sin, most, rot = _rope_tables(cos, sin, d, device, who)
    q_norm = _norm_weight(q_norm, d, device, who, "q_norm")
    k_norm = _norm_weight(k_norm, d, device, who, "k_norm")
    slots = _ints(slots, _I32, rows, device, who, "slots")
    if rot:
        if positions is None:
            raise ValueError(f"{who}: a rotation needs positions")
        positions = _ints(positions, _I64, rows, device, who, "positions")
    if device < 0:
        x = qkv.float().view(rows, num_heads + 2 * hkv, d)
        at = positions.clamp(0, most - 1) if rot else None
        c, s = (cos[at], sin[at]) if rot else (None, None)
        _store_formula(cache, slots, _head_formula(x[:, num_heads:num_heads + hkv], k_norm, eps, c, s, interleaved),
                       x[:, num_heads + hkv:])
        return _head_formula(x[:, :num_heads], q_norm, eps, c, s, interleaved).to(qkv.dtype)
    if qkv.dtype is not _BF16:
        raise ValueError(f"{who}: qkv must be bfloat16 on the GPU (got {qkv.dtype})")
    if qkv.stride(1) != 1 or qkv.stride(0) % 8 or qkv.data_ptr() % 16:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    q = torch.empty_strided((rows, num_heads, d), (num_heads * d, d, 1), dtype=_BF16, device=qkv.device)
    if rows:
        at, stride = qkv.data_ptr(), qkv.stride(0)
        _call("paged_append", device, *args, at, stride, at + 2 * num_heads * d, stride, at + 2 * (num_heads + hkv) * d,
              stride, rows, num_heads, slots.data_ptr(), positions.data_ptr() if rot else None,
              cos.data_ptr() if rot else None, sin.data_ptr() if rot else None, most, rot, interleaved,
              None if q_norm is None else q_norm.data_ptr(), None if k_norm is None else k_norm.data_ptr(), eps,
              q.data_ptr())
    return q


# -- reading back and moving ---------------------------------------------------
def read_paged(cache: PagedKV, slots: torch.Tensor) -> tuple:
    """(k, v) [T, Hkv, D] bf16: the rows at slots [T], zeros for slots outside the cache."""
    who = "read_paged"
    args = _cache_args(cache, who)
    pages, hkv, page, d = args[7:]
    device = cache.k.get_device()
    slots = _ints(slots, _I32, None, device, who, "slots")
    rows = slots.shape[0]
    if device < 0:
        live = ((slots >= 0) & (slots < pages * page)).view(-1, 1, 1)
        at = slots.clamp(0, pages * page - 1).long()
        out = []
        for held, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
            y = held[at // page, :, at % page].float()
            if scale is not None:
                y = y * scale[at // page, :, at % page].unsqueeze(-1)
            out.append(torch.where(live, y, torch.zeros_like(y)).to(_BF16))
        return tuple(out)
    k, v = (torch.empty((rows, hkv, d), dtype=_BF16, device=slots.device) for _ in range(2))
    if rows:
        _call("paged_read", device, *args, slots.data_ptr(), rows, k.data_ptr(), v.data_ptr())
    return k, v


def move_paged(cache: PagedKV, src: torch.Tensor, dst: torch.Tensor) -> None:
    """The rows at slots src [n] to slots dst [n], as they are held.

    All are read before any is written, so the two may overlap (the accepted path
    of a drafted tree moves up behind the cache).  A pair with a slot outside the cache
    moves nothing; the dst are distinct."""
    who = "move_paged"
    args = _cache_args(cache, who)
    pages, hkv, page, d = args[7:]
    device = cache.k.get_device()
    src = _ints(src, _I32, None, device, who, "src")
    rows = src.shape[0]
    dst = _ints(dst, _I32, rows, device, who, "dst")
    if device < 0:
        live = (src >= 0) & (src < pages * page) & (dst >= 0) & (dst < pages * page)
        a, b = src[live].long(), dst[live].long()
        for held in cache:
            if held is not None:
                held[b // page, :, b % page] = held[a // page, :, a % page].clone()
    elif rows:
        need = _lib.load().nkv_paged_move_workspace(hkv, d, cache.k_scale is not None, rows)
        ws = torch.empty(need, dtype=torch.uint8, device=src.device)
        _call("paged_move", device, *args, src.data_ptr(), dst.data_ptr(), rows, ws.data_ptr())


# -- attention -----------------------------------------------------------------
def tree_masks(parents: torch.Tensor) -> torch.Tensor:
    """The masks of drafted trees: parents [..., n] (integers, n <= 64) gives for each
    token the one of its tree that it follows, before it in the tree, or -1 for the cache;
    int64 [..., n], bit j of token i's mask: it is j or follows j.

    One operation a token: made once for a tree's shape and kept."""
    if parents.dtype not in (_I32, _I64) or parents.dim() < 1 or not 1 <= parents.shape[-1] <= MAX_TREE:
        raise ValueError(f"tree_masks: parents must be int32 or int64 [..., n], n from 1 to {MAX_TREE} "
                         f"(got {parents.dtype} {tuple(parents.shape)})")
    n = parents.shape[-1]
    if not parents.is_cuda:
        order = torch.arange(n)
        if bool(((parents >= order) | (parents < -1)).any()):
            raise ValueError("tree_masks: a token's parent comes before it in the tree, or is -1")
    parents = parents.to(_I64)
    masks = torch.zeros(parents.shape, dtype=_I64, device=parents.device)
    for i in range(n):
        p = parents[..., i:i + 1]
        above = torch.where(p < 0, torch.zeros_like(p), masks.gather(-1, p.clamp(0, n - 1)))
        masks[..., i:i + 1] = above | ((1 << i) - (1 << 64) if i == 63 else 1 << i)
    return masks


def _attend_formula(q, cache, tables, lengths, starts, max_new, tree, scale) -> torch.Tensor:
    pages, hkv, page, d = cache.k.shape
    T, hq, _ = q.shape
    out = torch.zeros(T, hq, d)
    B = lengths.shape[0]
    starts = [b * max_new for b in range(B + 1)] if starts is None else starts.clamp(0, T).tolist()
    for b in range(B):
        n = min(starts[b + 1] - starts[b], max_new)
        length = min(max(int(lengths[b]), 0), tables.shape[1] * page)
        older = length - (starts[b + 1] - starts[b])
        key = torch.arange(length)
        ids = tables[b].long()[key // page]
        ok = (ids >= 0) & (ids < pages)
        at, off = ids.clamp(0, pages - 1), key % page
        k, v = (t[at, :, off].float() * (1.0 if c is None else c[at, :, off].unsqueeze(-1))
                for t, c in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        for i in range(n):
            t = starts[b] + i
            seen = key <= older + i
            if tree is not None:
                bit = (tree[t] >> (key - older).clamp(0, 63)) & 1
                seen = (key < older) | (bit.bool() & (key - older < MAX_TREE))
            seen = seen & ok
            if not bool(seen.any()):
                continue
            x = q[t].float().view(hkv, hq // hkv, d)
            w = torch.softmax(torch.matmul(x, k[seen].permute(1, 2, 0)) * scale, dim=-1)
            out[t] = torch.matmul(w, v[seen].transpose(0, 1)).reshape(hq, d)
    return out.to(q.dtype)


def attend_paged(q: torch.Tensor, cache: PagedKV, tables: torch.Tensor, lengths: torch.Tensor, *,
                 starts: torch.Tensor | None = None, max_new: int | None = None, tree: torch.Tensor | None = None,
                 scale: float | None = None) -> torch.Tensor:
    """Attention of new tokens q [T, Hq, D] over their sequences' keys: [T, Hq, D].

    Sequence b has lengths[b] keys in the pages tables[b] (int32 [B, most pages]), its new
    tokens' (appended before) the last of them.  Its queries are rows starts[b] ..
    starts[b + 1] - 1 (starts ascending [B + 1]), at most max_new of them (default T, of trees
    at most 64; a closer bound launches less; rows behind it give 0); without starts every sequence has T / B.  A
    query sees the keys up to its own token's, or with ``tree`` (int64 masks [T], or
    int32 ones of 32 tokens; at most 64 new tokens a sequence: ``tree_masks``) the keys before the new ones and those that its mask names.
    Rows that see nothing, or that belong to no sequence, are 0.  scale: of the
    logits (default D^-0.5)."""
    who = "attend_paged"
    args = _cache_args(cache, who)
    pages, hkv, page, d = args[7:]
    device = cache.k.get_device()
    if q.dim() != 3 or q.shape[2] != d or q.shape[1] < 1 or q.shape[1] % hkv or q.get_device() != device:
        raise ValueError(f"{who}: q must be [T, a multiple of {hkv}, {d}] on the cache's device "
                         f"(got {tuple(q.shape)} on {q.device})")
    T, hq, _ = q.shape
    if hq // hkv > 64:
        raise ValueError(f"{who}: at most 64 query heads share a KV head (got {hq // hkv})")
    _no_gradients(who, q)
    if (tables.dtype is not _I32 and tables.dtype is not _I64) or tables.dim() != 2 or tables.get_device() != device:
        raise ValueError(f"{who}: tables must be int32 [B, pages] on the cache's device "
                         f"(got {tables.dtype} {tuple(tables.shape)} on {tables.device})")
    B, most = tables.shape
    lengths = _ints(lengths, _I32, B, device, who, "lengths")
    if starts is None:
        if B == 0 and T or B and T % B:
            raise ValueError(f"{who}: without starts all {B} sequences have as many rows (got {T})")
        each = T // B if B else 0
        if max_new is not None and max_new != each:
            raise ValueError(f"{who}: without starts max_new is T / B = {each} (got {max_new})")
        max_new = each
    else:
        starts = _ints(starts, _I32, B + 1, device, who, "starts")
        if max_new is None:
            max_new = T if tree is None else MAX_TREE
        max_new = min(int(max_new), T)
        if T and max_new < 1:
            raise ValueError(f"{who}: max_new must be positive (got {max_new})")
    if tree is not None:
        if tree.dtype is _I32:
            tree = tree.to(_I64) & 0xffffffff   # (bit 31 is a token's, not a sign)
        tree = _ints(tree, _I64, T, device, who, "tree")
        if max_new > MAX_TREE:
            raise ValueError(f"{who}: a tree has at most {MAX_TREE} tokens (max_new is {max_new})")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"{who}: scale must be positive and finite (got {scale})")
    if T and B and (most < 1 or most * page > 2 ** 31 - 4097):
        raise ValueError(f"{who}: a page table covers from one page to 2^31 - 4097 tokens (got {most} pages of {page})")
    if device < 0:
        return _attend_formula(q, cache, tables, lengths, starts, max_new, tree, scale) if T else torch.empty_like(q)
    if q.dtype is not _BF16:
        raise ValueError(f"{who}: q must be bfloat16 on the GPU (got {q.dtype})")
    s = q.stride()
    if s[2] != 1 or (hq > 1 and s[1] != d) or s[0] % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    out = torch.empty_strided((T, hq, d), (hq * d, d, 1), dtype=_BF16, device=q.device)
    if T == 0:
        return out
    if B == 0:
        return out.zero_()
    if tables.dtype is not _I32:
        tables = _to_i32(tables)
    if tables.stride(1) != 1:
        tables = tables.contiguous()
    need = _workspace(device, B, T, max_new, hq, hkv, d, most, page, starts is not None)
    # (dropped behind the launch: the stream orders its reuse)
    ws = torch.empty(need, dtype=_F32, device=q.device) if need else None
    _call("paged_attend", device, *args, q.data_ptr(), q.stride(0), T, hq, tables.data_ptr(), tables.stride(0), most,
          lengths.data_ptr(), B, None if starts is None else starts.data_ptr(), max_new,
          None if tree is None else tree.data_ptr(), scale, out.data_ptr(), ws.data_ptr() if need else None)
    return out


def _workspace(device: int, *sizes) -> int:
    fn = _lib.load().nkv_paged_attend_workspace
    if device == _current_device():
        return fn(*sizes)
    with torch.cuda.device(device):
        return fn(*sizes)


__all__ = ["PagedKV", "append_paged", "attend_paged", "move_paged", "new_paged_kv", "qkv_append_paged", "read_paged",
           "tree_masks"]
