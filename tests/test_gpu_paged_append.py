"""Rows written to a paged cache, read back and moved, against their definition in 64 bits.

Tolerances, with u = 2^-24 the half step of fp32 and 2^-8 bf16's:
* a head's sum of up to 128 squares is a chain of 16 a lane and 3 joins: 20 u; the
  root halves it, and root, division, the mean's product and r * w, x * (r w) add 6 u: 16 u;
* a rotated value is two products and a sum: 3 u of the terms' magnitude more.
So fp32 values are off by less than 20 u < 2^-19 of their terms' magnitude, and bf16
ones by 2^-8 |ref| more.  A code's y * 127 / a: the pair's terms are at most twice the
row's maximum a in magnitude, so y and a are off by 2^-18 a each and the code by 0.5 + 2 * 127 * 2^-18 < 0.5 + 2^-10.
"""

import pytest
import torch

from _paged_ref import heads_ref, held, make_cache, rope_tables

pytestmark = pytest.mark.gpu


def _close(got, ref, mag):
    err = (got.double() - ref).abs()
    assert bool((err <= 2.0 ** -8 * ref.abs() + 2.0 ** -18 * mag + 1e-30).all()), float(err.max())


def _rows(T, hq, hkv, d, seed, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (hq + 2 * hkv) * d
    x = torch.randn(T, w + pad, generator=g, device="cuda") * torch.randn(w + pad, generator=g, device="cuda").exp()
    return x.bfloat16()[:, :w]


def _check(cache, before, slots, k, kmag, v):
    """The slots hold k and v, all else is as before."""
    page = cache.k.shape[2]
    live = (slots >= 0) & (slots < cache.k.shape[0] * page)
    at = slots[live].long()
    p, o = at // page, at % page
    for which, y, mag in ((0, k, kmag), (1, v, v.abs())):
        y, mag = y[live], mag[live]
        if cache.k_scale is None:
            _close(cache[which][p, :, o], y, mag)
        else:
            top = y.abs().amax(-1)
            s = cache[2 + which][p, :, o].double()
            assert bool(((s - top / 127).abs() <= 2.0 ** -17 * top / 127).all())
            code = cache[which][p, :, o].double()
            assert float((code - y * (127 / top).unsqueeze(-1)).abs().max()) <= 0.5 + 2.0 ** -10
        rest = torch.ones(cache.k.shape[0], page, dtype=torch.bool, device="cuda")
        rest[p, o] = False
        assert torch.equal(cache[which].transpose(1, 2)[rest], before[which].transpose(1, 2)[rest])
        if cache.k_scale is not None:
            assert torch.equal(cache[2 + which].transpose(1, 2)[rest], before[2 + which].transpose(1, 2)[rest])


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("T,hq,hkv,d,page,rot,inter,norm", [
    (1, 32, 8, 128, 64, 128, False, True), (1, 1, 1, 64, 16, 64, True, False), (5, 40, 8, 64, 32, 32, False, True),
    (33, 16, 8, 128, 16, 64, True, True), (257, 3, 3, 128, 256, 16, False, False), (300, 8, 2, 64, 4096, 48, True, True),
    (100, 7, 1, 128, 128, 112, False, True), (64, 4, 4, 128, 64, 0, False, True)])
def test_qkv_append(kv, T, hq, hkv, d, page, rot, inter, norm):
    from nanokv_amd.paged import PagedKV, qkv_append_paged, read_paged
    pages = -(-T // page) + 2
    cache = make_cache(pages, hkv, page, d, kv, "cuda", seed=T)
    before = PagedKV(*(None if t is None else t.clone() for t in cache))
    qkv = _rows(T, hq, hkv, d, T + hq, pad=8 * (T % 3))
    g = torch.Generator(device="cuda").manual_seed(1)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T].to(torch.int32)
    slots[1::7] = torch.tensor([-1, pages * page, 2 ** 31 - 1, -2 ** 31] * T, dtype=torch.int32, device="cuda")[:len(slots[1::7])]
    pos = torch.randint(0, 500, (T,), generator=g, device="cuda")
    pos[0] = 0
    cos, sin = rope_tables(500, rot, "cuda") if rot else (None, None)
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=g, device="cuda")).bfloat16() for _ in range(2)) if norm else (None, None)
    q = qkv_append_paged(cache, qkv, slots, pos if rot else None, cos, sin, hq, q_norm=wq, k_norm=wk, eps=1e-5,
                         interleaved=inter)
    x = qkv.reshape(T, hq + 2 * hkv, d)
    c, s = (cos[pos], sin[pos]) if rot else (None, None)
    _close(q, *heads_ref(x[:, :hq], wq, 1e-5, c, s, inter))
    k, kmag = heads_ref(x[:, hq:hq + hkv], wk, 1e-5, c, s, inter)
    _check(cache, before, slots, k, kmag, x[:, hq + hkv:].double())
    rk, rv = read_paged(cache, slots)
    live = (slots >= 0) & (slots < pages * page)
    at = slots.clamp(0, pages * page - 1).long()
    for got, which in ((rk, 0), (rv, 1)):
        want = held(cache, which)[at // page, :, at % page] * live.view(-1, 1, 1)
        # (code * scale in fp32, then bf16: 2^-24 and 2^-8)
        assert bool(((got.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -23) * want.abs()).all())


def test_positions_are_clamped_to_the_table_and_other_integers_taken():
    from nanokv_amd.paged import qkv_append_paged
    cache = make_cache(2, 2, 16, 64, "bf16", "cuda")
    qkv = _rows(4, 4, 2, 64, 3)
    cos, sin = rope_tables(10, 64, "cuda")
    slots = torch.arange(4, device="cuda")
    q = qkv_append_paged(cache, qkv, slots, torch.tensor([-5, 0, 9, 2 ** 40], device="cuda"), cos, sin, 4)
    r = qkv_append_paged(cache, qkv, slots.int(), torch.tensor([0, 0, 9, 9], device="cuda", dtype=torch.int32), cos, sin, 4)
    assert torch.equal(q, r)


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("T,hkv,d,page", [(1, 8, 128, 64), (129, 1, 64, 16), (77, 5, 128, 32)])
def test_append_rows_bit_for_bit(kv, T, hkv, d, page):
    """Rows that come rotated: bf16 is copied; codes of bf16 values are rne(127 y / a) with exact ties."""
    from nanokv_amd.paged import append_paged
    from nanokv_amd.q8 import quantize_q8
    cache = make_cache(-(-T // page) + 1, hkv, page, d, kv, "cuda")
    wide = _rows(T, hkv, hkv, d, 5)                      # k and v are column ranges of wider rows
    k, v = (wide[:, i * hkv * d:(i + 1) * hkv * d].unflatten(1, (hkv, d)) for i in range(2))
    slots = torch.randperm(cache.k.shape[0] * page, device="cuda")[:T]
    append_paged(cache, k, v, slots)
    p, o = slots // page, slots % page
    for which, y in ((0, k), (1, v)):
        if kv == "bf16":
            assert torch.equal(cache[which][p, :, o], y)
        else:
            t = quantize_q8(y.contiguous())
            assert torch.equal(cache[which][p, :, o], t.q) and torch.equal(cache[2 + which][p, :, o], t.scale)


def test_rows_that_no_code_holds():
    from nanokv_amd.paged import append_paged, read_paged
    cache = make_cache(1, 1, 16, 64, "int8", "cuda")
    y = torch.randn(5, 1, 64, device="cuda").bfloat16()
    y[1] = 0
    y[2, 0, 5] = float("inf")
    y[3, 0, 9] = float("nan")
    y[4] = 2.0 ** -126
    append_paged(cache, y, y, torch.arange(5, device="cuda"))
    s = cache.k_scale[0, 0, :5]
    assert float(s[1]) == 0 and float(s[4]) == 0 and bool(s[2:4].isnan().all()) and bool(s[0] > 0)
    assert bool((cache.k[0, 0, 1:5] == 0).all()) and torch.equal(cache.k[0, 0, :5], cache.v[0, 0, :5])
    k, v = read_paged(cache, torch.arange(5, device="cuda"))
    assert bool(k[2:4].isnan().all()) and bool((k[1] == 0).all()) and torch.equal(k[:2], v[:2])


@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_a_cache_in_another_order(kv):
    """[pages, page, Hkv, D] in memory, and one layer of [pages, L, ...], are written and read in place."""
    from nanokv_amd.paged import PagedKV, append_paged, qkv_append_paged, read_paged
    dense = make_cache(3, 4, 32, 64, kv, "cuda")
    k = torch.empty(3, 32, 4, 64, dtype=dense.k.dtype, device="cuda").transpose(1, 2)
    layers = torch.empty(2, 3, 2, 4, 32, 64, dtype=dense.k.dtype, device="cuda")
    qkv = _rows(20, 4, 4, 64, 9)
    slots = torch.randperm(96, device="cuda")[:20]
    for view_k, view_v in ((k, k.clone(memory_format=torch.preserve_format)), (layers[0, :, 1], layers[1, :, 1])):
        view_k.copy_(dense.k), view_v.copy_(dense.v)
        other = PagedKV(view_k, view_v, *(None if t is None else t.clone() for t in dense[2:]))
        same = PagedKV(*(None if t is None else t.clone() for t in dense))
        for c in (other, same):
            qkv_append_paged(c, qkv, slots, None, None, None, 4)
            append_paged(c, qkv[:3, :256].unflatten(1, (4, 64)), qkv[:3, 256:512].unflatten(1, (4, 64)), slots[:3])
        for a, b in zip(other, same):
            assert a is None or torch.equal(a, b)
        for a, b in zip(read_paged(other, slots), read_paged(same, slots)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_moves_read_before_they_write(kv):
    from nanokv_amd.paged import PagedKV, move_paged
    cache = make_cache(70, 8, 16, 128, kv, "cuda")
    before = PagedKV(*(None if t is None else t.clone() for t in cache))
    # every row one place on (each slot is read and written), some pairs that move nothing
    src = torch.arange(0, 1100, device="cuda", dtype=torch.int32)
    dst = src + 1
    src[5], dst[9], src[30] = -1, 70 * 16, 2 ** 31 - 1
    move_paged(cache, src, dst)
    for which in range(4):
        if cache[which] is None:
            continue
        flat = cache[which].transpose(1, 2).flatten(0, 1)
        want = before[which].transpose(1, 2).flatten(0, 1).clone()
        was = want.clone()
        want[1:1101] = was[0:1100]
        want[6], want[10], want[31] = was[6], was[10], was[31]
        assert torch.equal(flat, want)


def test_no_rows():
    from nanokv_amd.paged import append_paged, move_paged, qkv_append_paged, read_paged
    cache = make_cache(1, 2, 16, 64, "bf16", "cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert qkv_append_paged(cache, torch.empty(0, 6 * 64, dtype=torch.bfloat16, device="cuda"), none, None, None, None,
                            2).shape == (0, 2, 64)
    rows = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    append_paged(cache, rows, rows, none)
    move_paged(cache, none, none)
    assert read_paged(cache, none)[0].shape == (0, 2, 64)


def test_another_stream_and_a_graph():
    """A captured append is replayed with other slots, positions and rows."""
    from nanokv_amd.paged import append_paged, qkv_append_paged
    cache, want = (make_cache(4, 2, 16, 128, "int8", "cuda") for _ in range(2))
    cos, sin = rope_tables(100, 128, "cuda")
    qkv, slots, pos = _rows(6, 4, 2, 128, 0).contiguous(), torch.arange(6, device="cuda", dtype=torch.int32), \
        torch.arange(6, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        qkv_append_paged(cache, qkv, slots, pos, cos, sin, 4)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q = qkv_append_paged(cache, qkv, slots, pos, cos, sin, 4)
    for step in range(3):
        qkv.copy_(_rows(6, 4, 2, 128, step + 1))
        slots.copy_(torch.randperm(64, device="cuda")[:6])
        pos.add_(7)
        g.replay()
        assert torch.equal(q, qkv_append_paged(want, qkv, slots, pos, cos, sin, 4))
    torch.cuda.synchronize()
    append_paged(want, torch.zeros(1, 2, 128, dtype=torch.bfloat16, device="cuda"),
                 torch.zeros(1, 2, 128, dtype=torch.bfloat16, device="cuda"), torch.tensor([-1], device="cuda"))
    live = want.k_scale != make_cache(4, 2, 16, 128, "int8", "cuda").k_scale
    assert torch.equal(cache.k[live], want.k[live]) and torch.equal(cache.v_scale[live], want.v_scale[live])
