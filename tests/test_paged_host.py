"""The paged cache's operators without a GPU: their formulas, and the calls they refuse."""

import ctypes

import pytest
import torch

from _paged_ref import heads_ref, held, make_cache, rope_tables
from nanokv_amd import _lib
from nanokv_amd.paged import (PagedKV, append_paged, move_paged, new_paged_kv, qkv_append_paged, read_paged)


def _copy(cache):
    return PagedKV(*(None if t is None else t.clone() for t in cache))


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("inter", [False, True])
def test_append_formula(kv, inter):
    g = torch.Generator().manual_seed(1)
    cache = make_cache(3, 2, 16, 64, kv, "cpu")
    qkv = torch.randn(10, 8 * 64, generator=g).bfloat16()
    cos, sin = rope_tables(50, 32, "cpu")
    slots = torch.tensor([5, -1, 40, 0, 47, 48, 17, 18, 19, 31])
    pos = torch.arange(10)
    w = (1 + 0.1 * torch.randn(64, generator=g)).bfloat16()
    q = qkv_append_paged(cache, qkv, slots, pos, cos, sin, 4, q_norm=w, k_norm=None, interleaved=inter)
    x = qkv.view(10, 8, 64)
    ref, mag = heads_ref(x[:, :4], w, 1e-6, cos[pos], sin[pos], inter)
    assert bool(((q.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -18 * mag).all())
    k, v = read_paged(cache, slots)
    assert bool((k[1] == 0).all()) and bool((v[5] == 0).all())
    live = (slots >= 0) & (slots < 48)
    ref, mag = heads_ref(x[:, 4:6], None, 1e-6, cos[pos], sin[pos], inter)
    # 8 bits: half a step of the row's largest / 127, its value rounded to bf16
    step = (ref.abs().amax(-1, keepdim=True) / 127 * (0.5 + 2.0 ** -10)) if kv == "int8" else 0.0
    assert bool(((k.double() - ref).abs() <= 2.0 ** -8 * (ref.abs() + step) + 2.0 ** -18 * mag + step)[live].all())
    if kv == "bf16":
        assert torch.equal(v[live], x[live][:, 6:])


@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_moves_read_before_they_write(kv):
    cache = make_cache(2, 2, 16, 64, kv, "cpu")
    was = _copy(cache)
    move_paged(cache, torch.tensor([3, 4, 9, -1]), torch.tensor([4, 3, 32, 5]))
    for which in (0, 1):
        a, b = held(cache, which), held(was, which)
        assert torch.equal(a[0, :, 4], b[0, :, 3]) and torch.equal(a[0, :, 3], b[0, :, 4])
        assert torch.equal(a[0, :, 5:], b[0, :, 5:]) and torch.equal(a[1], b[1])


def test_append_rows_and_new_caches():
    for dtype in (torch.bfloat16, torch.int8):
        cache = new_paged_kv(2, 1, 16, 64, dtype, device="cpu")
        assert (cache.k_scale is None) == (dtype is torch.bfloat16)
        append_paged(cache, torch.ones(1, 1, 64), torch.full((1, 1, 64), 2.0), torch.tensor([20]))
        k, v = read_paged(cache, torch.tensor([20, 21]))
        assert bool((k[0] == 1).all()) and bool((v[0] == 2).all()) and bool((k[1] == 0).all())
    with pytest.raises(ValueError, match="dtype"):
        new_paged_kv(2, 1, 16, 64, torch.float16, device="cpu")
    with pytest.raises(ValueError, match="power of two"):
        new_paged_kv(2, 1, 24, 64, device="cpu")
    with pytest.raises(ValueError, match="64 or 128"):
        new_paged_kv(2, 1, 16, 96, device="cpu")


@pytest.mark.parametrize("change,words", [
    (dict(k=torch.zeros(3, 2, 16, 64)), "bfloat16 or int8"),
    (dict(v=torch.zeros(3, 2, 16, 64, dtype=torch.int8)), "bfloat16 or int8"),
    (dict(v=torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16).transpose(1, 2)), "lie alike"),
    (dict(k=torch.zeros(3, 2, 64, 16, dtype=torch.bfloat16).transpose(2, 3),
          v=torch.zeros(3, 2, 64, 16, dtype=torch.bfloat16).transpose(2, 3)), "lie alike"),
    (dict(k_scale=torch.zeros(3, 2, 16)), "no scales")])
def test_caches_that_are_refused(change, words):
    cache = make_cache(3, 2, 16, 64, "bf16", "cpu")._replace(**change)
    rows = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: append_paged(cache, rows, rows, torch.zeros(1, dtype=torch.int32)),
                 lambda: read_paged(cache, torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ValueError, match=words):
            call()


@pytest.mark.parametrize("scale", [None, torch.zeros(3, 2, 16, dtype=torch.float16), torch.zeros(3, 2, 8),
                                   torch.zeros(3, 2, 32)[:, :, ::2]])
def test_scales_that_are_refused(scale):
    cache = make_cache(3, 2, 16, 64, "int8", "cpu")._replace(v_scale=scale)
    with pytest.raises(ValueError, match="dense float32 scales"):
        read_paged(cache, torch.zeros(1, dtype=torch.int32))


COS, SIN = rope_tables(8, 64, "cpu")


@pytest.mark.parametrize("change,words", [
    (dict(qkv=torch.zeros(2, 500)), "qkv must be"), (dict(num_heads=0), "qkv must be"),
    (dict(qkv=torch.zeros(1, 2, 512)), "qkv must be"),
    (dict(slots=torch.zeros(3, dtype=torch.int32)), "slots must be"), (dict(slots=torch.zeros(2)), "slots must be"),
    (dict(positions=None), "needs positions"), (dict(positions=torch.zeros(1, dtype=torch.long)), "positions must be"),
    (dict(cos=None), "come together"), (dict(cos=COS[:, :4], sin=SIN[:, :4]), "cos and sin"),
    (dict(cos=torch.zeros(8, 40), sin=torch.zeros(8, 40)), "cos and sin"), (dict(cos=COS.double()), "cos and sin"),
    (dict(q_norm=torch.zeros(32)), "q_norm must be"), (dict(k_norm=torch.zeros(1, 64)), "k_norm must be"),
    (dict(qkv=torch.zeros(2, 512, requires_grad=True)), "gradient")])
def test_appends_that_are_refused(change, words):
    args = dict(cache=make_cache(3, 2, 16, 64, "bf16", "cpu"), qkv=torch.zeros(2, 512),
                slots=torch.zeros(2, dtype=torch.int32), positions=torch.zeros(2, dtype=torch.long), cos=COS, sin=SIN,
                num_heads=4) | change
    with pytest.raises(ValueError, match=words):
        qkv_append_paged(**args)


def test_rows_that_are_refused():
    cache = make_cache(3, 2, 16, 64, "bf16", "cpu")
    ok = torch.zeros(2, 2, 64)
    for k, v, slots in ((torch.zeros(2, 3, 64), ok, torch.zeros(2, dtype=torch.int32)),
                        (ok, torch.zeros(3, 2, 64), torch.zeros(2, dtype=torch.int32)),
                        (ok, ok, torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ValueError):
            append_paged(cache, k, v, slots)
    with pytest.raises(ValueError, match="dst must be"):
        move_paged(cache, torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))


# -- the library's own checks ------------------------------------------------------
P = ctypes.c_void_p(64)       # never dereferenced: every call below fails its checks
CACHE = dict(k=P, v=P, ks=None, vs=None, sp=2048, sh=1024, st=64, pages=3, hkv=2, page=16, d=64)
BAD_CACHES = [(dict(d=96), b"head_dim"), (dict(page=24), b"page_size"), (dict(page=8), b"page_size"),
              (dict(page=8192), b"page_size"), (dict(k=None), b"NULL"), (dict(ks=P), b"both scales"),
              (dict(pages=0), b"positive"), (dict(hkv=0), b"positive"), (dict(pages=2 ** 31 - 1), b"2^31"),
              (dict(st=32), b"overlap"), (dict(sh=-8), b"negative"), (dict(k=ctypes.c_void_p(72)), b"16-byte"),
              (dict(sp=2044), b"16-byte"), (dict(st=2 ** 26), b"too far apart")]


def refused(rc, words):
    return rc in (_lib.NKV_ERR_ARG, _lib.NKV_ERR_UNSUPPORTED) and words in _lib.load().nkv_last_error()


@pytest.mark.parametrize("change,words", BAD_CACHES)
def test_the_library_refuses_a_cache(change, words):
    lib, c = _lib.load(), list((CACHE | change).values())
    assert refused(lib.nkv_paged_append(*c, P, 512, P, 512, P, 512, 1, 4, P, P, P, P, 8, 64, 0, P, P, 1e-6, P, None), words)
    assert refused(lib.nkv_paged_read(*c, P, 1, P, P, None), words)
    assert refused(lib.nkv_paged_move(*c, P, P, 1, P, None), words)


def test_the_library_refuses_rows():
    lib, c = _lib.load(), list(CACHE.values())
    good = dict(q=P, qs=512, k=P, ks=512, v=P, vs=512, rows=1, heads=4, slots=P, pos=P, cos=P, sin=P, most=8, rot=64,
                inter=0, qw=P, kw=P, eps=1e-6, out=P)
    for change, words in ((dict(rows=-1), b"negative"), (dict(rows=2 ** 27), b"2^27"), (dict(rot=72), b"rotary_dim"),
                          (dict(rot=80), b"rotary_dim"), (dict(rot=-16), b"rotary_dim"), (dict(k=None), b"non-NULL"),
                          (dict(slots=None), b"non-NULL"), (dict(out=None), b"q_rows and q_out"),
                          (dict(pos=None), b"rotation"), (dict(most=0), b"rotation"), (dict(qs=511), b"16-byte"),
                          (dict(v=ctypes.c_void_p(70)), b"16-byte"), (dict(cos=ctypes.c_void_p(68)), b"16-byte")):
        assert refused(lib.nkv_paged_append(*c, *(good | change).values(), None), words), change
    assert lib.nkv_paged_append(*c, *(good | dict(rows=0)).values(), None) == _lib.NKV_OK
    assert refused(lib.nkv_paged_read(*c, P, -1, P, P, None), b"rows")
    assert refused(lib.nkv_paged_read(*c, None, 1, P, P, None), b"non-NULL")
    assert refused(lib.nkv_paged_move(*c, P, P, 1, None, None), b"workspace")
    assert lib.nkv_paged_move_workspace(8, 128, 0, 5) == 5 * 2 * 8 * 256
    assert lib.nkv_paged_move_workspace(8, 128, 1, 5) == 5 * 2 * 8 * 132
