"""attend_paged and tree_masks without a GPU: their formulas, and the calls they refuse."""

import ctypes

import pytest
import torch

from _paged_ref import attend_ref, make_cache
from nanokv_amd import _lib
from nanokv_amd.paged import attend_paged, tree_masks
from test_paged_host import BAD_CACHES, CACHE, P, refused


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("tree", [False, True])
def test_formula(kv, tree):
    g = torch.Generator().manual_seed(0)
    cache = make_cache(9, 2, 16, 64, kv, "cpu")
    tables = torch.tensor([[3, 0, 5, -1], [7, 99, 2, 1], [4, 6, 8, -1]])
    lengths = torch.tensor([35, 64, 2])
    starts = torch.tensor([1, 4, 4, 9])
    q = torch.randn(11, 6, 64, generator=g).bfloat16()
    masks = torch.randint(-2 ** 40, 2 ** 40, (11,), generator=g) if tree else None
    got = attend_paged(q, cache, tables, lengths, starts=starts, tree=masks)
    ref, mag = attend_ref(q, cache, tables, lengths, starts, masks)
    # fp32: logits below 30, off by 70 * 30 * 2^-24; two such weights
    assert bool(((got.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -11 * mag).all())
    assert bool((got[0] == 0).all()) and bool((got[9:] == 0).all())
    line = attend_paged(q[:9], cache, tables, lengths, scale=0.2)
    ref, mag = attend_ref(q[:9], cache, tables, lengths, scale=0.2, n_each=3)
    assert bool(((line.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -10 * mag).all())


def test_masks_of_trees():
    m = tree_masks(torch.tensor([[-1, 0, 0, 1, -1], [-1, 0, 1, 2, 3]]))
    assert m.tolist() == [[1, 3, 5, 11, 16], [1, 3, 7, 15, 31]]
    line = tree_masks(torch.arange(-1, 63, dtype=torch.int32))
    assert line[62] == 2 ** 63 - 1 and line[63] == -1
    for bad in (torch.tensor([0]), torch.tensor([-1, 1]), torch.tensor([-2]), torch.zeros(65, dtype=torch.long) - 1,
                torch.tensor([-1.0]), torch.tensor(-1), torch.zeros(2, 0, dtype=torch.long)):
        with pytest.raises(ValueError, match="tree_masks"):
            tree_masks(bad)


Q = torch.zeros(4, 4, 64)


@pytest.mark.parametrize("change,words", [
    (dict(q=torch.zeros(4, 3, 64)), "q must be"), (dict(q=torch.zeros(4, 4, 128)), "q must be"),
    (dict(q=torch.zeros(4, 256)), "q must be"), (dict(q=torch.zeros(4, 130, 64)), "at most 64 query heads"),
    (dict(q=torch.zeros(4, 4, 64, requires_grad=True)), "gradient"),
    (dict(tables=torch.zeros(2, 3)), "tables must be"), (dict(tables=torch.zeros(2, dtype=torch.int32)), "tables must be"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths must be"), (dict(lengths=torch.zeros(2)), "lengths must be"),
    (dict(q=torch.zeros(5, 4, 64)), "as many rows"), (dict(max_new=1), "without starts"),
    (dict(starts=torch.zeros(2, dtype=torch.int32)), "starts must be"),
    (dict(starts=torch.zeros(3, dtype=torch.int32), max_new=0), "positive"),
    (dict(tree=torch.zeros(3, dtype=torch.int64)), "tree must be"), (dict(tree=torch.zeros(4)), "tree must be"),
    (dict(q=torch.zeros(130, 4, 64), tree=torch.zeros(130, dtype=torch.int64)), "at most 64 tokens"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(tables=torch.zeros(2, 0, dtype=torch.int32)), "page table")])
def test_refusals(change, words):
    args = dict(q=Q, cache=make_cache(3, 2, 16, 64, "bf16", "cpu"), tables=torch.zeros(2, 3, dtype=torch.int32),
                lengths=torch.zeros(2, dtype=torch.int32)) | change
    with pytest.raises(ValueError, match=words):
        attend_paged(**args)


def test_no_rows():
    cache = make_cache(3, 2, 16, 64, "bf16", "cpu")
    none = torch.zeros(0, dtype=torch.int32)
    assert attend_paged(Q[:0], cache, torch.zeros(0, 3, dtype=torch.int32), none).shape == (0, 4, 64)
    assert bool((attend_paged(Q, cache, torch.zeros(0, 3, dtype=torch.int32), none,
                              starts=torch.zeros(1, dtype=torch.int32)) == 0).all())


def test_the_library_refuses_before_any_device_work():
    lib = _lib.load()
    good = dict(q=P, qs=256, rows=4, heads=4, tables=P, ts=3, most=3, lengths=P, batch=2, starts=None, new=2, tree=None,
                scale=0.1, out=P, ws=P)

    def call(cache=None, **change):
        return lib.nkv_paged_attend(*(CACHE | (cache or {})).values(), *(good | change).values(), None)

    for change, words in BAD_CACHES:
        assert refused(call(change), words), change
    assert refused(call(dict(ks=ctypes.c_void_p(72), vs=P)), b"scales must lie")
    assert refused(call(dict(hkv=300), batch=65535, rows=65535, new=1, heads=300, most=1), b"2^24 pairs")
    assert refused(call(dict(hkv=1), batch=1, rows=2 ** 20, new=2 ** 20, heads=64, most=4096), b"65535 query tiles")
    assert refused(call(dict(hkv=300), batch=4096, rows=4096, new=1, heads=300, most=65536), b"2^31 pieces of 32 keys")
    for change, words in ((dict(batch=-1), b"65535 sequences"), (dict(batch=65536, rows=131072), b"65535 sequences"),
                          (dict(new=0), b"max_new"), (dict(new=2 ** 20 + 1), b"max_new"), (dict(heads=3), b"multiple"),
                          (dict(heads=130), b"64 query heads"), (dict(most=0), b"page table"),
                          (dict(most=2 ** 27), b"page table"), (dict(rows=5), b"without starts"),
                          (dict(new=65, rows=130, tree=P), b"a tree has"), (dict(scale=0.0), b"scale"),
                          (dict(scale=float("nan")), b"scale"), (dict(q=None), b"non-NULL"),
                          (dict(lengths=None), b"non-NULL"), (dict(qs=255), b"16-byte"),
                          (dict(out=ctypes.c_void_p(72)), b"16-byte"), (dict(batch=0, starts=P), b"need a sequence"),
                          (dict(most=1000, ws=None), b"workspace"), (dict(most=1000, ws=ctypes.c_void_p(72)), b"workspace")):
        assert refused(call(**change), words), change
    assert call(rows=0, starts=P) == _lib.NKV_OK
    assert lib.nkv_paged_attend_workspace(0, 4, 1, 4, 2, 64, 3, 16, 0) == 0
    assert lib.nkv_paged_attend_workspace(1, 1, 1, 4, 2, 64, 1, 16, 0) == 0
    assert lib.nkv_paged_attend_workspace(1, 1, 1, 4, 2, 64, 1000, 16, 0) > 0
