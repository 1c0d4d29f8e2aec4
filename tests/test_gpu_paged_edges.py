"""The paged operators on the GPU at the ends of their arguments: integers past 32 bits, thousands of sequences
and of rows of padding."""

import pytest
import torch

from _paged_ref import make_cache
from test_gpu_paged_attend import _check, _q, _setup

pytestmark = pytest.mark.gpu
FAR = [2 ** 32 + 5, -2 ** 63, 2 ** 63 - 1, 2 ** 32, 2 ** 31, -2 ** 32 + 7]


@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_slots_past_32_bits_lie_outside_the_cache(kv):
    from nanokv_amd.paged import PagedKV, append_paged, move_paged, qkv_append_paged, read_paged
    cache = make_cache(3, 2, 16, 64, kv, "cuda")
    was = PagedKV(*(None if t is None else t.clone() for t in cache))
    far, near = torch.tensor(FAR, device="cuda"), torch.arange(len(FAR), device="cuda")
    rows = torch.ones(len(FAR), 2, 64, dtype=torch.bfloat16, device="cuda")
    append_paged(cache, rows, rows, far)
    qkv_append_paged(cache, torch.ones(len(FAR), 8 * 64, dtype=torch.bfloat16, device="cuda"), far, None, None, None, 4)
    move_paged(cache, far, near)
    move_paged(cache, near, far)
    assert all(torch.equal(a, b) for a, b in zip(cache, was) if a is not None)
    assert all(bool((t == 0).all()) for t in read_paged(cache, far))


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("n", [1, 30])
def test_lengths_tables_and_starts_past_32_bits(kv, n):
    from nanokv_amd.paged import attend_paged
    cache, tables, lens = _setup([160, 160], 2, 16, 64, kv, seed=1, poison=False)
    tables = tables[:, :10].contiguous()
    q = _q(2 * n, 8, 64, 2)
    full = attend_paged(q, cache, tables, lens)
    got = attend_paged(q, cache, tables, torch.tensor([2 ** 32 + 3, -2 ** 63 + 4], device="cuda"))
    assert torch.equal(got[:n], full[:n]) and bool((got[n:] == 0).all())
    far = tables.long()
    far[0, 3], far[0, 5], far[1, 0], far[1, 9] = 2 ** 32, 2 ** 32 + 1, -2 ** 63, 2 ** 63 - 1
    got = attend_paged(q, cache, far, lens)
    _check(got, q, cache, far, lens, n_each=n)
    starts = torch.tensor([0, n, 2 ** 32 + n], device="cuda")
    assert torch.equal(attend_paged(q, cache, tables, lens, starts=starts, max_new=n),
                       attend_paged(q, cache, tables, lens, starts=starts.clamp(max=2 * n), max_new=n))


@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_thousands_of_sequences(kv):
    """A token of each of 4500 sequences (their chunks of 64 fall into blocks of two), a few of them long, many
    empty; then without a new token for most."""
    from nanokv_amd.paged import attend_paged
    B = 4500
    lengths = [(37 * b) % 40 if b % 3 else 0 for b in range(B)]
    lengths[70], lengths[2500], lengths[-1] = 3000, 1500, 700
    cache, tables, lens = _setup(lengths, 1, 16, 64, kv, seed=8, poison=False)
    q = _q(B, 2, 64, 1)
    _check(attend_paged(q, cache, tables, lens), q, cache, tables, lens)
    counts = [1 if b % 50 == 7 or b > B - 9 else 0 for b in range(B)]
    starts = torch.tensor([0] + counts).cumsum(0).int().cuda()
    n = int(starts[-1])
    got = attend_paged(q[:n], cache, tables, lens, starts=starts, max_new=1)
    _check(got, q[:n], cache, tables, lens, starts)


@pytest.mark.parametrize("kv,hkv,d", [("bf16", 1, 128), ("int8", 1, 64)])
def test_a_shared_list_of_many_query_tiles(kv, hkv, d):
    """450 sequences of up to 20 new tokens whose tables are wide: one list of key tiles, several chunks of units."""
    from nanokv_amd.paged import attend_paged
    lengths = [20 + (53 * b) % 60 for b in range(450)]
    lengths[200], lengths[449] = 2600, 900
    cache, tables, lens = _setup(lengths, hkv, 16, d, kv, seed=9, poison=False)
    tables = torch.nn.functional.pad(tables, (0, 2048 - tables.shape[1]), value=-1)
    q = _q(9000, 2 * hkv, d, 2)
    _check(attend_paged(q, cache, tables, lens), q, cache, tables, lens, n_each=20)


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("n,wide", [(1, 1), (3, 1), (30, 1), (30, 4096), (300, 1)])
def test_rows_of_padding(kv, n, wide):
    """Thousands of rows of no sequence before, behind and (past max_new) between the others: all 0, whatever
    the memory held, and the others as without them."""
    from nanokv_amd.paged import attend_paged
    cache, tables, lens = _setup([n + 70, n, n + 5, 2 * n], 2, 16, 64, kv, seed=n, poison=False)
    tables = torch.nn.functional.pad(tables, (0, wide), value=-1)
    rows = [(3001, n), (3001 + n, 0), (3001 + n, 1500), (4501 + n, 1)]       # first row, rows of each sequence
    starts = torch.tensor([r for r, _ in rows] + [4502 + n], dtype=torch.int32, device="cuda")
    T = 4502 + n + 2017
    q = _q(T, 8, 64, 3)
    junk = torch.full((4, T, 8, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    del junk                                                                # (the output may take its memory)
    got = attend_paged(q, cache, tables, lens, starts=starts, max_new=n)
    live = torch.zeros(T, dtype=torch.bool, device="cuda")
    for first, count in rows:
        live[first:first + min(count, n)] = True
    assert bool((got[~live] == 0).all())
    some = [0, 3]                                                           # sequences whose rows are all there
    for b in some:
        first, count = rows[b]
        one = torch.tensor([0, count], dtype=torch.int32, device="cuda")
        alone = attend_paged(q[first:first + count].contiguous(), cache, tables[b:b + 1], lens[b:b + 1], starts=one,
                             max_new=n)
        tol = 2 * 3.03 * 2.0 ** -8 * float(cache.v.float().abs().max()) * (1.0 if kv == "bf16" else 0.025)
        assert float((got[first:first + count].float() - alone.float()).abs().max()) <= tol


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("n,hq,hkv,d,older,wide", [
    (4, 4, 1, 128, 60, 0), (16, 1, 1, 64, 1000, 0), (7, 4, 2, 64, 3, 0), (16, 4, 1, 128, 40, 0), (13, 5, 1, 64, 200, 0),
    (60, 8, 2, 128, 37, 0), (64, 4, 1, 64, 100, 0), (50, 4, 2, 128, 500, 4096), (40, 8, 1, 64, 90, 4096), (12, 4, 1, 64, 5, 4096)])
def test_values_that_some_queries_see(tree, n, hq, hkv, d, older, wide):
    """NaN and infinities in some dims of several new tokens: the outputs are the formula's, infinities, NaN and
    what is finite alike, whatever those that do not see them have beside them in a tile."""
    from _paged_ref import attend_ref
    from nanokv_amd.paged import attend_paged, tree_masks
    g = torch.Generator().manual_seed(n)
    cache, tables, lens = _setup([older + n, n, older // 2 + n], hkv, 16, d, "bf16", seed=n)
    tables = torch.nn.functional.pad(tables, (0, wide // 16), value=-1)
    for b in range(3):
        first = int(lens[b]) - n
        for i in {1, 2, n // 2, n - 1} if b < 2 else {n - 2}:
            at = first + i
            dims = torch.randint(0, d, (3,), generator=g)
            for dim, bad in zip(dims.tolist(), (float("nan"), float("inf"), float("-inf"))):
                cache.v[int(tables[b, at // 16]), :, at % 16, dim] = bad
    masks = None
    if tree:
        parents = torch.tensor([-1] + [int(torch.randint(-1, i, (1,), generator=g)) for i in range(1, n)])
        masks = tree_masks(parents.cuda()).repeat(3)
    q = _q(3 * n, hq, d, 3, scale=0.7)
    got = attend_paged(q, cache, tables, lens, tree=masks)
    ref, mag = attend_ref(q, cache, tables, lens, tree=masks, n_each=n)
    fine = ref.isfinite()
    assert bool(fine.any()) and not bool(fine.all())
    got = got.double().cpu()
    same = (got == ref) | (got.isnan() & ref.isnan())
    assert bool(same[~fine].all()), (got[~fine][~same[~fine]][:4], ref[~fine][~same[~fine]][:4])
    many = n * hq // hkv > 16
    c = 2.0 ** -13 + (2.02 * 2.0 ** -8 if many else 0.0)      # (logits below 20 and 2000 keys: 2 e + 2 n u < 2^-13)
    tol = 2.0 ** -8 * (ref.abs() + c * mag) + c * mag
    assert bool(((got - ref).abs() <= tol)[fine].all())


@pytest.mark.parametrize("kv,B,n,older", [("bf16", 1, 512, 1536), ("bf16", 4, 1, 16384), ("bf16", 2, 4, 8192),
                                          ("int8", 2, 4, 8192), ("int8", 4, 1, 16384)])
def test_values_that_are_not_finite_take_no_longer(kv, B, n, older):
    """A NaN value that some queries see: the call takes the time of one without, or little more."""
    from nanokv_amd.paged import attend_paged
    cache, tables, lens = _setup([older + n] * B, 8, 64, 128, kv, seed=1, poison=False)
    q = _q(B * n, 32, 128, 3)

    def us():
        times = []
        for _ in range(8):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(4):
                attend_paged(q, cache, tables, lens)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b) * 250)
        return min(times)

    clean = us()
    for at in (older + n // 2, older // 2):
        if kv == "bf16":
            cache.v[int(tables[0, at // 64]), :, at % 64, 3] = float("nan")
        else:
            cache.v_scale[int(tables[0, at // 64]), :, at % 64] = float("nan")
        assert us() < 3 * clean + 50


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,hq,hkv,page,tree", [(26, 4, 2, 64, True), (9, 5, 1, 16, True), (33, 2, 2, 256, False),
                                                (26, 8, 2, 16, True), (64, 5, 1, 64, True), (150, 8, 2, 64, False)])
def test_shared_lists_of_every_kind(kv, d, n, hq, hkv, page, tree):
    """Tiles of 64 and of 128 columns, shared and cut over workgroups, in both formats: trees and short chunks
    behind a few thousand keys."""
    from nanokv_amd import _lib
    from nanokv_amd.paged import attend_paged, tree_masks
    older = [3000, 0, 2111]
    lengths = [o + n for o in older]
    cache, tables, lens = _setup(lengths, hkv, page, d, kv, seed=n)
    rows = n * (hq // hkv)
    assert rows > 16
    most = tables.shape[1]
    assert _lib.load().nkv_paged_attend_workspace(3, 3 * n, n, hq, hkv, d, most, page, 0) > 0      # (the list is shared)
    masks = None
    if tree:
        g = torch.Generator().manual_seed(n)
        parents = [torch.tensor([-1] + [int(torch.randint(-1, i, (1,), generator=g)) for i in range(1, n)]) for _ in range(3)]
        masks = tree_masks(torch.stack(parents).cuda()).flatten()
    q = _q(3 * n, hq, d, n)
    want = attend_paged(q, cache, tables, lens, tree=masks)
    _check(want, q, cache, tables, lens, tree=masks, n_each=n)
    starts = torch.tensor([3, n + 3, n + 3, 2 * n + 1], dtype=torch.int32, device="cuda")
    q = _q(2 * n + 5, hq, d, n + 1)
    masks = None if masks is None else masks[:2 * n + 5].contiguous()
    got = attend_paged(q, cache, tables, lens, starts=starts, max_new=n, tree=masks)
    _check(got, q, cache, tables, lens, starts, tree=masks)


@pytest.mark.parametrize("n,older", [(1, 70), (3, 500), (20, 70), (24, 3000)])
@pytest.mark.parametrize("which,bad", [(2, float("nan")), (3, float("nan")), (3, float("inf"))])
def test_scales_that_are_not_finite(n, older, which, bad):
    """A scale of a seen and of a drafted row of an 8-bit cache, of its key or of its value: the outputs are the
    formula's (infinity times a code: infinite, or NaN for 0), those that do not see the row have none of it.
    (Infinite scales of keys lie outside what a cache holds: their logits are infinite where those of infinite
    keys would be NaN.)"""
    from _paged_ref import attend_ref
    from nanokv_amd.paged import attend_paged
    cache, tables, lens = _setup([older + n, older + n], 2, 16, 128, "int8", seed=n)
    cache[which][int(tables[0, 2]), :, 5] = bad                                    # key 37 of the first sequence
    at = older + n // 2
    cache[which][int(tables[1, at // 16]), :, at % 16] = bad                       # a new token of the second
    q = _q(2 * n, 8, 128, 5, scale=0.1)
    got = attend_paged(q, cache, tables, lens).double().cpu()
    ref, mag = attend_ref(q, cache, tables, lens, n_each=n)
    fine = ref.isfinite()
    assert bool(((got == ref) | (got.isnan() & ref.isnan()))[~fine].all())
    c = 2.0 ** -13 + (2.02 * 2.0 ** -8 if 4 * n > 16 else 0.0)
    assert bool(((got - ref).abs() <= 2.0 ** -8 * (ref.abs() + c * mag) + c * mag)[fine].all())
