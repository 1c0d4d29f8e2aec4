"""attend_paged against softmax(scale q k^T) v in 64 bits, hidden keys left out.

Tolerances, u = 2^-24, A = scale * max |q| * max |k| (so that sum |q_i k_i| scale <= A):
a logit is a sum of D <= 128 products, off by (D + 3) u A (codes: one scale more, u A);
its weight's exponent is off by that and 2 u A, exp2 by 2^-22: relative error of a weight
e = (D + 8) u A + 2^-22.  Weights and their sum (of n keys: n u, and 64 joins) are both off by e, so the
output by (2 e + 2 n u + 2^-16) of sum p |v|, P's high and low bf16 parts (2^-16) and V's scale included.
The kernel of many columns rounds P to bf16: 2^-8 of numerator and denominator each.
Then one rounding to bf16, 2^-8 |ref|.
"""

import pytest
import torch

from _paged_ref import attend_ref, held, make_cache

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _check(got, q, cache, tables, lengths, starts=None, tree=None, scale=None, n_each=1, many=None):
    ref, mag = attend_ref(q, cache, tables, lengths, starts, tree, scale, n_each)
    T, hq, d = q.shape
    hkv = cache.k.shape[1]
    kmax = held(cache, 0).nan_to_num(0, 0, 0).norm(dim=-1).max()
    a = float((d ** -0.5 if scale is None else scale) * q.double().nan_to_num(0, 0, 0).norm(dim=-1).max() * kmax)
    c = 2 * ((d + 8) * U * a + 2.0 ** -22) + 2 * (int(lengths.max()) + 64) * U + 2.0 ** -16
    if many is None:
        counts = torch.full((1,), n_each) if starts is None else starts[1:] - starts[:-1]
        many = int(counts.max()) * (hq // hkv) > 16
    c += 2.02 * 2.0 ** -8 if many else 0.0
    err = (got.double().cpu() - ref).abs()
    bad = ~(err <= 2.0 ** -8 * (ref.abs() + c * mag) + c * mag + 1e-37)
    assert not bool(bad.any()), (int(bad.sum()), float(err.nan_to_num(1e9).max()), bad.nonzero()[:4].tolist())


def _tables(lengths, page, pages, seed=0, spare=1):
    """Page tables of distinct pages in no order; what lies behind a sequence's last page is no page."""
    g = torch.Generator().manual_seed(seed)
    most = max(1, max(-(-n // page) for n in lengths)) + spare
    order = torch.randperm(pages, generator=g).tolist()
    t = torch.full((len(lengths), most), -1, dtype=torch.int32)
    for b, n in enumerate(lengths):
        for j in range(-(-n // page)):
            t[b, j] = order.pop()
    return t.cuda()


def _setup(lengths, hkv, page, d, kv, seed=0, poison=True, pages=None):
    """A cache whose unused slots hold NaN (scales, in 8 bits), its tables and lengths."""
    pages = pages or sum(-(-n // page) for n in lengths) + 3
    cache = make_cache(pages, hkv, page, d, kv, "cuda", seed)
    tables = _tables(lengths, page, pages, seed)
    if poison:
        used = torch.zeros(pages, page, dtype=torch.bool)
        for b, n in enumerate(lengths):
            for j in range(n):
                used[int(tables[b, j // page]), j % page] = True
        free = (~used).cuda()
        for t in (cache[:2] if kv == "bf16" else cache[2:]):
            t.transpose(1, 2)[free] = float("nan")
    return cache, tables, torch.tensor(lengths, dtype=torch.int32, device="cuda")


def _q(T, hq, d, seed, scale=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(T, hq, d, generator=g, device="cuda") * scale).bfloat16()


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (8, 8, 64), (5, 1, 128), (16, 1, 64), (2, 1, 128), (14, 2, 64),
                                      (32, 1, 128), (64, 1, 64), (24, 8, 128)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_one_token(kv, hq, hkv, d, page):
    from nanokv_amd.paged import attend_paged
    lengths = [1, 0, 16, 17, 63, 64, 65, 300, 129, 2]
    cache, tables, lens = _setup(lengths, hkv, page, d, kv, seed=hq)
    q = _q(len(lengths), hq, d, page)
    got = attend_paged(q, cache, tables, lens)
    _check(got, q, cache, tables, lens)
    assert bool((got[1] == 0).all())


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("lengths,hq,hkv,d,page", [([20001], 4, 1, 128, 64), ([5000, 3, 12345], 8, 2, 64, 16),
                                                   ([4096] * 4, 8, 8, 128, 128), ([70000], 2, 2, 64, 4096)])
def test_long_caches_in_runs(kv, lengths, hq, hkv, d, page):
    from nanokv_amd.paged import attend_paged
    cache, tables, lens = _setup(lengths, hkv, page, d, kv, seed=3, poison=False)
    q = _q(len(lengths), hq, d, 1)
    _check(attend_paged(q, cache, tables, lens), q, cache, tables, lens)


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("each,hq,hkv,d", [(2, 8, 2, 128), (4, 4, 1, 64), (3, 10, 2, 128), (5, 4, 1, 128), (16, 4, 1, 64),
                                           (17, 8, 2, 128), (13, 5, 1, 64), (33, 8, 2, 128), (64, 7, 1, 64), (1, 8, 2, 64)])
def test_drafts_in_order(kv, each, hq, hkv, d):
    """Several new tokens of every sequence, some of more than its keys: the first rows see nothing."""
    from nanokv_amd.paged import attend_paged
    lengths = [each, 1, 0, 200 + each, 64 + each // 2]
    cache, tables, lens = _setup(lengths, hkv, 16, d, kv, seed=each)
    q = _q(each * len(lengths), hq, d, each)
    _check(attend_paged(q, cache, tables, lens), q, cache, tables, lens, n_each=each)


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("counts,older,hq,hkv,d,page", [
    ([130, 1, 0, 57, 300], [0, 500, 40, 64, 3], 8, 2, 128, 64), ([1, 2, 3], [100, 0, 7], 4, 1, 64, 16),
    ([257], [1000], 6, 2, 128, 32), ([40, 3], [0, 2000], 16, 1, 64, 16), ([90, 20], [10, 0], 5, 1, 128, 128),
    ([33], [0], 64, 1, 128, 16), ([700, 650], [0, 0], 4, 4, 64, 256)])
@pytest.mark.parametrize("padding", [0, 5])
def test_ragged_prompts(kv, counts, older, hq, hkv, d, page, padding):
    """Prompts and their next chunks; rows of no sequence and rows behind max_new are 0."""
    from nanokv_amd.paged import attend_paged
    cache, tables, lens = _setup([c + o for c, o in zip(counts, older)], hkv, page, d, kv, seed=sum(counts))
    starts = [padding]
    for c in counts:
        starts.append(starts[-1] + c)
    starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
    q = _q(int(starts[-1]) + 2 * padding, hq, d, 5)
    torch.full((1 << 22,), float("nan"), device="cuda")          # what new memory may hold
    got = attend_paged(q, cache, tables, lens, starts=starts, max_new=max(counts))
    _check(got, q, cache, tables, lens, starts)
    loose = attend_paged(q, cache, tables, lens, starts=starts)
    _check(loose, q, cache, tables, lens, starts, many=True)
    short = max(1, max(counts) // 3)
    less = attend_paged(q, cache, tables, lens, starts=starts, max_new=short)
    keep = torch.zeros(len(q), dtype=torch.bool)
    for b, c in enumerate(counts):
        keep[int(starts[b]):int(starts[b]) + min(c, short)] = True
    assert bool((less[~keep.cuda()] == 0).all())
    _check(torch.where(keep.cuda()[:, None, None], less, got), q, cache, tables, lens, starts, many=True)


def _random_tree(n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.tensor([int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for i in range(n)])


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("n,older,hq,hkv,d", [(1, 50, 4, 1, 128), (3, 29, 4, 1, 64), (4, 0, 8, 2, 128), (16, 48, 1, 1, 64),
                                              (26, 1000, 32, 8, 128), (64, 63, 4, 1, 128), (64, 5000, 8, 1, 64),
                                              (33, 7, 10, 2, 128)])
def test_trees(kv, n, older, hq, hkv, d):
    from nanokv_amd.paged import attend_paged, tree_masks
    lengths = [older + n, n, older // 2 + n]
    cache, tables, lens = _setup(lengths, hkv, 32, d, kv, seed=n)
    masks = tree_masks(torch.stack([_random_tree(n, i) for i in range(3)]).cuda()).flatten()
    q = _q(3 * n, hq, d, n)
    _check(attend_paged(q, cache, tables, lens, tree=masks), q, cache, tables, lens, tree=masks, n_each=n)
    # masks of any bits: nothing of the tree, all of it and past its end, not itself
    masks[::3], masks[1::3] = 0, -1
    if n > 2:
        masks[2::3] ^= 1
    got = attend_paged(q, cache, tables, lens, tree=masks)
    _check(got, q, cache, tables, lens, tree=masks, n_each=n)
    assert bool((got[n] == 0).all()) or bool(masks[n] != 0)
    starts = torch.tensor([0, n, n, 2 * n], dtype=torch.int32, device="cuda")
    got = attend_paged(q, cache, tables, lens, starts=starts, max_new=n, tree=masks)
    _check(got, q, cache, tables, lens, starts, tree=masks)


@pytest.mark.parametrize("n", [1, 3, 30])
def test_a_tree_of_a_line_is_a_draft_in_order(n):
    from nanokv_amd.paged import attend_paged, tree_masks
    cache, tables, lens = _setup([300, 40, n], 2, 16, 128, "bf16")
    q = _q(3 * n, 8, 128, 0)
    masks = tree_masks(torch.arange(-1, n - 1).cuda()).repeat(3)
    assert torch.equal(attend_paged(q, cache, tables, lens, tree=masks), attend_paged(q, cache, tables, lens))


def test_tree_masks_on_the_gpu():
    from nanokv_amd.paged import tree_masks
    parents = torch.stack([_random_tree(64, i) for i in range(5)])
    masks = tree_masks(parents)
    assert torch.equal(masks, tree_masks(parents.int().cuda()).cpu())
    for row, m in zip(parents.tolist(), masks.tolist()):
        for i in range(64):
            want, j = 0, i
            while j >= 0:
                want, j = want | 1 << j, row[j]
            assert m[i] & ((1 << 64) - 1) == want


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("n,hq,hkv,d,older", [(3, 4, 1, 128, 70), (12, 8, 2, 64, 0), (40, 4, 2, 128, 5000), (6, 2, 1, 64, 3000)])
def test_what_hidden_keys_hold_reaches_no_output(bad, n, hq, hkv, d, older):
    """A drafted token of NaN or infinite values: those that see it are NaN, the others as ever."""
    from nanokv_amd.paged import attend_paged, tree_masks
    parents = torch.tensor([-1, -1] + [int(i % 2) for i in range(n - 2)])
    masks = tree_masks(parents.cuda()).repeat(2)
    cache, tables, lens = _setup([older + n, n + 1], hkv, 16, d, "bf16", seed=2)
    q = _q(2 * n, hq, d, 3)
    for b in range(2):
        at = int(lens[b]) - n + 1                         # token 1: hidden from token 0 and its line
        cache.v[int(tables[b, at // 16]), :, at % 16, 3::5] = bad
        cache.k[int(tables[b, at // 16]), :, at % 16, 1] = bad
    sees = ((masks >> 1) & 1).bool()
    got = attend_paged(q, cache, tables, lens, tree=masks)
    assert bool(got[~sees].isfinite().all())
    ref, _ = attend_ref(q, cache, tables, lens, tree=masks, n_each=n)
    clean = ref[~sees.cpu()]
    assert bool(clean.isfinite().all())
    tol = 2.0 ** -8 * clean.abs() + 2.0 ** -6 * clean.abs().amax()      # (its exactness is test_trees')
    assert bool(((got[~sees].double().cpu() - clean).abs() <= tol).all())
    if bad != bad:
        assert bool(got[sees].isnan().all())
    # in order: tokens before it are clean
    line = attend_paged(q, cache, tables, lens)
    assert bool(line.view(2, n, hq, d)[:, 0].isfinite().all())


@pytest.mark.parametrize("n", [1, 30])
def test_values_at_the_end_of_the_range(n):
    """Infinite values that are seen: the output's infinity and NaN are the formula's."""
    from nanokv_amd.paged import attend_paged
    cache, tables, lens = _setup([100 + n], 1, 16, 64, "bf16", poison=False)
    q = _q(n, 4, 64, 1)
    cache.v[int(tables[0, 2]), 0, 5, 7] = float("inf")
    cache.v[int(tables[0, 2]), 0, 6, 8] = float("nan")
    got = attend_paged(q, cache, tables, lens)
    assert bool((got[..., 7] == float("inf")).all()) and bool(got[..., 8].isnan().all())
    rest = [i for i in range(64) if i not in (7, 8)]
    assert bool(got[..., rest].isfinite().all())


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("n", [1, 20])
def test_pages_outside_the_cache_hide_their_keys(kv, n):
    from nanokv_amd.paged import attend_paged
    cache, tables, lens = _setup([500, 300, 90], 2, 16, 128, kv, seed=4)
    tables[0, 3], tables[0, 7], tables[1, 0], tables[1, 1] = -1, 2 ** 31 - 1, cache.k.shape[0], -2 ** 31
    tables[2] = -7
    q = _q(3 * n, 8, 128, 2)
    got = attend_paged(q, cache, tables, lens)
    _check(got, q, cache, tables, lens, n_each=n)
    assert bool((got[2 * n:] == 0).all())


@pytest.mark.parametrize("n", [1, 40])
def test_lengths_outside_the_table(n):
    """A length past the table counts up to its end, a negative one as 0."""
    from nanokv_amd.paged import attend_paged
    cache, tables, lens = _setup([160, 160], 2, 16, 64, "bf16", seed=1, poison=False)
    tables = tables[:, :10].contiguous()
    q = _q(2 * n, 4, 64, 2)
    full = attend_paged(q, cache, tables, lens)
    got = attend_paged(q, cache, tables, torch.tensor([161, -1], dtype=torch.int32, device="cuda"))
    assert torch.equal(got[:n], full[:n]) and bool((got[n:] == 0).all())
    got = attend_paged(q, cache, tables, torch.tensor([2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda"))
    assert torch.equal(got[:n], full[:n]) and bool((got[n:] == 0).all())


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("n", [1, 35])
def test_other_orders_in_memory_and_scales_of_logits(kv, n):
    """Caches [pages, page, Hkv, D], rows of q and tables that lie apart, int64 lengths; scale."""
    from nanokv_amd.paged import PagedKV, attend_paged
    cache, tables, lens = _setup([300, 77], 4, 32, 128, kv, seed=6)
    k, v = (torch.empty(cache.k.shape[0], 32, 4, 128, dtype=cache.k.dtype, device="cuda").transpose(1, 2) for _ in range(2))
    other = PagedKV(k.copy_(cache.k), v.copy_(cache.v), cache.k_scale, cache.v_scale)
    wide = _q(2 * n, 3 * 8, 128, 3)
    q = wide[:, 8:16]
    table = torch.stack([tables, tables + 5], 1)[:, 0]
    for scale in (0.02, 0.3):
        want = attend_paged(q.contiguous(), cache, tables, lens, scale=scale)
        _check(want, q.contiguous(), cache, tables, lens, scale=scale, n_each=n)
        assert torch.equal(attend_paged(q, other, table, lens.long(), scale=scale), want)
        assert torch.equal(attend_paged(q.transpose(1, 2).contiguous().transpose(1, 2), other, tables.long(), lens, scale=scale), want)


def test_sequences_may_share_pages():
    from nanokv_amd.paged import attend_paged
    cache, tables, _ = _setup([400], 2, 16, 128, "bf16", poison=False)
    q = _q(3, 8, 128, 0)
    shared = tables.expand(3, -1)
    lens = torch.tensor([400, 100, 400], dtype=torch.int32, device="cuda")
    _check(attend_paged(q, cache, shared, lens), q, cache, shared, lens)


@pytest.mark.parametrize("n", [1, 24])
def test_streams_and_graphs(n):
    """Two captured calls replayed in turn with other lengths and queries, and calls on a second stream."""
    from nanokv_amd.paged import attend_paged
    cache, tables, lens = _setup([9000, 400, 3000], 2, 64, 128, "bf16", poison=False)
    q = _q(3 * n, 8, 128, 0)
    attend_paged(q, cache, tables, lens)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = attend_paged(q, cache, tables, lens)
        graphs.append((g, out))
    side = torch.cuda.Stream()
    for step in range(4):
        lens.copy_(torch.tensor([[9000, 64, 1], [1, 400, 3000], [5, 5, 5], [8999, 0, 2999]][step]))
        q.copy_(_q(3 * n, 8, 128, step))
        want = attend_paged(q, cache, tables, lens)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beside = attend_paged(q, cache, tables, lens)
        torch.cuda.current_stream().wait_stream(side)
        for g, out in graphs:
            g.replay()
            assert torch.equal(out, want) and torch.equal(beside, want)
        if step < 2:
            _check(want, q, cache, tables, lens, n_each=n)


def test_no_rows_and_no_sequences():
    from nanokv_amd.paged import attend_paged
    cache, tables, lens = _setup([10], 1, 16, 64, "bf16")
    none = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    assert attend_paged(none, cache, tables, lens).shape == (0, 4, 64)
    assert attend_paged(none, cache, tables[:0], lens[:0]).shape == (0, 4, 64)
    q = _q(2, 4, 64, 0)
    got = attend_paged(q, cache, tables[:0], lens[:0], starts=torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert bool((got == 0).all())
    got = attend_paged(q, cache, tables, lens, starts=torch.tensor([2, 2], dtype=torch.int32, device="cuda"))
    assert bool((got == 0).all())


def test_far_offsets_in_a_cache_past_32_bits():
    """Pages whose elements and bytes lie past 2^31 and 2^32 from the cache's start."""
    from nanokv_amd.paged import PagedKV, append_paged, attend_paged, read_paged
    pages, hkv, page, d = 40000, 8, 64, 128             # 5.2 GB of keys
    k = torch.zeros(pages, hkv, page, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    cache = PagedKV(k, v)
    far = [pages - 1, 33000, 16500, 2]
    g = torch.Generator(device="cuda").manual_seed(0)
    kn, vn = (torch.randn(200, hkv, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    at = torch.arange(200, device="cuda")
    slots = torch.tensor(far, device="cuda")[at // page] * page + at % page
    append_paged(cache, kn, vn, slots)
    assert all(torch.equal(a, b) for a, b in zip(read_paged(cache, slots), (kn, vn)))
    small = PagedKV(k[torch.tensor(far, device="cuda")].contiguous(), v[torch.tensor(far, device="cuda")].contiguous())
    lens = torch.tensor([200], dtype=torch.int32, device="cuda")
    for n in (1, 30):
        q = _q(n, 32, d, n)
        a = attend_paged(q, cache, torch.tensor([far], dtype=torch.int32, device="cuda"), lens)
        b = attend_paged(q, small, torch.arange(4, dtype=torch.int32, device="cuda")[None], lens)
        assert torch.equal(a, b)


@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_more_sequences_than_lanes(kv):
    """A token of each of 150 sequences, some empty, some of no new token."""
    from nanokv_amd.paged import attend_paged
    lengths = [(37 * b) % 230 for b in range(150)]
    cache, tables, lens = _setup(lengths, 2, 16, 64, kv, seed=5)
    q = _q(150, 4, 64, 9)
    _check(attend_paged(q, cache, tables, lens), q, cache, tables, lens)
    counts = [0] * 70 + [b % 3 for b in range(80)]                     # (the first 64 hold no query)
    starts = torch.tensor([0] + counts).cumsum(0).int().cuda()
    n = int(starts[-1])
    got = attend_paged(q[:n], cache, tables, lens, starts=starts, max_new=2)
    _check(got, q[:n], cache, tables, lens, starts)


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("cap", [300, 4608])
def test_more_query_tiles_than_lanes(kv, cap):
    """100 sequences of up to 20 new tokens under tables of `cap` tokens: a workgroup a unit, or a shared list."""
    from nanokv_amd.paged import attend_paged
    lengths = [20 + (53 * b) % 200 for b in range(100)]
    cache, tables, lens = _setup(lengths, 1, 16, 64, kv, seed=6)
    tables = torch.nn.functional.pad(tables, (0, max(0, cap // 16 - tables.shape[1])), value=-1)
    q = _q(2000, 4, 64, 10)
    _check(attend_paged(q, cache, tables, lens), q, cache, tables, lens, n_each=20)
    counts = [0] * 66 + [(7 * b) % 21 for b in range(34)]
    starts = torch.tensor([0] + counts).cumsum(0).int().cuda()
    n = int(starts[-1])
    got = attend_paged(q[:n], cache, tables, lens, starts=starts, max_new=20)
    _check(got, q[:n], cache, tables, lens, starts, many=True)


def test_nan_keys_make_nan_outputs():
    """A NaN key that a query sees: its output is NaN, other queries' are not."""
    from nanokv_amd.paged import attend_paged
    cache, tables, lens = _setup([200, 200], 1, 16, 64, "bf16", seed=7)
    cache.k[int(tables[0, 3]), 0, 5] = float("nan")                     # key 53 of the first sequence
    for each in (1, 40):
        got = attend_paged(_q(2 * each, 4, 64, 11), cache, tables, lens)
        assert bool(got[:each].isnan().all()) and not bool(got[each:].isnan().any())


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("n", [3, 40])
def test_trees_longer_than_their_sequences_or_than_max_new(kv, n):
    """Sequences that hold fewer keys than their trees have tokens (the first ones lie before key 0), and
    trees cut off at max_new: their rows behind it are 0."""
    from nanokv_amd.paged import attend_paged, tree_masks
    cache, tables, lens = _setup([n, n - 2, 0, 1, 70], 2, 16, 128, kv, seed=n)
    masks = tree_masks(torch.stack([_random_tree(n, i) for i in range(5)]).cuda()).flatten()
    q = _q(5 * n, 8, 128, n)
    _check(attend_paged(q, cache, tables, lens, tree=masks), q, cache, tables, lens, tree=masks, n_each=n)
    starts = torch.arange(0, 5 * n + 1, n, dtype=torch.int32, device="cuda")
    got = attend_paged(q, cache, tables, lens, starts=starts, max_new=n - 1, tree=masks)
    kept = torch.arange(5 * n, device="cuda") % n != n - 1
    want = attend_paged(q, cache, tables, lens, starts=starts, max_new=n, tree=masks)
    assert torch.equal(got[kept], want[kept]) and bool((got[~kept] == 0).all())


@pytest.mark.parametrize("n,older", [(1, 70), (5, 9000), (40, 70), (33, 9000)])
def test_infinite_values_that_a_query_sees(n, older):
    """A value of +inf in one dim: +inf there for the queries that see it, the others as without it."""
    from nanokv_amd.paged import attend_paged
    cache, tables, lens = _setup([older + n], 1, 16, 128, "bf16", seed=n)
    q = _q(n, 4, 128, 5, scale=0.5)
    at = older + n // 2
    want = attend_paged(q, cache, tables, lens)
    cache.v[int(tables[0, at // 16]), 0, at % 16, 7] = float("inf")
    got = attend_paged(q, cache, tables, lens)
    sees = torch.arange(n, device="cuda") >= n // 2
    assert bool((got[sees, :, 7] == float("inf")).all())
    got[sees, :, 7] = want[sees, :, 7]
    # a column computed again has other roundings: each result is off by at most (1 + 2.02) 2^-8 of the largest
    # value (the output's rounding and P's, the tolerance above), so two by twice that
    top = float(cache.v.float().nan_to_num(0, 0, 0).abs().max())
    assert float((got.float() - want.float()).abs().max()) <= 2 * 3.03 * 2.0 ** -8 * top
