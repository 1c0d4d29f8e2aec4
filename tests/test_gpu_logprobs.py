"""token_logprobs against its definition in 64 bits.

Tolerances, u = 2^-24: an element's y = m - x is off by u y, its exponent's
argument by 3 u y, and exp2 by 2^-22 relative; a lane adds up to vocab / 256 + 16 of them in a
chain, and lanes, wavefronts, pieces and moves of the maximum join in at most 64 steps of 4 u.
So with n = vocab / 256 + 16 + 256 roundings, s = sum of e^-y and w = sum of y e^-y
(the maximum left out), w2 = sum of y^2 e^-y:
  ds = (n u + 2^-22) s + 4 u w,  dw = (n u + 2^-21) w + 4 u w2;
(an exponential below the normal range, y > 87, may be 0: what such terms add up to
joins ds and dw in full: e^-87.3365 = 2^-126, the smallest that exp2 gives);
log p is off by ds / (1 + s) + 4 u (|log p| + 1), the entropy by
ds / (1 + s) + (dw + w ds) / (1 + s) + 8 u (H + tiny).
"""

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _check(x, tokens, top, got):
    """x [rows, vocab] as the kernel reads it."""
    rows, vocab = x.shape
    xd = x.double()
    m = xd.amax(1, keepdim=True)
    y = (m - xd).clamp(max=800.0)
    e = torch.exp(-y)
    one = torch.zeros_like(e, dtype=torch.bool).scatter_(1, xd.argmax(1, keepdim=True), True)
    e = e.masked_fill(one, 0.0)
    s, w, w2 = e.sum(1), (y * e).sum(1), (y * y * e).sum(1)
    n = vocab / 256 + 16 + 256
    ds, dw = (n * U + 2.0 ** -22) * s + 4 * U * w, (n * U + 2.0 ** -21) * w + 4 * U * w2
    small = y > 87
    ds, dw = ds + (e * small).sum(1), dw + (y * e * small).sum(1)
    z = torch.log1p(s)

    def close(a, ref, tol):
        ok = (a.double() - ref).abs() <= tol
        ok |= (ref == float("-inf")) & (a == float("-inf"))
        assert bool(ok.all()), (a[~ok][:4], ref[~ok][:4])

    inside = (tokens >= 0) & (tokens < vocab)
    lp = xd.gather(1, tokens.clamp(0, vocab - 1)[:, None])[:, 0] - m[:, 0] - z
    assert bool(got.logprob[~inside].isnan().all())
    close(got.logprob[inside], lp[inside], (ds / (1 + s) + 4 * U * (lp.abs() + 1))[inside])
    h = z + w / (1 + s)
    close(got.entropy, h, ds / (1 + s) + (dw + w * ds) / (1 + s) + 8 * U * h + 1e-37)
    assert got.top_ids.shape == (rows, top) and got.top_logprobs.shape == (rows, top)
    best = torch.sort(x.float(), dim=1, descending=True, stable=True)
    assert torch.equal(got.top_ids, best.indices[:, :top])
    lp = best.values[:, :top].double() - m - z[:, None]
    close(got.top_logprobs, lp, (ds / (1 + s))[:, None] + 4 * U * (lp.abs() + 1))


def _logits(rows, vocab, dtype, seed, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (2, 7, 0), (1, 63, 63), (5, 64, 64), (4, 1000, 20),
                                            (1, 4095, 5), (2, 4097, 64), (1, 32003, 20), (7, 151936, 20),
                                            (1, 151936, 64), (1030, 2049, 5), (1, 400001, 3)])
def test_rows(dtype, rows, vocab, top):
    from nanokv_amd.logprobs import token_logprobs
    x = _logits(rows, vocab, dtype, vocab + top)
    tokens = torch.randint(0, vocab, (rows,), device="cuda")
    tokens[rows // 2] = x[rows // 2].argmax()
    _check(x, tokens, top, token_logprobs(x, tokens, top))


@pytest.mark.parametrize("vocab", [300, 20011, 151936])
def test_confident_rows_keep_their_digits(vocab):
    """One token far above the others: entropies and log probabilities far below fp32's step of 1."""
    from nanokv_amd.logprobs import token_logprobs
    x = _logits(6, vocab, torch.float32, 1, scale=0.5)
    for i, up in enumerate((5.0, 20.0, 30.0, 40.0, 60.0, 90.0)):
        x[i, (i * 71) % vocab] = up
    tokens = (torch.arange(6, device="cuda") * 71) % vocab
    got = token_logprobs(x, tokens, 4)
    _check(x, tokens, 4, got)
    # (the last row's e^-90 lies below the normal range: 0)
    assert bool((got.logprob[1:5] < 0).all()) and bool((got.entropy[:5] > 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [130, 6000, 100000])
def test_ties_and_orders(dtype, vocab):
    """Equal logits go by their ids; rows in order make every element a candidate."""
    from nanokv_amd.logprobs import token_logprobs
    g = torch.Generator(device="cuda").manual_seed(3)
    ramp = torch.linspace(-8, 8, vocab, device="cuda")
    x = torch.stack([torch.zeros(vocab, device="cuda"), torch.randint(0, 3, (vocab,), generator=g, device="cuda") * 0.5,
                     ramp, ramp.flip(0), (torch.arange(vocab, device="cuda") % 97).float() / 16,
                     torch.where(torch.arange(vocab, device="cuda") % 2 == 0, 0.0, -0.0)]).to(dtype)
    tokens = torch.randint(0, vocab, (6,), generator=g, device="cuda")
    for top in (1, 20, 64):
        _check(x, tokens, top, token_logprobs(x, tokens, top))


@pytest.mark.parametrize("vocab", [200, 40000, 151936])
def test_tokens_that_are_not_allowed(vocab):
    from nanokv_amd.logprobs import token_logprobs
    x = _logits(5, vocab, torch.bfloat16, 8)
    x[:, torch.rand(vocab, device="cuda") < 0.5] = float("-inf")
    x[1] = float("-inf")
    x[1, 5] = -3.0                                    # one token is left
    x[2] = float("-inf")
    x[2, [3, 150, vocab - 1]] = 2.0                   # fewer than the alternatives
    x[3] = torch.finfo(torch.bfloat16).min            # masked with the type's lowest value
    x[3, 17] = 0.0
    x[4, ::2] = torch.finfo(torch.bfloat16).min
    tokens = torch.tensor([0, 5, 4, 17, vocab - 1], device="cuda")
    _check(x, tokens, 20, token_logprobs(x, tokens, 20))


@pytest.mark.parametrize("vocab", [50, 30000])
def test_rows_without_a_distribution(vocab):
    """All -inf, NaN or +inf: every number is NaN, the order of the logits stays (NaN first)."""
    from nanokv_amd.logprobs import token_logprobs
    x = _logits(5, vocab, torch.float32, 2)
    x[0] = float("-inf")
    x[1, 33] = float("nan")
    x[2, [7, 40]] = float("inf")
    x[3] = float("nan")
    x[4, [2, 49]] = torch.tensor([float("inf"), float("nan")], device="cuda")
    tokens = torch.tensor([3, 4, 7, 9, 11], device="cuda")
    got = token_logprobs(x, tokens, 12)
    for t in (got.logprob, got.entropy, got.top_logprobs):
        assert bool(t.isnan().all())
    assert torch.equal(got.top_ids, torch.sort(x, dim=1, descending=True, stable=True).indices[:, :12])
    one = torch.zeros(1, 40, device="cuda")
    one[0, 3] = float("inf")                          # a single +inf
    got = token_logprobs(one, torch.tensor([3], device="cuda"), 2)
    assert bool(got.logprob.isnan().all()) and got.top_ids.tolist() == [[3, 0]]


def test_rows_in_place_shapes_and_tokens():
    from nanokv_amd.logprobs import token_logprobs
    wide = _logits(9, 5003, torch.bfloat16, 4)
    x = wide[1::2, 3:4999]                            # rows apart, off the 16-byte boundaries
    tokens = torch.tensor([-1, 0, 4995, 4996], device="cuda")
    _check(x, tokens, 6, token_logprobs(x, tokens.int(), 6))
    t = token_logprobs(x.t()[:1000].t().unsqueeze(0), tokens[None], 3)
    assert t.logprob.shape == (1, 4) and t.top_ids.shape == (1, 4, 3)
    one = token_logprobs(wide[0], torch.tensor(7, device="cuda"))
    assert one.logprob.shape == () and one.top_ids.shape == (0,)
    assert torch.equal(one.logprob, token_logprobs(wide[:1], torch.tensor([7], device="cuda")).logprob[0])
    none = token_logprobs(wide[:0], tokens[:0], 2)
    assert none.logprob.shape == (0,) and none.top_ids.shape == (0, 2)
    same = wide[:1].expand(6, -1)
    got = token_logprobs(same, torch.full((6,), 7, device="cuda"), 1)
    assert torch.equal(got.logprob, one.logprob.expand(6)) and torch.equal(got.entropy, got.entropy[:1].expand(6))


def test_streams_and_graphs():
    """Two captured calls replayed in turn, on other logits, between eager work."""
    from nanokv_amd.logprobs import token_logprobs
    x = _logits(2, 151936, torch.float32, 5)
    tokens = torch.tensor([1, 2], device="cuda")
    token_logprobs(x, tokens, 20)
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = token_logprobs(x, tokens, 20)
        graphs.append((g, out))
    for step in range(4):
        x.copy_(_logits(2, 151936, torch.float32, 10 + step))
        tokens.add_(11)
        eager = token_logprobs(x, tokens, 20)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beside = token_logprobs(x, tokens, 20)
        torch.cuda.current_stream().wait_stream(side)
        for g, out in graphs:
            g.replay()
            for a, b, c in zip(out, eager, beside):
                assert torch.equal(a, b) and torch.equal(a, c)
