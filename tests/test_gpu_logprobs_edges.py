"""token_logprobs of rows whose largest logit, or that of some piece of them, lies far from 0:
masks of large finite values, logits of any size.

The tolerances are those of test_gpu_logprobs: past 2^16 an element's y = m - x is taken
directly, off by u y as they count it."""

import pytest
import torch

from test_gpu_logprobs import _check, _logits

pytestmark = pytest.mark.gpu

MASKS = [-65504.0, -65536.0, -1e9, -2.0 ** 32, -1e10, -1e12, -1e20, -1e30, -5e37, -3e38]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 151936), (6, 9000), (1030, 3001)])
@pytest.mark.parametrize("mask", MASKS)
def test_masks_of_large_finite_values(dtype, rows, vocab, mask):
    """A masked prefix longer than any run, whole masked runs between others, one token left, none masked."""
    from nanokv_amd.logprobs import token_logprobs
    x = _logits(rows, vocab, dtype, 7)
    x[0::4, :vocab * 2 // 3] = mask                    # the first pieces hold nothing else
    keep = x[1::4, vocab // 2 + 1].clone()
    x[1::4] = mask                                     # one token is left
    x[1::4, vocab // 2 + 1] = keep
    x[2::4, torch.arange(vocab, device="cuda") % 2048 >= 100] = mask
    tokens = torch.randint(0, vocab, (rows,), device="cuda")
    tokens[0::4] = vocab - 1                           # one that is allowed
    for top in (0, 5, 64):
        got = token_logprobs(x, tokens, top)
        _check(x, tokens, top, got)
    assert bool(got.logprob.isfinite().all()) and bool(got.entropy.isfinite().all())
    assert bool(got.top_logprobs.isfinite().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [5, 1500, 40000])
@pytest.mark.parametrize("size", [65536.0, 2.0 ** 24, 2.0 ** 32, 1e10, 1e12, 1e30, 5e37, 1.6e38])
def test_logits_of_any_size(dtype, vocab, size):
    """Rows of one value, with a few values a step apart, of both signs; ties of the largest in every run."""
    from nanokv_amd.logprobs import token_logprobs
    g = torch.Generator(device="cuda").manual_seed(vocab)
    step = torch.randint(0, 4, (6, vocab), generator=g, device="cuda").float()
    big = torch.tensor(size, device="cuda")
    ulp = big * torch.finfo(dtype).eps
    x = torch.stack([big.expand(vocab), -big.expand(vocab), big + step[2] * ulp, -big - step[3] * ulp,
                     step[4] * big / 2, (step[5] - 2) * big / 2]).to(dtype)
    tokens = torch.randint(0, vocab, (6,), generator=g, device="cuda")
    for top in (0, 3):
        got = token_logprobs(x, tokens, top)
        finite = x.isfinite().all(1)                   # (three times 1.6e38 is infinite: no distribution)
        assert bool(finite[:4].all()) and bool(got.logprob[~finite].isnan().all())
        got = type(got)(*(t[finite] for t in got))
        _check(x[finite], tokens[finite], top, got)
        assert bool(got.logprob.isfinite().all()) and bool(got.entropy.isfinite().all())


@pytest.mark.parametrize("vocab", [3000, 151936])
def test_the_maximum_moves_between_sizes(vocab):
    """A run's maximum climbs from one size to the next: far below 0, near it, far above."""
    from nanokv_amd.logprobs import token_logprobs
    steps = torch.tensor([-1e37, -1e30, -1e12, -1e10, -70000.0, -60000.0, -5.0, 3.0, 60000.0, 70000.0, 1e10, 1e12, 1e30, 1e37],
                         device="cuda")
    at = torch.arange(vocab, device="cuda")
    up = steps[at * len(steps) // vocab]               # over the row
    fast = steps[(at // 1024) % len(steps)]            # from iteration to iteration
    x = torch.stack([up, up.flip(0), fast, fast.flip(0), torch.where(up < 60000, up, -1e10),
                     torch.where(fast.abs() < 60000, fast, -1e12)])
    tokens = torch.randint(0, vocab, (6,), device="cuda")
    for top in (0, 20):
        _check(x, tokens, top, token_logprobs(x, tokens, top))
