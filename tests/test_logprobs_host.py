"""token_logprobs without a GPU: its formulas, and the calls it refuses."""

import ctypes

import pytest
import torch

from nanokv_amd import _lib
from nanokv_amd.logprobs import token_logprobs


def test_formula():
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(3, 4, 50, generator=g) * 3).bfloat16()
    x[0, 0, :40] = float("-inf")
    x[1, 1] = 2.0
    tokens = torch.randint(0, 50, (3, 4), generator=g)
    tokens[2, 3], tokens[2, 2] = -1, 50
    t = token_logprobs(x, tokens, 5)
    lp = torch.log_softmax(x.double(), -1)
    h = -torch.where(lp > float("-inf"), lp.exp() * lp, 0.0).sum(-1)
    inside = (tokens >= 0) & (tokens < 50)
    # fp32 log_softmax of 50 terms: 60 roundings of 2^-24 relative to values below 50
    assert torch.allclose(t.logprob[inside].double(), lp.gather(-1, tokens.clamp(0, 49)[..., None])[..., 0][inside],
                          atol=60 * 50 * 2.0 ** -24, rtol=0)
    assert bool(t.logprob[~inside].isnan().all()) and torch.allclose(t.entropy.double(), h, atol=2e-4)
    assert t.top_ids[1, 1].tolist() == [0, 1, 2, 3, 4] and t.top_ids.dtype == torch.int64


def test_rows_without_a_distribution():
    x = torch.zeros(3, 8)
    x[0] = float("-inf")
    x[1, 3] = float("nan")
    x[2, 2] = float("inf")
    t = token_logprobs(x, torch.tensor([0, 1, 2]), 2)
    assert all(bool(v.isnan().all()) for v in t[:3])
    assert t.top_ids.tolist() == [[0, 1], [3, 0], [2, 0]]


@pytest.mark.parametrize("change,words", [
    (dict(logits=torch.zeros(2, 8, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (dict(logits=torch.zeros(2, 0)), "vocabulary"),
    (dict(tokens=torch.zeros(3, dtype=torch.long)), "tokens must be"),
    (dict(tokens=torch.zeros(2)), "tokens must be"),
    (dict(top=9), "top must be"), (dict(top=-1), "top must be"), (dict(top=2.0), "top must be"),
    (dict(top=True), "top must be"),
    (dict(logits=torch.zeros(1, 8).expand(2 ** 24, 8), tokens=torch.zeros(1, dtype=torch.long).expand(2 ** 24)), "16777215 rows"),
    (dict(logits=torch.zeros(2, 8, requires_grad=True)), "gradient")])
def test_refusals(change, words):
    args = dict(logits=torch.zeros(2, 8), tokens=torch.zeros(2, dtype=torch.long), top=2) | change
    with pytest.raises(ValueError, match=words):
        token_logprobs(**args)


def test_the_library_refuses_before_any_device_work():
    lib = _lib.load()
    p = ctypes.c_void_p(64)       # never dereferenced
    good = dict(logits=p, kind=0, stride=100, rows=2, vocab=100, tokens=p, top=5, lp=p, h=p, tl=p, ti=p, ws=p)

    def call(**change):
        a = good | change
        return lib.nkv_token_logprobs(a["logits"], a["kind"], a["stride"], a["rows"], a["vocab"], a["tokens"], a["top"],
                                      a["lp"], a["h"], a["tl"], a["ti"], a["ws"], None)

    for change, words in ((dict(kind=3), b"type of logits"), (dict(vocab=0), b"vocab"), (dict(rows=-1), b"rows"),
                          (dict(top=65), b"top must be"), (dict(top=101), b"top must be"), (dict(logits=None), b"NULL"),
                          (dict(tl=None), b"NULL"), (dict(logits=ctypes.c_void_p(66)), b"aligned"),
                          (dict(vocab=151936, ws=None, rows=1), b"workspace"), (dict(rows=2 ** 24), b"2^24 - 1")):
        assert call(**change) == _lib.NKV_ERR_ARG and words in lib.nkv_last_error(), change
    assert call(rows=0) == _lib.NKV_OK
    assert lib.nkv_token_logprobs_workspace(1, 151936, 20) > 0
    assert lib.nkv_token_logprobs_workspace(4096, 151936, 20) == 0
