"""The Qwen3 decoder over paged caches without a GPU: the module's routing on the operators' formulas."""

import pytest
import torch

from _dense_ref import dense_logits, one_step, serve
from nanokv_amd.attention import Attention, Context, attach_paged_cache, get_context, reset_context, set_context
from nanokv_amd.paged import PagedKV
from nanokv_amd.qwen3 import Qwen3Config, Qwen3ForCausalLM, init_random_

TINY = dict(vocab_size=64, hidden_size=128, intermediate_size=192, num_hidden_layers=2, num_attention_heads=4,
            num_key_value_heads=2, head_dim=64, max_position_embeddings=512)


def _model(**more):
    model = Qwen3ForCausalLM(Qwen3Config(**(TINY | more)))
    init_random_(model, 3, std=0.2)
    return model


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("bias", [False, True])
def test_a_server_run(kv, bias):
    """Batches, chunks, trees and moved rows give what each sequence gives alone in one step: the same
    rows of the cache, up to fp32's order of sums, which moves a held value to its neighbour
    (1/127 of its row's largest, or 2^-8 of itself) about once in 10^4: far below 0.5% of the logits."""
    model, twin = _model(attention_bias=bias), _model(attention_bias=bias)

    def check(name, h, ends):
        want = torch.stack([one_step(twin, "cpu", kv, s)[-1] for s in ends])
        got = model.compute_logits(h)
        assert float((got - want).norm() / want.norm()) < 0.005, name

    serve(model, "cpu", kv, check)
    assert get_context() == Context()


def test_a_step_against_the_decoder_in_64_bits():
    """fp32 modules, bf16 rows in the cache: the tolerance is that of the sparse decoder's test
    (a position that is off by one moves the logits by 9%)."""
    model = _model()
    ids = torch.randint(0, 64, (60,), generator=torch.Generator().manual_seed(0)).tolist()
    ref = dense_logits(model, ids)
    assert float((one_step(model, "cpu", "bf16", ids).double() - ref).norm() / ref.norm()) < 0.025


def test_wiring():
    model = _model()
    caches = model.attach_paged(6, 32)
    layers = [m for m in model.modules() if isinstance(m, Attention)]
    assert [m.layer_id for m in layers] == [0, 1] and all(m.dense() is c for m, c in zip(layers, caches))
    assert all(isinstance(c, PagedKV) and c.k.shape == (6, 2, 32, 64) and m.k_cache is c.k for m, c in zip(layers, caches))
    assert attach_paged_cache(model, 2, 16, torch.int8)[1].k_scale.shape == (2, 2, 16)

    class Off:
        enabled = True

    layers[0].sparse_rt = Off()
    assert layers[0].dense() is None
    Off.enabled = False
    assert layers[0].dense() is layers[0].paged_cache
    with pytest.raises(ValueError, match="no attention modules"):
        attach_paged_cache(torch.nn.Linear(2, 2), 2)


def test_steps_that_are_refused():
    model = _model()
    ids, at = torch.zeros(2, dtype=torch.long), torch.zeros(2, dtype=torch.long)
    tables, lengths = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="attach_paged"):
        model.paged_step(ids, at, at, tables, lengths)
    model.attach_paged(3, 16)
    with pytest.raises(ValueError, match="alike"):
        model.paged_step(ids, at[:1], at, tables, lengths)
    with pytest.raises(ValueError, match="lengths must be"):
        model.paged_step(ids, at, at, tables, lengths[:1])
    assert get_context() == Context()                 # (a step that raises leaves none behind)
    layer, x = model.model.layers[0].self_attn.attn, torch.zeros(1, 4, 64)
    try:
        set_context(False)
        with pytest.raises(ValueError, match="slot_mapping"):
            layer(x, x[:, :2], x[:, :2])
        set_context(False, slot_mapping=torch.zeros(1, dtype=torch.int32))
        with pytest.raises(ValueError, match="block_tables and context_lens"):
            layer(x, x[:, :2], x[:, :2])
    finally:
        reset_context()
    with pytest.raises(ValueError, match="one row at a time"):
        model.token_logprobs(torch.zeros(2, 128), torch.zeros(2, dtype=torch.long), rows=0)
    with pytest.raises(ValueError, match="tokens must be"):
        model.token_logprobs(torch.zeros(2, 128), torch.zeros(3, dtype=torch.long))


def test_lengths_from_the_references_prefill_context():
    """The reference's prefill context gives cu_seqlens_k, not context_lens."""
    model = _model()
    model.attach_paged(4, 16)
    layer = model.model.layers[0].self_attn.attn
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(5, n, 64, generator=g) for n in (4, 2, 2))
    starts = torch.tensor([0, 3, 5], dtype=torch.int32)
    tables = torch.tensor([[1], [3]], dtype=torch.int32)
    slots = torch.tensor([16, 17, 18, 48, 49])
    out = []
    try:
        for lens in (dict(cu_seqlens_k=starts), dict(context_lens=torch.tensor([3, 2], dtype=torch.int32))):
            set_context(True, cu_seqlens_q=starts, max_seqlen_q=3, slot_mapping=slots, block_tables=tables, **lens)
            out.append(layer(q, k, v))
    finally:
        reset_context()
    assert torch.equal(*out)


def test_logprobs_of_hidden_rows():
    model = _model()
    h = torch.randn(7, 128, generator=torch.Generator().manual_seed(1))
    tokens = torch.arange(7)
    whole = model.token_logprobs(h, tokens, 3)
    parts = model.token_logprobs(h, tokens, 3, rows=2)
    assert all(torch.allclose(a.double(), b.double(), atol=1e-5) for a, b in zip(whole, parts))
    lp = torch.log_softmax(model.compute_logits(h), -1)
    assert torch.allclose(whole.logprob, lp.gather(1, tokens[:, None])[:, 0], atol=1e-5)
    assert model.token_logprobs(h[:0], tokens[:0], 3).top_ids.shape == (0, 3)
