"""The Qwen3 decoder over paged caches on the GPU: prompts, tokens and drafted trees of several
sequences at once, a captured step, log probabilities of prompts.

The reference is the decoder in 64 bits, dense over each sequence (_dense_ref); tolerances are those
of the sparse decoder's test: 2.5% of the logits, where a position that is off by one moves them by 9%."""

import pytest
import torch

from _dense_ref import dense_logits, one_step, serve

pytestmark = pytest.mark.gpu
TOL = 0.025


def _model(seed=3, **more):
    from nanokv_amd.qwen3 import Qwen3Config, Qwen3ForCausalLM, init_random_
    cfg = Qwen3Config(**(dict(vocab_size=512, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
                              num_attention_heads=8, num_key_value_heads=2, max_position_embeddings=4096) | more))
    model = Qwen3ForCausalLM(cfg)
    init_random_(model, seed)
    return model.to(device="cuda", dtype=torch.bfloat16)


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("more", [{}, {"attention_bias": True}, {"head_dim": 64, "num_key_value_heads": 8}])
def test_a_server_run(kv, more):
    model = _model(**more)

    def check(name, h, ends):
        ref = torch.stack([dense_logits(model, s)[-1] for s in ends])
        got = model.compute_logits(h).double().cpu()
        e = float((got - ref).norm() / ref.norm())
        print(f"{name}: {e:.4f}", flush=True)
        assert e <= TOL, name

    serve(model, "cuda", kv, check)


def test_one_launch_is_the_modules_chain():
    """Norms, rotation and writes in one launch, or module by module (a hook asks for that):
    the same up to the modules' additional roundings."""
    model = _model()
    ids = torch.randint(0, 512, (50,), generator=torch.Generator().manual_seed(1)).tolist()
    fused = one_step(model, "cuda", "bf16", ids).float()
    calls = []
    for layer in model.model.layers:
        layer.self_attn.attn.register_forward_hook(lambda *a: calls.append(1))
    chain = one_step(model, "cuda", "bf16", ids).float()
    assert len(calls) == 2
    assert float((fused - chain).norm() / chain.norm()) < TOL


def test_eight_bit_projections_over_eight_bit_caches():
    from nanokv_amd.qwen3 import quantize_linears_
    model = _model(seed=5)
    ids = torch.randint(0, 512, (80,), generator=torch.Generator().manual_seed(1)).tolist()
    plain = one_step(model, "cuda", "int8", ids).float()
    quantize_linears_(model)
    got = one_step(model, "cuda", "int8", ids).float()
    # (the codes' own error: the 8-bit decoder's test bounds it)
    assert float((got - plain).norm() / plain.norm()) < 0.1


def test_a_captured_step_is_replayed():
    """A decode step of three sequences, captured once: tokens, positions, slots, tables and
    lengths change in place; each replay gives the eager step's bits."""
    models = [_model(), _model()]
    for m in models:
        m.attach_paged(40, 16)
    tables = torch.randperm(40, generator=torch.Generator().manual_seed(0))[:36].view(3, 12).to(torch.int32).cuda()
    lens = torch.tensor([5, 90, 33])
    ids = torch.arange(128).cuda()
    starts = torch.tensor([0, 5, 95, 128], dtype=torch.int32).cuda()

    def slots(places):
        return torch.tensor([int(tables[b, p // 16]) * 16 + p % 16 for b, p in places]).cuda()

    prompt = [(b, p) for b in range(3) for p in range(int(lens[b]))]
    for m in models:
        m.paged_step(ids, torch.tensor([p for _, p in prompt]).cuda(), slots(prompt), tables, lens.cuda().int(),
                     starts=starts, max_new=90)
    tok, pos, slot, length = (torch.zeros(3, dtype=t).cuda() for t in (torch.long, torch.long, torch.int32, torch.int32))

    def fill(step):
        tok.copy_(torch.tensor([3, 5, 7]) + step)
        pos.copy_(lens + step)
        slot.copy_(slots([(b, int(lens[b]) + step) for b in range(3)]))
        length.copy_(lens + step + 1)

    fill(0)
    eager = models[0]
    eager.compute_logits(eager.paged_step(tok, pos, slot, tables, length))
    models[1].compute_logits(models[1].paged_step(tok, pos, slot, tables, length))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = models[1].compute_logits(models[1].paged_step(tok, pos, slot, tables, length))
    for step in range(1, 6):
        fill(step)
        want = eager.compute_logits(eager.paged_step(tok, pos, slot, tables, length))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), step


def test_log_probabilities_of_a_prompt():
    """The sparse prefill's and the paged step's, against those of their logits."""
    from nanokv_amd.sparse import M12Config
    model = _model(vocab_size=3001)
    ids = torch.randint(0, 3001, (200,), generator=torch.Generator().manual_seed(4)).cuda()
    model.attach(M12Config(max_model_len=512, num_heads=8, num_kv_heads=2))
    last, lp = model.prefill_logprobs(ids, top=4, chunk=90)
    model.reset()
    assert torch.equal(last, model.prefill(ids, chunk=90)) and lp.logprob.shape == (199,)
    h = []
    model.reset()
    hook = model.model.register_forward_hook(lambda m, i, o: h.append(o))
    model.prefill(ids, chunk=90)
    hook.remove()
    h = torch.cat(h)[:-1]
    x = model.compute_logits(h)
    # the head's product takes other rows at a time: a logit is rounded to bf16 by 2^-8 of itself
    # each time, so log p, a difference of a logit and a mean of all, moves by 4 * 2^-8 max |x|
    tol = 4 * 2.0 ** -8 * float(x.abs().max()) + 1e-4
    ref = torch.log_softmax(x.double(), -1).gather(1, ids[1:, None])[:, 0]
    for t in (lp, model.token_logprobs(h, ids[1:], 4), model.token_logprobs(h, ids[1:], 4, rows=7)):
        assert float((t.logprob.double() - ref).abs().max()) <= tol
        assert t.top_ids.shape == (199, 4) and bool((t.top_logprobs[:, :-1] >= t.top_logprobs[:, 1:]).all())
    assert torch.equal(model.token_logprobs(h, ids[1:], 4, rows=199).top_ids[:, 0], x.argmax(-1))


def test_log_probabilities_of_a_prompt_of_one_token_are_refused_and_of_no_rows_are_none():
    from nanokv_amd.sparse import M12Config
    model = _model()
    model.attach(M12Config(max_model_len=512, num_heads=8, num_kv_heads=2))
    with pytest.raises(ValueError, match="at least 2 tokens"):          # (as prefill)
        model.prefill_logprobs(torch.tensor([7], device="cuda"), top=3)
    last, lp = model.prefill_logprobs(torch.tensor([7, 8], device="cuda"), top=3)
    assert last.shape == (512,) and lp.logprob.shape == (1,) and lp.top_ids.shape == (1, 3)
    lp = model.token_logprobs(torch.empty(0, 512, dtype=torch.bfloat16, device="cuda"), torch.empty(0, dtype=torch.long, device="cuda"))
    assert lp.entropy.shape == (0,) and lp.top_logprobs.shape == (0, 0)
