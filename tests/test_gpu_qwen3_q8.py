"""A whole Qwen3 decoder with 8-bit projections on the GPU (quantize_linears_).

Prompt chunks and tokens go through the integer products against an independent
float64 decoder (tests/_qwen3_ref.py) of the same weights as they are held (the
codes times their scales), so what differs is the rows' quantisation.  A row's code
is off by at most half a step of peak / 127, uniformly: peak / rms / (127 sqrt(12))
relative to the row, 1.1% for a normal row (peak 5 rms) and 2.3% for a gated product's (peak 10
rms).  Two layers have six of the first and two of the second, and the head one more:
sqrt(7 * 1.1^2 + 2 * 2.3^2) = 4.4% if every error reached the logits whole; the
attention averages values, so its outputs are below that.  The bound is 6%.
"""

import numpy as np
import pytest
import torch

from tests._qwen3_ref import RefQwen3
from tests._util import to_np

pytestmark = pytest.mark.gpu

TOL = 0.06


def _rel(a, b):
    return float(np.linalg.norm(np.asarray(a, np.float64) - b) / np.linalg.norm(b))


def _model(seed, bias=False):
    from nanokv_amd.qwen3 import Qwen3Config, Qwen3ForCausalLM, init_random_
    cfg = Qwen3Config(vocab_size=512, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
                      num_attention_heads=8, num_key_value_heads=2, max_position_embeddings=4096, attention_bias=bias)
    model = Qwen3ForCausalLM(cfg)
    init_random_(model, seed)
    return model.to(device="cuda", dtype=torch.bfloat16)


def test_prefill_and_decode_match_float64_reference():
    from nanokv_amd.qwen3 import Q8Linear, quantize_linears_
    from nanokv_amd.sparse import M12Config

    m12 = M12Config(max_model_len=2048, num_heads=8, num_kv_heads=2)
    model = _model(7)
    state = dict(model.state_dict())
    assert quantize_linears_(model) == 9
    for name, m in model.named_modules():
        if isinstance(m, Q8Linear):
            key = "lm_head_weight" if name == "lm_head_q8" else name + ".weight"
            state[key] = m.weight_q8.double() * m.weight_scale.double()[:, None]
    ref = RefQwen3(state, model.config, m12)
    model.attach(m12)
    caps = []
    for layer in model.model.layers:
        layer.self_attn.attn.register_forward_hook(lambda m, i, o: caps.append(to_np(o)))
    prompt = torch.randint(0, 512, (1024,), generator=torch.Generator().manual_seed(3))
    logits = model.prefill(prompt.cuda(), chunk=512)
    ref.forward(prompt[:512], "first")
    ref_logits = ref.forward(prompt[512:], "chunk")
    for i, o in enumerate(caps):
        assert _rel(o, ref.attn_out[i // 2][i % 2]) <= TOL
    e = _rel(to_np(logits), ref_logits[-1].numpy())
    print(f"prefill logits rel err {e:.4f}", flush=True)
    assert e <= TOL
    pos = 1024
    for step in range(3):
        caps.clear()
        tok = logits.argmax().view(1)
        logits = model.decode(tok, pos)
        ref_logits = ref.forward(tok.cpu(), "decode")
        pos += 1
        for i, o in enumerate(caps):
            assert _rel(o, ref.attn_out[-1][i]) <= TOL
        e = _rel(to_np(logits), ref_logits[-1].numpy())
        print(f"decode {step}: logits rel err {e:.4f}", flush=True)
        assert e <= TOL


@pytest.mark.parametrize("bias", [False, True])
def test_decode_graph_replays_match_eager_decode(bias):
    """One captured token step, replayed, against decode() of a twin: the same bits."""
    from nanokv_amd.qwen3 import quantize_linears_
    from nanokv_amd.sparse import M12Config

    models = []
    for _ in range(2):
        m = _model(11, bias)
        if bias:
            for layer in m.model.layers:
                layer.self_attn.qkv_proj.bias.copy_(torch.linspace(-1, 1, layer.self_attn.qkv_proj.out_features))
        quantize_linears_(m)
        m.attach(M12Config(max_model_len=2048, num_heads=8, num_kv_heads=2))
        models.append(m)
    eager, graphed = models
    prompt = torch.randint(0, 512, (1024,), generator=torch.Generator().manual_seed(4)).cuda()
    la, lb = eager.prefill(prompt, chunk=512), graphed.prefill(prompt, chunk=512)
    assert torch.equal(la, lb)
    for step in range(8):
        tok = la.argmax().view(1)
        lb = graphed.decode_graph(tok, 1024 + step).clone()
        la = eager.decode(tok, 1024 + step)
        torch.cuda.synchronize()
        assert torch.equal(la, lb), step
    assert graphed._graph is not None
    quantize_linears_(graphed)                    # nothing left but the head: the captured step is dropped
    assert graphed._graph is None


def test_a_short_prompt_and_a_draft_length_chunk():
    """Prompts of 2 to 40 tokens run through the few-row products."""
    from nanokv_amd.qwen3 import quantize_linears_
    from nanokv_amd.sparse import M12Config

    model = _model(5)
    plain = _model(5)
    quantize_linears_(model)
    for m in (model, plain):
        m.attach(M12Config(max_model_len=2048, num_heads=8, num_kv_heads=2))
    for n in (2, 7, 40):
        prompt = torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(n)).cuda()
        outs = []
        for m in (model, plain):
            m.reset()
            outs.append(to_np(m.prefill(prompt)))
        # against bf16 weights their own quantisation counts too: sqrt(2) times the bound above
        assert _rel(outs[0], outs[1]) <= 2 ** 0.5 * TOL
