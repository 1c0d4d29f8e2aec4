"""The decoder with 8-bit projections, on CPU tensors (the operators' formulas):
what quantize_linears_ replaces, what the layer then calls, and what is refused."""

import pytest
import torch
import torch.nn.functional as F
from torch import nn

from nanokv_amd import q8, qwen3

CFG = dict(vocab_size=64, hidden_size=256, intermediate_size=384, num_hidden_layers=2, num_attention_heads=4,
           num_key_value_heads=2, max_position_embeddings=64)


class _Mean(nn.Module):
    """Stands for the sparse attention: each query head gets its KV head's value."""

    def forward(self, q, k, v):
        return v.repeat_interleave(q.shape[1] // v.shape[1], dim=1)


def _model(bias=False, tie=True, dtype=torch.bfloat16):
    torch.manual_seed(1)
    model = qwen3.Qwen3ForCausalLM(qwen3.Qwen3Config(**CFG, attention_bias=bias, tie_word_embeddings=tie)).to(dtype)
    qwen3.init_random_(model, 2)
    for layer in model.model.layers:
        layer.self_attn.attn = _Mean()
        if bias:
            layer.self_attn.qkv_proj.bias.copy_(torch.randn(layer.self_attn.qkv_proj.out_features))
    return model


def _forward(model, rows=5):
    ids = torch.arange(rows) * 7 % CFG["vocab_size"]
    with torch.no_grad():
        return model.compute_logits(model(ids, torch.arange(rows)))


@pytest.mark.parametrize("bias,tie", [(False, True), (True, False)])
def test_quantize_linears_replaces_the_projections_and_the_head(bias, tie):
    model = _model(bias, tie)
    want = _forward(model).double()
    weights = {n: m.weight.clone() for n, m in model.named_modules() if isinstance(m, qwen3.Linear)}
    assert qwen3.quantize_linears_(model) == 2 * 4 + 1
    assert not any(isinstance(m, nn.Linear) for m in model.modules())
    for name, w in weights.items():
        m = model.get_submodule(name)
        assert type(m) is qwen3.Q8Linear and (m.out_features, m.in_features) == tuple(w.shape)
        # half a step of a row's scale
        err = (q8.dequantize_q8(m.weight).double() - w.double()).abs()
        assert bool((err <= (0.5 + 2.0 ** -1) * m.weight_scale.double()[:, None]).all())
    got = _forward(model).double()
    # 8 bits a row: codes off by up to 1 / 254 of a row's peak (about 4 of its rms), 1e-2 a product's
    # rms at most, in 8 products one after the other that add up as independent errors
    assert float((got - want).norm() / want.norm()) < 0.05
    assert model.get_parameter("model.embed_tokens.weight").dtype == torch.bfloat16


def test_the_head_can_stay():
    model = _model()
    assert qwen3.quantize_linears_(model, lm_head=False) == 8 and model.lm_head_q8 is None
    h = torch.randn(2, CFG["hidden_size"]).bfloat16()
    assert torch.equal(model.compute_logits(h), F.linear(h, model.lm_head_weight))


def test_a_layer_is_its_operators():
    layer = _model(bias=False).model.layers[0]
    qwen3.quantize_linears_(layer)
    g = torch.Generator().manual_seed(5)
    h, res = (torch.randn(3, 256, generator=g).bfloat16() for _ in range(2))
    attn, mlp = layer.self_attn, layer.mlp
    got = layer(torch.arange(3), h, res)
    qkv, r = q8.norm_linear_q8(h, layer.input_layernorm.weight, 1e-6, attn.qkv_proj.weight, res)
    x = attn.attend(torch.arange(3), qkv)
    x, r = q8.rmsnorm_q8(x, layer.post_attention_layernorm.weight, 1e-6, r)
    y = q8.linear_q8(q8.linear_silu_mul_q8(x, mlp.gate_up_proj.weight), mlp.down_proj.weight)
    assert torch.equal(got[0], y) and torch.equal(got[1], r)
    # the MLP on its own, and a layer without a residual
    assert torch.equal(mlp(h), q8.linear_q8(q8.linear_silu_mul_q8(h, mlp.gate_up_proj.weight), mlp.down_proj.weight))
    assert torch.equal(layer(torch.arange(3), h, None)[1],
                       (h.float() + attn.attend(torch.arange(3), q8.norm_linear_q8(
                           h, layer.input_layernorm.weight, 1e-6, attn.qkv_proj.weight)[0]).float()).bfloat16())


class _Adapter(nn.Module):
    """A wrapper that shows the wrapped module's parameters and adds a term."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner
        self.weight, self.bias = inner.weight, getattr(inner, "bias", None)
        self.eps = getattr(inner, "eps", None)

    def forward(self, *args):
        y = self.inner(*args)
        return (y[0] + 1, *y[1:]) if isinstance(y, tuple) else y + 1


@pytest.mark.parametrize("path", ["input_layernorm", "self_attn.qkv_proj", "post_attention_layernorm", "mlp.gate_up_proj",
                                  "mlp.down_proj", "self_attn.o_proj"])
@pytest.mark.parametrize("how", ["adapter", "hook", "instance"])
def test_a_replaced_module_is_called(path, how):
    layer = _model().model.layers[0]
    qwen3.quantize_linears_(layer)
    parent, _, leaf = path.rpartition(".")
    owner = layer.get_submodule(parent)
    inner, seen = getattr(owner, leaf), []
    if how == "adapter":
        setattr(owner, leaf, _Adapter(inner))
        getattr(owner, leaf).register_forward_hook(lambda *a: seen.append(1))
    elif how == "hook":
        inner.register_forward_hook(lambda *a: seen.append(1))
    else:
        forward = inner.forward
        inner.forward = lambda *a: (seen.append(1), forward(*a))[1]
    h, res = torch.randn(2, 256).bfloat16(), torch.randn(2, 256).bfloat16()
    layer(torch.arange(2), h, res)
    assert seen == [1]


def test_projections_replaced_before_stay():
    layer = _model().model.layers[0]
    layer.self_attn.o_proj = _Adapter(layer.self_attn.o_proj)
    layer.mlp.down_proj.register_forward_hook(lambda *a: None)
    # (the adapter's inner Linear is a projection of its own)
    qwen3.quantize_linears_(layer)
    assert type(layer.self_attn.o_proj) is _Adapter and type(layer.mlp.down_proj) is qwen3.Linear
    assert type(layer.self_attn.qkv_proj) is qwen3.Q8Linear


def test_state_and_casts():
    a, b = _model(bias=True), _model(bias=True)
    qwen3.quantize_linears_(a)
    qwen3.quantize_linears_(b)
    for m in b.modules():
        if isinstance(m, qwen3.Q8Linear):
            m.weight_q8.zero_()
            m.weight_scale.zero_()
    b.load_state_dict(a.state_dict())
    assert torch.equal(_forward(a), _forward(b))
    scales = [m.weight_scale.clone() for m in a.modules() if isinstance(m, qwen3.Q8Linear)]
    a.to(torch.float32).to(torch.bfloat16)
    after = [m for m in a.modules() if isinstance(m, qwen3.Q8Linear)]
    assert all(m.weight_scale.dtype == torch.float32 and torch.equal(m.weight_scale, s) for m, s in zip(after, scales))
    assert all(m.weight_q8.dtype == torch.int8 for m in after)


def test_refusals(tmp_path):
    model = _model()
    with torch.no_grad():
        model.model.layers[1].mlp.down_proj.weight[3, 5] = float("nan")
    with pytest.raises(ValueError, match="layers.1.mlp.down_proj.*NaN"):
        qwen3.quantize_linears_(model)
    assert sum(isinstance(m, qwen3.Q8Linear) for m in model.modules()) == 0      # nothing was replaced
    with pytest.raises(ValueError, match="multiple of 16"):
        qwen3.Q8Linear(torch.randn(4, 24).bfloat16())
    with pytest.raises(ValueError):
        qwen3.Q8Linear(torch.randn(4).bfloat16())
    model = _model()
    qwen3.quantize_linears_(model)
    for call in (lambda: qwen3.init_random_(model), lambda: qwen3.load_checkpoint(model, str(tmp_path))):
        with pytest.raises(ValueError, match="8 bits already"):
            call()
    with pytest.raises(ValueError, match="weights must be"):
        qwen3.from_pretrained(str(tmp_path), weights="int4")
