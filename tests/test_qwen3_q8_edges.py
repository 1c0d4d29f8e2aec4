"""quantize_linears_ at its edges, on CPU tensors: captured steps, the untied head,
hooks, shared projections."""

import pytest
import torch
from torch import nn

from nanokv_amd import qwen3
from tests.test_qwen3_q8_modules import _forward, _model


class _Graph:
    """Stands for a captured step."""

    def __init__(self):
        self.replays = 0

    def replay(self):
        self.replays += 1


class _Runtime:
    """Stands for a layer's runtime in steady decode."""
    device_ring = False

    def device_ring_ready(self):
        return True

    def ring_replayed(self):
        pass


def _captured(model, monkeypatch):
    """A model whose decode_graph() captures and replays _Graphs and steps eagerly into `steps`."""
    model.runtimes = [_Runtime()]
    steps, graphs = [], []
    monkeypatch.setattr(model, "decode", lambda token, position: steps.append(position), raising=False)

    def capture(graph):
        graphs.append(graph())
        return graphs[-1]

    class Capturing:
        def __init__(self, *a):
            pass

        __enter__ = __exit__ = lambda self, *a: None

    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: capture(_Graph))
    monkeypatch.setattr(torch.cuda, "graph", Capturing)
    monkeypatch.setattr(_Runtime, "decode_state", lambda self: None, raising=False)
    monkeypatch.setattr(_Runtime, "restore_decode_state", lambda self, st: None, raising=False)
    monkeypatch.setattr(qwen3, "set_context", lambda *a, **k: None)
    return steps, graphs


@pytest.mark.parametrize("part", [lambda m: m, lambda m: m.model, lambda m: m.model.layers[1],
                                  lambda m: m.model.layers[0].mlp])
def test_a_captured_step_does_not_outlive_its_weights(part, monkeypatch):
    """Whatever part of the model is quantised: the replay would read weights that were freed."""
    model = _model()
    steps, graphs = _captured(model, monkeypatch)
    tok = torch.tensor([3])
    for position in range(3):
        model.decode_graph(tok, position)
    assert steps == [0] and len(graphs) == 1 and graphs[0].replays == 2
    qwen3.quantize_linears_(part(model))
    for position in range(3, 6):                  # an eager step, a capture, a replay
        model.decode_graph(tok, position)
    assert steps == [0, 3] and len(graphs) == 2 and [g.replays for g in graphs] == [2, 2]
    assert model.runtimes[0].device_ring
    other = _model()                              # nothing of this model is replaced: nothing is captured again
    model.decode_graph(tok, 6)
    assert len(graphs) == 2 and graphs[1].replays == 3 and other._graph is None


def test_weights_replaced_before_the_capture(monkeypatch):
    """The eager step in front of a capture is run again with the new weights."""
    model = _model()
    steps, graphs = _captured(model, monkeypatch)
    model.decode_graph(torch.tensor([3]), 0)
    qwen3.quantize_linears_(model.model)
    for position in range(1, 4):
        model.decode_graph(torch.tensor([3]), position)
    assert steps == [0, 1] and len(graphs) == 1 and graphs[0].replays == 2


@pytest.mark.parametrize("tie", [True, False])
def test_an_untied_head_is_held_once(tie):
    model = _model(tie=tie)
    n = 2 * 4 + 1
    head, embed = model.lm_head_weight, model.model.embed_tokens.weight
    assert qwen3.quantize_linears_(model) == n
    assert model.model.embed_tokens.weight is embed
    if tie:
        assert model.lm_head_weight is embed
    else:
        assert model.lm_head_weight is None and not any(p is head for p in model.parameters())
        assert "lm_head_weight" not in model.state_dict()
    want, held = _forward(model), model.lm_head_q8
    assert qwen3.quantize_linears_(model) == 0 and model.lm_head_q8 is held     # nothing is quantised again
    assert torch.equal(_forward(model), want)
    other = _model(tie=tie)
    with torch.no_grad():
        other.model.embed_tokens.weight.mul_(0.5)
    qwen3.quantize_linears_(other)
    other.load_state_dict(model.state_dict())
    assert torch.equal(_forward(other), want)
    model.to(torch.float32).to(torch.bfloat16)
    assert torch.equal(_forward(model), want)


def test_the_head_can_follow_the_projections():
    model = _model(tie=False)
    assert qwen3.quantize_linears_(model, lm_head=False) == 8 and model.lm_head_weight is not None
    assert qwen3.quantize_linears_(model) == 1 and model.lm_head_weight is None


def test_global_hooks_see_every_projection():
    layer = _model().model.layers[0]
    qwen3.quantize_linears_(layer)
    h, res = torch.randn(2, 256).bfloat16(), torch.randn(2, 256).bfloat16()
    seen = []
    hook = nn.modules.module.register_module_forward_hook(lambda m, i, o: seen.append(m))
    try:
        alone = layer.mlp(h)
        assert seen == [layer.mlp.gate_up_proj, layer.mlp.down_proj, layer.mlp]
        seen.clear()
        hooked = layer(torch.arange(2), h, res)
    finally:
        hook.remove()
    attn, mlp = layer.self_attn, layer.mlp
    assert [m for m in seen if isinstance(m, qwen3.Q8Linear)] == [attn.qkv_proj, attn.o_proj, mlp.gate_up_proj, mlp.down_proj]
    # the fused forms round less on the way: the norm's output (2^-8) and SiLU's factors are not rounded to
    # bf16 there, which moves values over a code's edge: a step of 1 / 127 of a row's peak (4 of its rms) in
    # some of its values, in two products one after the other
    for a, b in ((alone, layer.mlp(h)), (hooked[0], layer(torch.arange(2), h, res)[0])):
        assert float((a.double() - b.double()).norm() / b.double().norm()) < 2 * 4 / 127


def test_a_shared_projection_stays_shared():
    model = _model()
    a, b = (layer.mlp for layer in model.model.layers)
    b.down_proj = a.down_proj
    model.model.layers[1].self_attn = model.model.layers[0].self_attn
    assert qwen3.quantize_linears_(model, lm_head=False) == 5    # q|k|v, o, down once, gate|up twice
    assert type(a.down_proj) is qwen3.Q8Linear and b.down_proj is a.down_proj
    assert not any(isinstance(m, nn.Linear) for m in model.modules())
    _forward(model)


def test_a_projection_by_itself_is_refused():
    proj = qwen3.Linear(32, 16, bias=False)
    with pytest.raises(ValueError, match="Q8Linear"):
        qwen3.quantize_linears_(proj)
    assert not list(proj.children())


def test_weights_are_off_by_half_a_step():
    model = _model()
    weights = {n: m.weight.double() for n, m in model.named_modules() if isinstance(m, qwen3.Linear)}
    qwen3.quantize_linears_(model)
    for name, w in weights.items():
        q, scale = model.get_submodule(name).weight
        # the nearest code, and the scale's own rounding: 127 * 2^-24 of a step
        assert bool(((q.double() * scale.double()[:, None] - w).abs() <= (0.5 + 127 * 2.0 ** -24) * scale.double()[:, None]).all())
