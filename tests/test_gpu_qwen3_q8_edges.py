"""quantize_linears_ at its edges on the GPU."""

import pytest
import torch

from tests.test_gpu_qwen3_q8 import _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("part", [lambda m: m.model, lambda m: m.model.layers[1]])
def test_a_part_quantised_between_graph_steps(part):
    """The step captured before is dropped: the next ones are the eager twin's, bit for bit."""
    from nanokv_amd.qwen3 import quantize_linears_
    from nanokv_amd.sparse import M12Config

    eager, graphed = _model(11), _model(11)
    for m in (eager, graphed):
        m.attach(M12Config(max_model_len=2048, num_heads=8, num_kv_heads=2))
    prompt = torch.randint(0, 512, (1024,), generator=torch.Generator().manual_seed(4)).cuda()
    la, lb = eager.prefill(prompt, chunk=512), graphed.prefill(prompt, chunk=512)
    assert torch.equal(la, lb)
    for step in range(10):
        if step == 4:
            assert graphed._graph is not None
            torch.cuda.synchronize()
            for m in (eager, graphed):
                assert quantize_linears_(part(m)) > 0
        tok = la.argmax().view(1)
        lb = graphed.decode_graph(tok, 1024 + step).clone()
        la = eager.decode(tok, 1024 + step)
        torch.cuda.synchronize()
        assert torch.equal(la, lb), step
    assert graphed._graph is not None
