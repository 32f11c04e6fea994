"""What the entry points of top logits, distillation, beam selection and state
reordering promise beside their numbers: what they refuse, what autograd is told,
orders among equals, values bit for bit, the paths of the model around them."""
import pytest
import torch

from test_top_distill_beam import _dev, _gen, gpu


# --------------------------------------------------------------------------
# states that follow their beams
# --------------------------------------------------------------------------
@gpu
def test_reorder_states_tells_autograd():
    """What an operation saved of a state before is not silently another."""
    import paccmann_chemistry_amd as P
    dev = _dev()
    parents = torch.tensor([[1, 0], [0, 1]], dtype=torch.int32, device=dev)
    hidden = torch.randn(4, 8, generator=_gen(1)).to(dev)
    stack = torch.randn(2, 4, 3, generator=_gen(2)).to(dev)
    weight = torch.ones(3, 8, device=dev, requires_grad=True)
    out = torch.nn.functional.linear(hidden, weight)
    before = hidden._version, stack._version
    P.reorder_states(parents, [hidden, stack], [0, 1])
    assert (hidden._version, stack._version) == (before[0] + 1, before[1] + 1)
    with pytest.raises(RuntimeError, match='inplace operation'):
        out.sum().backward()
    with torch.inference_mode():
        state = torch.arange(4.0, device=dev).view(4, 1)
        P.reorder_states(parents, [state, hidden])
        assert state.view(-1).tolist() == [2.0, 1.0, 0.0, 3.0]
