"""The serving operators have no derivative: an input that carries one is refused, in either mode, not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from lit_gpt.kdn_ops.mx4 import MX4Tensor, mx4_linear, mx4_quantize
from lit_gpt.kdn_ops.sampling import sample_tokens


def _calls():
    x = torch.zeros(2, 64).bfloat16()
    w = MX4Tensor(torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.uint8), 64)
    l, e = torch.zeros(2, 8), torch.ones(2, 8)
    return {"quantize": (x, lambda t: mx4_quantize(t)),
            "linear x": (x, lambda t: mx4_linear(t, w)),
            "linear bias": (torch.zeros(8).bfloat16(), lambda t: mx4_linear(x, w, t)),
            "linear residual": (torch.zeros(2, 8).bfloat16(), lambda t: mx4_linear(x, w, residual=t)),
            "sample logits": (l, lambda t: sample_tokens(t, e)),
            "sample noise": (e, lambda t: sample_tokens(l, t)),
            "sample temperature": (torch.ones(2), lambda t: sample_tokens(l, e, temperature=t))}


@pytest.mark.parametrize("name", list(_calls()))
def test_gradients_are_refused(name):
    t, call = _calls()[name]
    with pytest.raises(RuntimeError, match="no backward"):
        call(t.clone().requires_grad_())
    with torch.no_grad(), pytest.raises(ValueError, match="device"):  # the call itself, on CPU tensors
        call(t.clone().requires_grad_())


@pytest.mark.parametrize("name", list(_calls()))
def test_tangents_are_refused(name):
    t, call = _calls()[name]
    with fwAD.dual_level():
        with pytest.raises(ValueError, match="device"):  # no tangent: the call itself, on CPU tensors
            call(t)
        for mode in (torch.no_grad(), torch.enable_grad()):
            with mode, pytest.raises(RuntimeError, match="no forward-mode"):
                call(fwAD.make_dual(t, torch.ones_like(t)))
