"""Heads of other types in ``GPT.forward``."""
import pytest
import torch
from torch import nn

from gpu_util import gpu_or_skip, log
from test_gpu_mx4_model_parts import _idx, _model

pytestmark = pytest.mark.gpu


class _OtherHead(nn.Module):
    def __init__(self, weight):
        super().__init__()
        self.weight = weight

    def forward(self, x):
        return 2 * (x @ self.weight.T)


class _WeightlessHead(nn.Module):
    def __init__(self, weight):
        super().__init__()
        self.w = weight

    def forward(self, x):
        return 2 * (x @ self.w.T)


@torch.no_grad()
def test_heads_of_other_types():
    """A head that has a weight gives that weight, whatever its type; one without is called."""
    dev = gpu_or_skip()
    log("case heads of other types")
    m = _model(dev)
    ref = m(_idx(dev))
    weight = m.lm_head.weight
    m.lm_head = _OtherHead(weight)
    assert torch.equal(m(_idx(dev)), ref)
    m.lm_head = _WeightlessHead(weight)
    assert float((m(_idx(dev)).float() - 2 * ref.float()).abs().max()) <= 2.0 ** -7 * float(ref.float().abs().max())
