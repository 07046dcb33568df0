"""A product with a weight of no rows."""
import pytest
import torch

from gpu_util import gpu_or_skip, log
from lit_gpt.kdn_ops.mx4 import mx4_linear, mx4_quantize

pytestmark = pytest.mark.gpu


def test_no_rows_of_the_weight():
    dev = gpu_or_skip()
    log("case mx4_linear N=0")
    w = mx4_quantize(torch.zeros(0, 64, device=dev))
    x = torch.zeros(2, 3, 64, device=dev, dtype=torch.bfloat16)
    r = torch.zeros(2, 3, 0, device=dev, dtype=torch.bfloat16)
    for gated in (False, True):
        assert mx4_linear(x, w, gated=gated).shape == (2, 3, 0)
        assert mx4_linear(x, w, residual=r, gated=gated).shape == (2, 3, 0)
        assert mx4_linear(x[:, 0], w, residual=r[:, 0], gated=gated).shape == (2, 0)
