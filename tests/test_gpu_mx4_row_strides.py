"""The product on rows that lie far apart: the last position of every sequence of a long batch."""
import pytest
import torch

from gpu_util import gpu_or_skip, log
from lit_gpt.kdn_ops.mx4 import mx4_linear, mx4_quantize
from lit_gpt.quantize import MX4Linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T,K", [(3, 8192, 264), (2, 4096, 520), (20, 8192, 264), (2, 1, 264)])
def test_last_positions(B, T, K):
    """Row strides above and below 2^21 elements give what dense rows give."""
    dev = gpu_or_skip()
    log(f"case mx4_linear rows {T * K} elements apart, B={B}")
    g = torch.Generator(device=dev).manual_seed(B)
    h = torch.randn(B, T, K, generator=g, device=dev, dtype=torch.bfloat16)
    rows = h[:, -1]
    lin = torch.nn.Linear(K, 72).to(dev).to(torch.bfloat16)
    m = MX4Linear(lin)
    r = torch.randn(B, T, 72, generator=g, device=dev, dtype=torch.bfloat16)[:, -1]
    with torch.no_grad():
        assert torch.equal(m(rows), m(rows.contiguous()))
        w = mx4_quantize(lin.weight)
        assert torch.equal(mx4_linear(rows, w, residual=r), mx4_linear(rows.contiguous(), w, residual=r.contiguous()))
