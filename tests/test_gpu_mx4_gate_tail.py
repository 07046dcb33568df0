"""The MX4 product's SwiGLU gate where the sigmoid is subnormal (arguments from -87.3 to -88.7), against float64: the
other half can bring the result back into the normal range."""
import pytest
import torch

from gpu_util import gpu_or_skip, log
from lit_gpt.kdn_ops.mx4 import mx4_linear, mx4_quantize

pytestmark = pytest.mark.gpu

ARGS = [-86.0, -87.0, -87.5, -88.0, -88.5]  # bf16 numbers
# the sigmoid's bound of 1e-5 (the exponential's argument is rounded to 2^-24 of up to 128), then bf16's rounding
TOL = 2.0 ** -8 + 1e-5


@pytest.mark.parametrize("act", ["bf16", "mx4"])
@pytest.mark.parametrize("M,K", [(1, 64), (5, 2304), (20, 64), (20, 2304), (300, 264)])
def test_gate_tail(M, K, act):
    """Few rows, tiles, and (20 rows of K 2304) sums of a split K: the biases alone give both halves."""
    dev = gpu_or_skip()
    log(f"case mx4 gate tail M={M} K={K} {act}")
    a = torch.tensor(ARGS * 5, dtype=torch.float64)
    N, scale = len(a), 2.0 ** 60
    w = mx4_quantize(torch.zeros(2 * N, K, device=dev))
    bias = torch.cat((a, torch.full((N,), scale, dtype=torch.float64))).bfloat16().to(dev)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).bfloat16().to(dev)
    y = mx4_linear(x if act == "bf16" else mx4_quantize(x), w, bias, gated=True)
    ref = scale * a * torch.exp(a) / (1 + torch.exp(a))
    err = float(((y.double().cpu() - ref).abs() / ref.abs()).max())
    log(f"  largest relative error {err:.2e}")
    assert err <= TOL
