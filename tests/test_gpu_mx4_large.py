"""Matrices whose offsets do not fit 32 bits, and that are converted in several launches."""
import pytest
import torch

from gpu_util import gpu_or_skip, log
from lit_gpt.kdn_ops.mx4 import mx4_dequantize, mx4_linear, mx4_quantize
from oracle import mx4_oracle as mo

pytestmark = pytest.mark.gpu


def _filled(dev, rows, cols):
    """bf16 [rows, cols] with rows that differ: random rows, scaled by powers of two."""
    g = torch.Generator(device=dev).manual_seed(rows)
    some = torch.randn(64, cols, generator=g, device=dev).bfloat16()
    x = torch.empty(rows, cols, device=dev, dtype=torch.bfloat16)
    for r in range(0, rows, 64):
        n = min(64, rows - r)
        torch.mul(some[:n], 2.0 ** (r // 64 % 7), out=x[r:r + n])
    return x


def test_quantize_in_several_launches():
    dev = gpu_or_skip()
    rows, cols = (1 << 15) + 67, 1 << 18  # 2^30 items of 8 elements and some more
    log(f"case mx4_quantize {rows} x {cols}")
    x = _filled(dev, rows, cols)
    q = mx4_quantize(x)
    at = [0, 1, 63, 64, (1 << 14) - 1, 1 << 14, (1 << 15) - 1, 1 << 15, (1 << 15) + 1, rows - 1]
    some = mx4_quantize(x[at])
    assert torch.equal(q.codes[at], some.codes) and torch.equal(q.scales[at], some.scales)
    want = mx4_dequantize(some, torch.bfloat16)
    del x
    assert torch.equal(mx4_dequantize(q, torch.bfloat16)[at], want)
    assert torch.equal(mx4_dequantize(q)[at], want.float())


@pytest.mark.parametrize("act", ["bf16", "mx4"])
def test_product_of_many_rows(act):
    dev = gpu_or_skip()
    M, N, K = (1 << 20) + 77, 2100, 2312
    log(f"case mx4_linear M={M} N={N} K={K} {act}")
    x = _filled(dev, M, K)
    g = torch.Generator(device=dev).manual_seed(1)
    w = mx4_quantize(torch.randn(N, K, generator=g, device=dev) / K ** 0.5)
    r = torch.randn(64, N, generator=g, device=dev).bfloat16().repeat(M // 64 + 1, 1)[:M]
    xin = mx4_quantize(x) if act == "mx4" else x
    y = mx4_linear(xin, w, residual=r)
    at = torch.cat([torch.arange(a, a + 40, device=dev) for a in (0, (1 << 19) - 20, 928800, (1 << 20) - 3, M - 40)])
    xd = (mx4_dequantize(mx4_quantize(x[at])) if act == "mx4" else x[at]).double()
    ref, size = mo.linear(xd, mx4_dequantize(w).double(), None, r[at].double())
    off = (y[at].double() - ref).abs()
    # as for smaller products: the rounding to bf16, and fp32 sums
    assert bool((off <= ref.abs() * 2.0 ** -8 + size * (K / 32 + 32) * 2.0 ** -24 + 1e-30).all())
