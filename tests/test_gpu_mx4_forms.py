"""The product in the forms that the other tests' sizes do not take: the larger tiles with and without a split of K, each
for both kinds of x and gated, and few rows where K is walked in chunks or a workgroup walks several tiles."""
import pytest
import torch

from gpu_util import gpu_or_skip, log
from lit_gpt.kdn_ops import _lib
from lit_gpt.kdn_ops.mx4 import mx4_dequantize, mx4_linear, mx4_quantize
from oracle import mx4_oracle as mo

pytestmark = pytest.mark.gpu


def _check(dev, M, N, K, act, gated, splits):
    log(f"case mx4_linear M={M} N={N} K={K} {act} gated={gated}")
    quantized, R = act == "mx4", 2 * N if gated else N
    # the form is the one meant: so many splits' sums in the workspace
    held = _lib.size("kdn_mx4_linear_workspace_size", M, N, K, int(quantized), int(gated))
    assert held == (splits * M * R * 4 if splits > 1 else 0)
    g = torch.Generator(device=dev).manual_seed(M + 3 * N + 7 * K)
    rand = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    w = mx4_quantize(rand(R, K) / K ** 0.5)
    x, b, r = rand(M, K).bfloat16(), (0.3 * rand(R)).bfloat16(), rand(M, N).bfloat16()
    xin = mx4_quantize(x) if quantized else x
    y = mx4_linear(xin, w, b, residual=r, gated=gated)
    xd = (mx4_dequantize(xin) if quantized else x).double()
    ref, size = mo.linear(xd, mx4_dequantize(w).double(), b.double(), r.double(), gated)
    off = (y.double() - ref).abs()
    # the rounding to bf16, and fp32 sums: 2^-24 of the terms' size for each of K / 32 partial sums, and 32 more for the
    # epilogue and the splits
    bound = ref.abs() * 2.0 ** -8 + size * (K / 32 + 32) * 2.0 ** -24 + 1e-30
    assert bool((off <= bound).all()), f"worst {float((off / bound).max()):.3g} of the bound"


FEW = [  # at most 16 rows; several tiles per workgroup: the gate's N 7208; K in chunks: the down product's 7208
    (1, 7208, 2304, True), (9, 7208, 2304, True), (16, 7208, 2304, True), (16, 9001, 2304, False), (5, 9999, 520, True),
    (9, 2304, 7208, False), (16, 2304, 7208, False), (16, 5001, 4104, False), (11, 6000, 4104, True), (16, 7208, 7208, True),
    (3, 700, 10504, False), (13, 701, 10504, True), (16, 32000, 2304, False), (2, 20001, 136, False)]


@pytest.mark.parametrize("act", ["bf16", "mx4"])
@pytest.mark.parametrize("M,N,K,gated", FEW)
def test_few_rows(M, N, K, gated, act):
    _check(gpu_or_skip(), M, N, K, act, gated, 1)


TILES = {
    # tile: (M, N, K, act, gated, splits)
    "32x128": [(33, 7208, 2304, "bf16", True, 1), (64, 2304, 7208, "bf16", False, 7), (33, 7208, 2304, "mx4", True, 1)],
    "64x128": [(2981, 257, 392, "bf16", False, 1), (1030, 130, 4104, "bf16", False, 7), (2981, 130, 392, "bf16", True, 1),
               (1030, 70, 4104, "bf16", True, 7), (2981, 257, 392, "mx4", False, 1), (700, 130, 4104, "mx4", False, 7),
               (2981, 130, 392, "mx4", True, 1), (700, 70, 4104, "mx4", True, 7), (64, 32000, 2304, "bf16", False, 1),
               (64, 32000, 2304, "mx4", False, 1)],
    "128x128": [(2337, 816, 392, "bf16", False, 1), (2049, 130, 4104, "bf16", False, 7), (1030, 1001, 392, "bf16", True, 1),
                (2049, 70, 7208, "bf16", True, 7), (2337, 816, 392, "mx4", False, 1), (2049, 130, 7208, "mx4", False, 6),
                (1223, 816, 392, "mx4", True, 1), (2049, 70, 7208, "mx4", True, 6), (301, 2304, 7128, "mx4", False, 4)],
    "128x256": [(2981, 1296, 392, "bf16", False, 1), (2337, 130, 11248, "bf16", False, 13), (2049, 1001, 392, "bf16", True, 1),
                (65, 3002, 11248, "bf16", True, 10), (2981, 1296, 392, "mx4", False, 1), (65, 12001, 10504, "mx4", False, 5),
                (2049, 1001, 392, "mx4", True, 1), (129, 3002, 11480, "mx4", True, 5)],
    "256x256": [(513, 20001, 392, "bf16", False, 1), (2981, 1296, 7208, "bf16", False, 3), (129, 32000, 392, "bf16", True, 1),
                (2337, 514, 10504, "bf16", True, 5), (513, 20001, 392, "mx4", False, 1), (2981, 1296, 10504, "mx4", False, 3),
                (129, 32000, 392, "mx4", True, 1), (400, 5003, 10504, "mx4", True, 3), (4096, 7208, 2304, "bf16", True, 1),
                (4096, 7208, 2304, "mx4", True, 1)],
}


@pytest.mark.parametrize("M,N,K,act,gated,splits", [c for t in TILES.values() for c in t])
def test_tiles(M, N, K, act, gated, splits):
    _check(gpu_or_skip(), M, N, K, act, gated, splits)
