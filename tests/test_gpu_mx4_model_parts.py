"""``quantize_mx4`` on models whose parts are not the model's own."""
import copy

import pytest
import torch
from torch import nn

from gpu_util import gpu_or_skip, log
from lit_gpt import model as model_mod
from lit_gpt.quantize import MX4Linear, quantize_mx4

pytestmark = pytest.mark.gpu


def _model(dev, **kw):
    torch.manual_seed(5)
    cfg = model_mod.Config.from_name("iso_kdn_1.3B", n_layer=2, n_head=2, n_embd=128, intermediate_size=392,
                                     kdn_info_scale=64.0, vocab_size=512, **kw)
    return model_mod.GPT(cfg).to(dev).to(torch.bfloat16).eval()


def _idx(dev):
    return torch.randint(0, 500, (2, 40), device=dev, generator=torch.Generator(dev).manual_seed(1))


@torch.no_grad()
def test_head_keeps_its_meaning():
    """``GPT.forward`` takes a linear head's weight alone: its MX4 form gains no bias."""
    dev = gpu_or_skip()
    log("case mx4 head with a bias")
    m = _model(dev)
    with_bias = copy.deepcopy(m)
    with_bias.lm_head = nn.Linear(128, 512).to(dev).to(torch.bfloat16)
    with_bias.lm_head.weight.copy_(m.lm_head.weight)
    with_bias.lm_head.bias.fill_(3.0)
    assert torch.equal(m(_idx(dev)), with_bias(_idx(dev)))
    quantize_mx4(m), quantize_mx4(with_bias)
    assert type(with_bias.lm_head) is MX4Linear
    assert torch.equal(m(_idx(dev)), with_bias(_idx(dev)))
