"""``quantize_mx4`` on models whose parts are not the model's own."""
import copy
import warnings

import pytest
import torch
from torch import nn
from torch.nn.utils import parametrize

from gpu_util import gpu_or_skip, log
from lit_gpt import model as model_mod
from lit_gpt.quantize import MX4Linear, MX4SwiGLU, quantize_mx4

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


class _Adapted(nn.Linear):
    """A linear layer whose call is more than its weight's product."""

    def forward(self, x):
        return super().forward(x) + 1


class _OtherSwiGLU(model_mod.SwiGLU):
    pass


class _OtherMLP(model_mod.LLaMAMLP):
    pass


@torch.no_grad()
def test_exchanged_parts_stay_and_are_named():
    dev = gpu_or_skip()
    log("case quantize_mx4 with exchanged parts")
    m = _model(dev)
    mlps = [b.mlp for b in m.transformer.h]

    def expect(where, build):
        other = copy.deepcopy(m)
        build(other)
        part = copy.deepcopy(other.transformer.h[1].mlp)
        with pytest.warns(UserWarning, match=where):
            quantize_mx4(other)
        x = torch.randn(2, 100, 128, device=dev, generator=torch.Generator(dev).manual_seed(2)).bfloat16()
        assert type(other.transformer.h[0].mlp.swiglu) is MX4SwiGLU
        if "head" not in where:
            assert torch.equal(other.transformer.h[1].mlp(x), part(x)) and type(other.lm_head) is MX4Linear
        return other

    def adapted(name):
        def build(o):
            sw = o.transformer.h[1].mlp.swiglu
            old = getattr(sw, name)
            setattr(sw, name, _Adapted(old.in_features, old.out_features, bias=False).to(dev).to(torch.bfloat16))
        return build

    for name in ("w1", "w2", "w3"):
        expect(r"transformer\.h\.1\.mlp", adapted(name))
    expect(r"transformer\.h\.1\.mlp", lambda o: setattr(o.transformer.h[1].mlp, "swiglu", _OtherSwiGLU(128, 392).to(dev).bfloat16()))
    expect(r"transformer\.h\.1\.mlp", lambda o: setattr(o.transformer.h[1], "mlp", _OtherMLP(m.config).to(dev).bfloat16()))
    head = _Adapted(128, 512, bias=False).to(dev).to(torch.bfloat16)
    assert expect("lm_head", lambda o: setattr(o, "lm_head", head)).lm_head is head
    # nothing to say: a second call, a head that is to stay, a parametrised weight (its value is what is quantised)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        other = copy.deepcopy(m)
        other.lm_head = head
        quantize_mx4(quantize_mx4(other, head=False), head=False)
        other = copy.deepcopy(m)

        class Double(nn.Module):
            def forward(self, w):
                return 2 * w
        w3 = other.transformer.h[1].mlp.swiglu.w3
        plain = copy.deepcopy(other)
        plain.transformer.h[1].mlp.swiglu.w3.weight.mul_(2)
        parametrize.register_parametrization(w3, "weight", Double())
        assert torch.equal(quantize_mx4(other)(_idx(dev)), quantize_mx4(plain)(_idx(dev)))
    assert [b.mlp for b in m.transformer.h] == mlps
