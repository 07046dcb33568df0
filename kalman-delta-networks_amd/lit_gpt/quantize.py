"""A ``GPT`` whose SwiGLU and head weights are held in MX4 (4.25 bits an element), for decoding.

The reference has no counterpart: its models run in bf16 and fp32.  The SwiGLU and the head hold two thirds of the
1.3B models' weights; the mixers, whose recurrences carry every rounding of their gates on, keep bf16.

    model = GPT.from_name("iso_kdn_1.3B").cuda().to(torch.bfloat16).eval()
    quantize_mx4(model)                      # in place
    dec = KDNDecoder(model, batch_size=B)
    tokens, logprobs = dec.generate(prompt, 128, temperature=0.8, top_p=0.95)
"""
from __future__ import annotations

import warnings

import torch
from torch import nn

from ._inference import clear_inference_caches, parts_exchanged
from .kdn_ops.mx4 import MX4Tensor, mx4_linear, mx4_quantize
from .model import GPT, LLaMAMLP, SwiGLU


def _hold(module: nn.Module, name: str, weight: torch.Tensor) -> None:
    t = mx4_quantize(weight.detach())
    module.register_buffer(name + "_codes", t.codes)
    module.register_buffer(name + "_scales", t.scales)


class MX4Linear(nn.Module):
    """``nn.Linear`` with an MX4 weight (bf16 activations, no backward).  ``bias`` False leaves its bias out."""

    def __init__(self, linear: nn.Linear, bias: bool = True) -> None:
        super().__init__()
        self.in_features, self.out_features = linear.in_features, linear.out_features
        _hold(self, "weight", linear.weight)
        keep = linear.bias if bias else None
        self.register_buffer("bias", None if keep is None else keep.detach().to(torch.bfloat16).clone())

    @property
    def mx4(self) -> MX4Tensor:
        return MX4Tensor(self.weight_codes, self.weight_scales, self.in_features)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return mx4_linear(x, self.mx4, self.bias)


class MX4SwiGLU(nn.Module):
    """``SwiGLU`` with MX4 weights, w1 and w2 packed: w3(silu(w1 x) * w2 x)."""

    def __init__(self, swiglu: SwiGLU) -> None:
        super().__init__()
        self.in_features, self.hidden_features = swiglu.w1.in_features, swiglu.w1.out_features
        _hold(self, "w12", torch.cat((swiglu.w1.weight.detach(), swiglu.w2.weight.detach())))
        _hold(self, "w3", swiglu.w3.weight)
        bf16 = lambda b: b.detach().to(torch.bfloat16)  # noqa: E731
        self.register_buffer("b12", None if swiglu.w1.bias is None else torch.cat((bf16(swiglu.w1.bias), bf16(swiglu.w2.bias))))
        self.register_buffer("b3", None if swiglu.w3.bias is None else bf16(swiglu.w3.bias).clone())

    @property
    def w12(self) -> MX4Tensor:
        return MX4Tensor(self.w12_codes, self.w12_scales, self.in_features)

    @property
    def w3(self) -> MX4Tensor:
        return MX4Tensor(self.w3_codes, self.w3_scales, self.hidden_features)

    def forward(self, x: torch.Tensor, residual=None) -> torch.Tensor:
        return mx4_linear(mx4_linear(x, self.w12, self.b12, gated=True), self.w3, self.b3, residual=residual)


def _is_linear(module) -> bool:
    """The call is the product with ``module.weight`` and the bias (a parametrised weight's value included)."""
    return isinstance(module, nn.Linear) and type(module).forward is nn.Linear.forward and "forward" not in module.__dict__


def _is_swiglu(module) -> bool:
    return type(module) is SwiGLU and "forward" not in module.__dict__ and all(_is_linear(m) for m in (module.w1, module.w2, module.w3))


@torch.no_grad()
def quantize_mx4(model: GPT, *, head: bool = True) -> GPT:
    """Replaces every block's SwiGLU and, with ``head``, the head by their MX4 forms, in place; returns ``model``.

    The weights must be on the GPU.  Activations must be bf16 (a bf16 model) and the model is for inference: its MX4
    products refuse inputs that need a gradient.  The replaced weights are released, packed copies of them too (by a
    ``KDNDecoder`` that has captured its step, at its next call, which captures it again), and hooks on the replaced
    parts with them.  A part of another type, whose call may be more than its weights' products, stays as it is, with a
    warning that names it."""
    if not isinstance(model, GPT):
        raise TypeError(f"quantize_mx4 takes a GPT, got {type(model).__name__}")
    clear_inference_caches(model)
    parts_exchanged(model)
    kept = []
    for i, block in enumerate(model.transformer.h):
        mlp = getattr(block, "mlp", None)
        swiglu = getattr(mlp, "swiglu", None)
        if type(mlp) is LLaMAMLP and _is_swiglu(swiglu):
            mlp.swiglu = MX4SwiGLU(swiglu)
        elif mlp is not None and not (type(mlp) is LLaMAMLP and type(swiglu) is MX4SwiGLU):
            kept.append(f"transformer.h.{i}.mlp")
    if head and _is_linear(model.lm_head):
        model.lm_head = MX4Linear(model.lm_head, bias=False)  # (``GPT.forward`` takes a linear head's weight alone)
    elif head and type(model.lm_head) is not MX4Linear:
        kept.append("lm_head")
    if kept:
        warnings.warn(f"quantize_mx4 leaves parts of other types than the model's own as they are: {', '.join(kept)}", stacklevel=3)
    return model


__all__ = ("MX4Linear", "MX4SwiGLU", "quantize_mx4")
