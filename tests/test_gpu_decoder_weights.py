"""A decoder with a captured step whose model's weights change: its tokens and logits are those of a decoder that never
captured a step before the change."""
import copy

import pytest
import torch

from gpu_util import gpu_or_skip, log
from lit_gpt import _inference, model as model_mod
from lit_gpt.decode import KDNDecoder
from lit_gpt.quantize import quantize_mx4

pytestmark = pytest.mark.gpu


def _model(dev, mixer, seed=3):
    torch.manual_seed(seed)
    cfg = model_mod.Config.from_name(mixer + "_kdn_1.3B", n_layer=2, n_head=2, n_embd=128, intermediate_size=392,
                                     kdn_info_scale=64.0, vocab_size=512)
    return model_mod.GPT(cfg).to(dev).to(torch.bfloat16).eval()


def _churn(dev):
    """Overwrite what the allocator has free."""
    torch.cuda.synchronize()
    for size in (1 << 10, 1 << 14, 1 << 17, 1 << 20, 1 << 23):
        for t in [torch.empty(size // 4, device=dev) for _ in range(40)]:
            t.fill_(float("nan"))
    torch.cuda.synchronize()


def _load_others(m, dev, mixer):
    m.load_state_dict(_model(dev, mixer, seed=4).state_dict())


CHANGES = {"quantize": lambda m, dev, mixer: quantize_mx4(m), "load": _load_others,
           "clear": lambda m, dev, mixer: _inference.clear_inference_caches(m)}


@pytest.mark.parametrize("prompt_len", [4, 40])  # (up to 64 rows rebuild the packed copies)
@pytest.mark.parametrize("change", list(CHANGES))
@pytest.mark.parametrize("mixer", ["iso", "diag"])
def test_generate_after_a_change(mixer, change, prompt_len):
    dev = gpu_or_skip()
    log(f"case decoder {mixer} {change} prompt {prompt_len}")
    m = _model(dev, mixer)
    B = 3
    prompt = torch.randint(0, 500, (B, prompt_len), device=dev)
    dec = KDNDecoder(m, B)
    before, _ = dec.generate(prompt, 5, temperature=0)
    assert dec.graph is not None
    CHANGES[change](m, dev, mixer)
    _churn(dev)
    got, lps = dec.generate(prompt, 5, temperature=0)
    want, want_lps = KDNDecoder(m, B).generate(prompt, 5, temperature=0)
    assert torch.equal(got, want) and torch.equal(lps, want_lps)
    if change == "clear":
        assert torch.equal(got, before)


@pytest.mark.parametrize("change", ["quantize", "clear"])
def test_step_after_a_change(change):
    """The change comes between two steps, with no prompt after it."""
    dev = gpu_or_skip()
    log(f"case decoder step {change}")
    m = _model(dev, "iso")
    idx = torch.randint(0, 500, (2, 10), device=dev)
    graph, eager = KDNDecoder(m, 2), KDNDecoder(m, 2, use_graph=False)
    graph.prefill(idx[:, :4]), eager.prefill(idx[:, :4])
    for t in range(4, 10):
        if t == 7:
            CHANGES[change](m, dev, "iso")
            _churn(dev)
        a, b = eager.step(idx[:, t]).clone(), graph.step(idx[:, t]).clone()
        torch.cuda.synchronize()
        assert torch.equal(a, b), t
    assert graph.state[0].seen_tokens == eager.state[0].seen_tokens == 10


def test_two_decoders_of_one_model():
    """Each captures again by itself; a copy of the model is not concerned."""
    dev = gpu_or_skip()
    log("case two decoders")
    m = _model(dev, "iso")
    kept = copy.deepcopy(m)
    prompt = torch.randint(0, 500, (2, 4), device=dev)
    decs = [KDNDecoder(m, 2), KDNDecoder(m, 2), KDNDecoder(kept, 2)]
    first = [d.generate(prompt, 4, temperature=0)[0] for d in decs]
    graphs = [d.graph for d in decs]
    quantize_mx4(m)
    second = [d.generate(prompt, 4, temperature=0)[0] for d in decs]
    assert torch.equal(second[0], second[1]) and torch.equal(second[2], first[2])
    assert decs[0].graph is not graphs[0] and decs[1].graph is not graphs[1] and decs[2].graph is graphs[2]
