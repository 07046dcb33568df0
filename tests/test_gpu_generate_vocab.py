"""``generate`` over the vocabulary without its padding."""
import pytest
import torch

from gpu_util import gpu_or_skip, log
from lit_gpt import model as model_mod
from lit_gpt.decode import KDNDecoder
from lit_gpt.kdn_ops.sampling import sample_tokens
from lit_gpt.quantize import quantize_mx4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mx4", [False, True])
def test_padding_is_not_drawn(mx4):
    dev = gpu_or_skip()
    log(f"case generate without the padding, mx4 {mx4}")
    torch.manual_seed(2)
    cfg = model_mod.Config.from_name("iso_kdn_1.3B", n_layer=1, n_head=2, n_embd=128, intermediate_size=392,
                                     kdn_info_scale=64.0, vocab_size=500)
    m = model_mod.GPT(cfg).to(dev).to(torch.bfloat16).eval()
    assert cfg.padded_vocab_size == 512
    with torch.no_grad():
        m.lm_head.weight[500:] *= 50  # the largest logits are the padding's
    if mx4:
        quantize_mx4(m)
    B = 3
    prompt = torch.randint(0, 500, (B, 5), device=dev)
    everything, _ = KDNDecoder(m, B).generate(prompt, 6, temperature=0)
    assert bool((everything >= 500).any())
    for settings in (dict(temperature=0), dict(top_p=0.9), dict(top_k=20)):
        g = torch.Generator(dev).manual_seed(7)
        tokens, lps = KDNDecoder(m, B).generate(prompt, 6, vocab_size=500, generator=g, **settings)
        assert bool((tokens < 500).all()) and bool((tokens >= 0).all())
        ref = KDNDecoder(m, B, use_graph=False)
        g = torch.Generator(dev).manual_seed(7)
        logits = ref.prefill(prompt)[:, -1]
        for i in range(6):
            noise = torch.empty(B, 500, device=dev).exponential_(generator=g) if settings.get("temperature") != 0 else None
            want, lp = sample_tokens(logits[:, :500].contiguous(), noise, **settings)
            assert torch.equal(tokens[:, i], want) and torch.equal(lps[:, i], lp)
            logits = ref.step(want).clone()
    for bad in (0, 513, -1):
        with pytest.raises(ValueError, match="vocab_size"):
            KDNDecoder(m, B).generate(prompt, 1, vocab_size=bad)
