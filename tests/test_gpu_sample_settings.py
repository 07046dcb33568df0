"""Settings that fp32 does not hold are taken as its nearest positive numbers."""
import pytest
import torch

from gpu_util import gpu_or_skip, log
from lit_gpt.kdn_ops.sampling import sample_tokens
from oracle import sample_oracle as so

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("settings", [dict(top_p=1e-50), dict(temperature=1e39), dict(temperature=1e300, top_p=0.5),
                                      dict(temperature=1e-50), dict(min_p=1e-50)], ids=str)
def test_settings_past_fp32(settings):
    dev = gpu_or_skip()
    log(f"case sample {settings}")
    g = torch.Generator().manual_seed(1)
    logits, noise = 2 * torch.randn(4, 999, generator=g), torch.empty(4, 999).exponential_(generator=g)
    tokens, lps = sample_tokens(logits.to(dev), noise.to(dev), **settings)
    for i in range(4):
        want, lp = so.sample(logits[i], noise[i], **settings)
        assert int(tokens[i]) == want
        assert abs(float(lps[i]) - lp) <= 2e-6 * (1 + abs(lp))
