"""More rows than one launch holds (its threads are counted in 32 bits, 1024 to a row)."""
import pytest
import torch

from gpu_util import gpu_or_skip, log
from lit_gpt.kdn_ops.sampling import sample_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("settings", [dict(temperature=0.0), dict(), dict(top_k=1), "per row"], ids=str)
def test_many_rows(settings):
    dev = gpu_or_skip()
    B, V = (1 << 22) + 5, 3
    log(f"case sample {B} rows {settings}")
    g = torch.Generator(device=dev).manual_seed(1)
    logits = torch.randn(B, V, generator=g, device=dev)
    noise = torch.empty(B, V, device=dev).exponential_(generator=g)
    greedy = torch.zeros(B, dtype=torch.bool, device=dev)
    if settings == "per row":
        greedy[::3] = True
        settings = dict(temperature=torch.where(greedy, 0.0, 1.0))
    elif settings:
        greedy[:] = True
    tokens, lps = sample_tokens(logits, noise, **settings)
    score = logits.double() - noise.double().log()
    want = torch.where(greedy, logits.argmax(-1), score.argmax(-1))
    # a draw whose two best scores differ by less than their fp32 quotients' rounding may take either
    best = score.topk(2, -1).values
    clear = greedy | (best[:, 0] - best[:, 1] > 1e-6)
    assert bool((tokens == want)[clear].all()) and bool(((tokens >= 0) & (tokens < V)).all())
    lp = torch.log_softmax(logits.double(), -1).gather(1, tokens.unsqueeze(1)).squeeze(1)
    assert bool(((lps.double() - lp).abs() <= 2e-6 * (1 + lp.abs())).all())
