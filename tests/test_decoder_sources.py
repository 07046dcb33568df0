"""What a decoder keeps of the model for its captured step, and when it takes the model for another one."""
import gc
import weakref

import pytest
import torch

from lit_gpt import _inference
from lit_gpt.model import GPT, SwiGLU


def _model():
    torch.manual_seed(0)
    return GPT.from_name("iso_kdn_1.3B", n_layer=2, n_head=2, n_embd=128, intermediate_size=72, vocab_size=64).eval()


def _changes():
    def load(m):
        m.load_state_dict(m.state_dict())

    def write(m):
        m.transformer.h[1].attn.o_proj.weight.mul_(2)

    def data(m):
        m.lm_head.weight.data = m.lm_head.weight.data.clone()

    def part(m):
        m.transformer.h[1].mlp.swiglu = SwiGLU(128, 72)

    def parameter(m):
        m.transformer.ln_f.weight = torch.nn.Parameter(torch.ones(128))

    def dtype(m):
        m.to(torch.bfloat16)
    return [load, write, data, part, parameter, dtype]


@pytest.mark.parametrize("change", _changes(), ids=lambda f: f.__name__)
@torch.no_grad()
def test_a_change_of_the_weights_is_seen(change):
    m = _model()
    s = _inference.StepSources(m)
    assert s.current() and s.same_parts(m)
    change(m)
    assert not s.current()


def test_exchanged_parts_are_seen_at_every_step():
    m, other = _model(), _model()
    s = _inference.StepSources(m)
    _inference.parts_exchanged(other)
    assert s.same_parts(m)
    _inference.parts_exchanged(m)
    assert not s.same_parts(m) and _inference.StepSources(m).same_parts(m)


@torch.no_grad()
def test_what_the_captured_step_reads_is_kept():
    """Replaced parameters and dropped packed copies live as long as the object does, and no longer."""
    m = _model()
    sw = m.transformer.h[0].mlp.swiglu
    pack = weakref.ref(_inference.packed_weight(sw, "w12", (sw.w1.weight, sw.w2.weight)))
    weight = weakref.ref(sw.w3.weight)
    s = _inference.StepSources(m)
    _inference.clear_inference_caches(m)
    del sw
    m.transformer.h[0].mlp.swiglu = SwiGLU(128, 72)
    gc.collect()
    assert pack() is not None and weight() is not None
    del s
    gc.collect()
    assert pack() is None and weight() is None
