"""The example decoder: prompts and captured steps run, repeat, and agree with one another."""
import importlib.util
import os

import pytest

import vkb

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("decode_step", os.path.join(ROOT, "examples", "decode_step.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_runs_and_repeats(cuda, example):
    import torch
    made, d = example.run(layers=2, batch=3, prompt=70, tokens=6, seed=1)
    again, _ = example.run(layers=2, batch=3, prompt=70, tokens=6, seed=1)
    assert made.shape == (6, 3) and torch.equal(made, again) and vkb.device_status() == 0
    assert bool(((made >= 0) & (made < example.VOCAB)).all())
    assert d.lens.tolist() == [70 + 5, 63 + 5, 56 + 5]


def test_steps_agree_with_the_prompt(cuda, example):
    """The logits of a sequence's last token, taken in as one prompt and token by token, differ by what the 8-bit cache
    (a page's codes rounded again as its scale grows) and fp16 make of two layers: the directions agree to 1e-3."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    tokens = [torch.randint(0, example.VOCAB, (n,), generator=g, device="cuda", dtype=torch.int32) for n in (40, 40)]
    whole = example.Decoder(2, 2, 64).prompt(tokens)
    d = example.Decoder(2, 2, 64)
    d.prompt([t[:30] for t in tokens])
    for i in range(30, 40):
        d.tokens.copy_(torch.stack([t[i] for t in tokens]))
        steps = d.step()
    cos = torch.nn.functional.cosine_similarity(whole, steps, dim=1)
    assert vkb.device_status() == 0 and float(cos.min()) > 0.999, cos
