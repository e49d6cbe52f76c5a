"""Edge cases of the decode-step operators' boundary that need no GPU."""
import math
import os
import re

import pytest

import vkb


def _freq(turns):
    return [(int(t) % (1 << 64)) / 2.0 ** 64 * 2 * math.pi for t in turns]


@pytest.mark.parametrize("rot,base,original,factor", [(128, 10000.0, 131072, 4.0), (64, 10000.0, 4096, 8.0), (128, 500.0, 8192, 2.0), (96, 1e6, 32768, 4.0)])
def test_parts_by_how_often_a_pair_turns(rot, base, original, factor):
    """Pair i turns original f_i / 2 pi times; the ramp is linear in i between the pair that turns 32 times and the one that
    would turn once (rounded outwards to whole pairs), which need not be among the rotated ones."""
    plain = _freq(vkb.rope_turns(rot, base=base, device="cpu")[0])
    parts = _freq(vkb.rope_turns(rot, base=base, scaling="parts", factor=factor, original=original, device="cpu")[0])
    place = [rot / 2 * math.log(original / (2 * math.pi * t)) / math.log(base) for t in (32.0, 1.0)]
    lo, hi = max(0, math.floor(place[0])), math.ceil(place[1])
    for i, (f, g) in enumerate(zip(plain, parts)):
        kept = 1 - min(1.0, max(0.0, (i - lo) / (hi - lo)))
        assert abs(g / (f * (kept + (1 - kept) / factor)) - 1) < 1e-9, i
        if original * f / (2 * math.pi) > 32:
            assert abs(g / f - 1) < 1e-12, i
    last = original * plain[-1] / (2 * math.pi)
    assert (parts[-1] / plain[-1] > 1 / factor + 1e-3) == (last > 1.1)      # divided in full only where it turns less than once


def test_no_non_coherent_loads_of_what_an_earlier_grid_writes():
    """These kernels are launched while the grid before may still be writing their inputs. Loads through the non-coherent path
    are for data that nobody writes while the kernel is resident; griddepcontrol.wait promises nothing for them."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "volta-kernel-bakeoff_b200", "csrc")
    for name in ("step.cuh", "norm.cu", "kv_cache.cu", "attention.cu", "attn_common.cuh", "attn_token.cuh", "attn_prompt.cuh", "sample.cu"):
        with open(os.path.join(root, name)) as f:
            text = f.read()
        for word in ("__ldg", ".nc.", "__restrict__"):
            assert word not in text, (name, word)


def test_arguments_that_are_no_tensors_are_refused():
    """None or a list in the place of a tensor is a refusal like any other, not an AttributeError."""
    import torch
    x = torch.zeros(2, 64)
    for name, call in {"x": lambda: vkb.rms_norm(None, x[0]), "logits": lambda: vkb.sample([0.0], x[0]),
                       "cache": lambda: vkb.attention(None, x, x, x), "k": lambda: vkb.KvCache(None, x, x, x)}.items():
        with pytest.raises(vkb.VkbError, match=name):
            call()


def test_grids_ask_the_device_for_its_sms():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "volta-kernel-bakeoff_b200", "csrc")
    for name in ("norm.cu", "kv_cache.cu", "attention.cu", "sample.cu"):
        with open(os.path.join(root, name)) as f:
            code = [line.split("//")[0] for line in f]
        assert not any(re.search(r"\b148\b", line) for line in code), name
