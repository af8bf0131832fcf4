"""PackedAttention's host side, without a device."""

import pytest
import torch

from xfold_cpu_b200 import native
from xfold_cpu_b200.nn import PackedAttention


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.half(),
                                  lambda m: m.double(), lambda m: m.to("cpu", torch.bfloat16),
                                  lambda m: torch.nn.Sequential(m).bfloat16()[0]])
def test_casts_keep_frequencies_and_slopes(cast):
    layer = PackedAttention(96, 6, 2, head_dim=128, distance=True, stretch=4.0)
    slopes = layer.slopes.clone()
    layer = cast(layer)
    assert layer.qkv.dtype != torch.float32
    assert layer.frequencies.dtype == layer.slopes.dtype == torch.float32
    assert torch.equal(layer.frequencies, native.rotary_frequencies(128, stretch=4.0))
    assert torch.equal(layer.slopes, slopes)
    assert PackedAttention(64, 2).bfloat16().slopes is None


def test_steps_outside_the_cache_are_refused():
    """Before anything is written: a negative index would be taken from the cache's end, and one
    row broadcast over the others."""
    layer = PackedAttention(64, 2)
    cache = layer.cache(3, 10)
    for t in cache:
        t.zero_()
    for x, filled, word in ((torch.zeros(3, 1, 64), -2, "filled"),
                            (torch.zeros(1, 1, 64), 0, "row"), (torch.zeros(3, 4, 64), 7, "full")):
        with pytest.raises(ValueError, match=word):
            layer.step(x.bfloat16(), cache, filled)
    assert not cache[0].any() and not cache[1].any()
