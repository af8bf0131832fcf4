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
