"""Prefixes, positions and document ids in 64 bits: values that 32 bits do not hold."""

import pytest
import torch

from test_gpu_masked_attention import DEV, check, inputs
from xfold_cpu_b200 import native

pytestmark = pytest.mark.gpu

MOST = torch.iinfo(torch.int64).max


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prefixes(dtype):
    q, k, v, dout = inputs(5, 2, 2, 150, 150, 32, dtype)
    prefix = torch.tensor([MOST, (1 << 32) + 3, 1 << 31, -MOST, 40], device=DEV)
    check(q, k, v, dout, causal=True, prefix=prefix)


def test_unsigned_and_short_types():
    q, k, v, _ = inputs(2, 2, 2, 70, 70, 32, torch.bfloat16)
    want = native.masked_attention(q, k, v, causal=True,
                                   prefix=torch.tensor([9, 70], dtype=torch.int32, device=DEV))
    for dtype in (torch.uint8, torch.int8, torch.int16, torch.int64):
        prefix = torch.tensor([9, 70], dtype=dtype, device=DEV)
        assert torch.equal(native.masked_attention(q, k, v, causal=True, prefix=prefix), want)
    wide = torch.tensor([9, (1 << 32) - 1], dtype=torch.int64).to(torch.uint32).to(DEV)
    assert torch.equal(native.masked_attention(q, k, v, causal=True, prefix=wide), want)
    with pytest.raises(ValueError):
        native.masked_attention(q, k, v, causal=True, prefix=torch.zeros(2, device=DEV))
    with pytest.raises(ValueError):
        native.masked_attention(q, k, v, causal=True,
                                prefix=torch.zeros(2, dtype=torch.uint64, device=DEV))
