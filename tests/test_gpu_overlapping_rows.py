"""Rows that overlap in memory (windows that slide by one value), as a user's `unfold` makes them."""

import pytest
import torch

from test_gpu_masked_attention import DEV, check
from test_gpu_rotary import check as check_rotary
from xfold_cpu_b200 import native

pytestmark = pytest.mark.gpu


def windows(B, H, n, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(B, H, n + d - 1, generator=g).to(dtype).to(DEV).unfold(-1, d, 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [20, 100])
def test_attention(n, dtype):
    q, k, v, dout = (windows(2, h, n, 64, dtype, i) for i, h in enumerate((4, 2, 2, 4)))
    check(q, k, v, dout, causal=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [20, 100])
def test_rotary(n, dtype):
    check_rotary(windows(2, 4, n, 64, dtype, 0), windows(2, 2, n, 64, dtype, 1),
                 native.rotary_frequencies(48).to(DEV))
