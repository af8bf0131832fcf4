"""Strides of dimensions of size one, which say nothing: zero (slices of broadcast tensors), odd, or far
out of range."""

import pytest
import torch

from test_gpu_masked_attention import DEV, check, inputs

pytestmark = pytest.mark.gpu


def with_strides(t, stride):
    """`t` with `stride` for its dimensions of size one."""
    return t.as_strided(t.shape, [stride if n == 1 and i < 3 else s
                                  for i, (n, s) in enumerate(zip(t.shape, t.stride()))])


@pytest.mark.parametrize("stride", [0, 1, 7, 1 << 41])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 64), (1, 1, 1, 1, 50, 64), (2, 4, 4, 1, 1, 64),
                                   (1, 1, 1, 300, 300, 64), (1, 8, 1, 1, 200, 128),
                                   (3, 1, 1, 200, 200, 32), (1, 6, 2, 20, 1, 64),
                                   (1, 4, 4, 150, 150, 64), (2, 2, 1, 1, 3, 16)])
def test_attention(shape, stride):
    q, k, v, dout = (with_strides(t, stride) for t in inputs(*shape, torch.bfloat16))
    check(q, k, v, dout, causal=True)
