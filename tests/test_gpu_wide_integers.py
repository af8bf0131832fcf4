"""Prefixes, positions and document ids in 64 bits: values that 32 bits do not hold."""

import pytest
import torch

from test_gpu_masked_attention import DEV, check, inputs
from test_gpu_rotary import reference as rotary_reference
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_positions(dtype, interleaved):
    """Positions around 2^32 and below zero.  An angle of 2^33 has a rounding of 2^-53 of it in the
    reference and two in the kernel, 3e-6, beside the small positions' 1e-6 (f32) or 2^-9."""
    q, k = (t[0] for t in (inputs(2, 3, 1, 40, 40, 64, dtype)[:1], inputs(2, 1, 1, 40, 40, 64, dtype)[:1]))
    freq = native.rotary_frequencies(48).to(DEV)
    positions = torch.arange(40).expand(2, 40) * 107_000_003 + torch.tensor([[1 << 31], [-(1 << 32)]])
    got = native.rotary(q, k, freq, positions=positions.to(DEV), interleaved=interleaved)
    tol = 4e-6 + (2.0 ** -9 if dtype == torch.bfloat16 else 0.0)
    for x, y in zip((q, k), got):
        ref = rotary_reference(x, freq, positions, interleaved, 1.0)
        assert (y.cpu().double() - ref).norm().item() <= tol * ref.norm().item()
    small = torch.arange(40, device=DEV) * 7
    for other in (torch.int16, torch.int64, torch.uint32):
        a = native.rotary(q, k, freq, positions=small.to(other), interleaved=interleaved)
        b = native.rotary(q, k, freq, positions=small.int(), interleaved=interleaved)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
