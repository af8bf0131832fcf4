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


IDS = torch.tensor([0, 1 << 32, 1 << 31, MOST, -1, -(1 << 32), MOST - 1, 7, (1 << 32) + 7, 1 << 40])


def some_ids(rows, n, seed, length=9):
    """Runs of ids whose low 32 bits agree or look negative; some ids come back later."""
    g = torch.Generator().manual_seed(seed)
    runs = IDS[torch.randint(0, len(IDS), (rows, n), generator=g)]
    return runs.repeat_interleave(length, 1)[:, :n]


def small(*ids):
    """The same documents as small numbers, row by row in the order in which they first come: the
    order decides which tiles are left out, and with it how sums are cut in two."""
    rows = max(t.shape[0] for t in ids)
    out = [[] for _ in ids]
    for b in range(rows):
        number = {}
        for t, to in zip(ids, out):
            to.append([-1 if i < 0 else number.setdefault(i, len(number))
                       for i in t.expand(rows, -1)[b].tolist()])
    return [torch.tensor(to, dtype=torch.int32) for to in out]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("causal", [False, True])
def test_documents(dtype, causal):
    """Every form of 64-bit ids gives the bits that small 32-bit ids give."""
    B, n = 3, 301
    q, k, v, dout = inputs(B, 4, 2, n, n, 64, dtype)
    wide = some_ids(B, n, 1)
    same, = small(wide)
    strided = torch.stack((wide, wide + 1), 1).to(DEV)[:, 0]
    for given, want in ((wide, same), (strided, same), (wide[0], small(wide[:1])[0]),
                        (wide[:1].expand(B, n), small(wide[:1])[0])):
        got = training_step(q, k, v, dout, causal, given.to(DEV))
        for a, b in zip(got, training_step(q, k, v, dout, causal, want.to(DEV))):
            assert torch.equal(a, b)


def training_step(q, k, v, dout, causal, documents):
    options = dict(causal=causal, documents=documents)
    out, saved = native.masked_attention(q, k, v, save=True, **options)
    return (out, *native.masked_attention_backward(dout, q, k, v, out, saved, **options))


@pytest.mark.parametrize("narrow", ["none", "queries", "keys"])
def test_documents_of_queries_and_keys(narrow):
    B, nq, nk = 2, 40, 500
    q, k, v, dout = inputs(B, 4, 2, nq, nk, 64, torch.bfloat16)
    q_ids, k_ids = some_ids(B, nq, 2, 3), some_ids(B, nk, 3, 20)
    if narrow == "queries":
        q_ids = q_ids.clamp(-1, 7).int()
    if narrow == "keys":
        k_ids = k_ids.clamp(-1, 7).int()[:1]
    ks, qs = small(k_ids.long(), q_ids.long())  # keys first, then queries
    got = training_step(q, k, v, dout, True, (q_ids.to(DEV), k_ids.to(DEV)))
    for a, b in zip(got, training_step(q, k, v, dout, True, (qs.to(DEV), ks.to(DEV)))):
        assert torch.equal(a, b)


def test_many_documents():
    """A document a token, in an order that fills the table everywhere."""
    n = 5000
    q, k, v, _ = inputs(1, 1, 1, n, n, 16, torch.bfloat16)
    ids = torch.randperm(n, generator=torch.Generator().manual_seed(5)) * 0x100000001 + (1 << 33)
    assert torch.equal(native.masked_attention(q, k, v, documents=ids.to(DEV)), v)
