"""Masked attention where calls are large enough for two row tiles a block (from two row tiles an SM
on), against a plain 64-bit implementation on the GPU.

Tolerances are those of the small cases, whose derivation does not look at sizes: 2 roundings of
2^-9 for out, 3 for a gradient, and for a row eight times as much of the larger of its own and
the mean row's norm."""

import math

import pytest
import torch

from test_gpu_masked_attention import DEV, TOL_GRAD, TOL_OUT, check, close, inputs
from xfold_cpu_b200 import _capi, native

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _no_device_error():
    _capi.device_error(clear=True)
    yield
    torch.cuda.synchronize()
    assert _capi.device_error(clear=True) == 0


def reference(q, k, v, dout=None, softcap=0.0, slopes=None, causal=False, prefix=None,
              documents=None):
    """(out[, dq, dk, dv]) in 64 bits, a row of the batch at a time."""
    B, H, nq, d = q.shape
    G, nk = k.shape[1:3]
    rep = H // G
    pos, key = torch.arange(nq, device=DEV) + nk - nq, torch.arange(nk, device=DEV)
    results = []
    for b in range(B):
        vis = torch.ones(nq, nk, dtype=torch.bool, device=DEV)
        if causal:
            vis = key[None] <= pos[:, None]
            if prefix is not None:
                vis = vis | (key < prefix[b])[None]
        if documents is not None:
            qd, kd = (x.expand(B, -1)[b] for x in documents)
            vis = vis & (qd[:, None] == kd[None]) & (kd >= 0)[None]
        some, seen = vis.any(1), vis.any(0)
        # what no query sees, or sees nothing, may hold anything
        qq = torch.where(some[:, None], q[b].double(), 0.0)
        kk, vv = (torch.where(seen[:, None], t[b].double(), 0.0).repeat_interleave(rep, 0)
                  for t in (k, v))
        x = d ** -0.5 * (qq @ kk.transpose(-1, -2))
        t = torch.tanh(x / softcap) if softcap else None
        s = softcap * t if softcap else x
        if slopes is not None:
            s = s - slopes.double()[:, None, None] * (pos[:, None] - key[None]).abs()
        s = s.masked_fill(~vis, -math.inf).masked_fill(~some[:, None], 0.0)
        p = torch.softmax(s, -1).masked_fill(~vis, 0.0)
        out = p @ vv
        row = [out]
        if dout is not None:
            do = torch.where(some[:, None], dout[b].double(), 0.0)
            dx = p * (do @ vv.transpose(-1, -2) - (do * out).sum(-1, keepdim=True)) * d ** -0.5
            if softcap:
                dx = dx * (1 - t * t)
            row += [dx @ kk, (dx.transpose(-1, -2) @ qq).view(G, rep, nk, d).sum(1),
                    (p.transpose(-1, -2) @ do).view(G, rep, nk, d).sum(1)]
        results.append([r.cpu() for r in row])
    return [torch.stack(r) for r in zip(*results)]


def two_row_tiles_a_block(q, k):
    rep = q.shape[1] // k.shape[1]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return q.shape[0] * k.shape[1] * -(-q.shape[2] // (128 // rep)) >= 2 * sms


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("d", [64, 128])
def test_padding_among_the_keys_of_a_block_s_second_tile(d, bad):
    """The second row tile of each block sees none of the first tile's keys, so its list starts
    seven key tiles after the block's; V of its padded keys holds NaN or infinities."""
    H, nq, nk, cut = 80, 256, 903, 7 * 64
    q, k, v, _ = inputs(2, H, H, nq, nk, d, BF16)
    assert two_row_tiles_a_block(q, k)
    q_ids = (torch.arange(nq, device=DEV) >= 128).int()[None]
    k_ids = (torch.arange(nk, device=DEV) >= cut).int().expand(2, nk).clone()
    g = torch.Generator().manual_seed(7)
    k_ids[(torch.rand(2, nk, generator=g) < 0.3).to(DEV)] = -1
    for t in (k, v):
        t.masked_fill_((k_ids < 0)[:, None, :, None], bad)
    ref, = reference(q, k, v, documents=(q_ids, k_ids))
    for save in (False, True):
        got = native.masked_attention(q, k, v, documents=(q_ids, k_ids), save=save)
        close(got[0] if save else got, ref, TOL_OUT[BF16], f"out, save={save}")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tiles", range(1, 8))
def test_every_last_buffer(d, tiles):
    """Two groups of warps take a row tile's key tiles in turn; the last is the one's or the
    other's, in a buffer's first or a later use."""
    q, k, v, _ = inputs(2, 80, 80, 256, 64 * tiles - 5, d, BF16)
    assert two_row_tiles_a_block(q, k)
    ref, = reference(q, k, v)
    for save in (False, True):
        got = native.masked_attention(q, k, v, save=save)
        close(got[0] if save else got, ref, TOL_OUT[BF16], f"out, save={save}")


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("softcap", [1e-300, 1e-40, 1e31, 1e38, 1e300])
def test_caps_that_f32_does_not_hold(dtype, softcap):
    """A tiny cap makes all scores one, without gradients of q and k; a huge one does nothing."""
    q, k, v, dout = inputs(1, 4, 2, 150, 150, 64, dtype)
    check(q, k, v, dout, causal=True, softcap=softcap)
    if softcap > 1:
        assert torch.equal(native.masked_attention(q.float(), k.float(), v.float(),
                                                   softcap=softcap),
                           native.masked_attention(q.float(), k.float(), v.float())) or \
            softcap < 2.0 ** 100


def test_scales_that_f32_does_not_hold():
    q, k, v, _ = inputs(1, 2, 2, 20, 20, 16, BF16)
    for scale in (1e39, -1e300):
        with pytest.raises(ValueError, match="scale"):
            native.masked_attention(q, k, v, scale=scale)
    with pytest.raises(ValueError, match="magnitude"):
        native.rotary(q, k, native.rotary_frequencies(16).to(DEV), magnitude=1e39)


SLOPES = [2.0 ** (-h / 2 - 1) for h in range(16)]


def mask_options(which, B, H, n, qkvo):
    """Options of a call; documents have padding inside and at the end, which holds NaN."""
    options = {}
    if "cap" in which:
        options["softcap"] = 3.0
    if "slopes" in which:
        options["slopes"] = torch.tensor([SLOPES[h % 16] for h in range(H)], device=DEV)
    if "causal" in which or "prefix" in which:
        options["causal"] = True
    if "prefix" in which:
        options["prefix"] = torch.tensor([n // 2 - 60 * b for b in range(B)], dtype=torch.int32,
                                         device=DEV)
    if "documents" in which:
        g = torch.Generator().manual_seed(9)
        ids = torch.arange(n).div(n // 3 + 1, rounding_mode="floor").int().repeat(B, 1)
        ids[torch.rand(B, n, generator=g) < 0.1] = -1
        ids[:, 70:75], ids[-1, n - 40:] = -1, -1
        ids = ids.to(DEV)
        options["documents"] = (ids, ids)
        for t in qkvo:
            t.masked_fill_((ids < 0)[:, None, :, None], math.nan)
    return options


MASKS = ["", "causal", "cap", "slopes", "slopes causal", "cap slopes causal", "prefix",
         "prefix slopes", "cap documents", "slopes causal documents", "causal documents"]


@pytest.mark.parametrize("which", MASKS)
@pytest.mark.parametrize("B,H,G,n,d", [(2, 80, 80, 300, 64), (2, 80, 20, 300, 128),
                                       (1, 120, 40, 333, 64), (2, 80, 80, 290, 24),
                                       (1, 150, 150, 259, 128)])
def test_two_row_tiles_a_block(B, H, G, n, d, which):
    """One head, four and three (whose tiles have 126 rows) to a K/V head, without the statistics
    (P in one part) and with them, and the gradients of so many heads."""
    q, k, v, dout = inputs(B, H, G, n, n, d, BF16)
    assert two_row_tiles_a_block(q, k)
    options = mask_options(which, B, H, n, (q, k, v, dout))
    ref = reference(q, k, v, dout, **options)
    close(native.masked_attention(q, k, v, **options), ref[0], TOL_OUT[BF16], "out without save")
    out, saved = native.masked_attention(q, k, v, save=True, **options)
    close(out, ref[0], TOL_OUT[BF16], "out")
    grads = native.masked_attention_backward(dout, q, k, v, out, saved, **options)
    for name, got, want in zip(("dq", "dk", "dv"), grads, ref[1:]):
        close(got, want, TOL_GRAD[BF16], name)


@pytest.mark.parametrize("which", MASKS)
@pytest.mark.parametrize("B,H,G,n,d", [(1, 4, 4, 1100, 64), (2, 4, 2, 700, 128),
                                       (1, 6, 2, 601, 128), (1, 8, 1, 530, 48)])
def test_gradients_in_one_part(B, H, G, n, d, which):
    """More than 512 tokens: several row and key tiles a block, P and dX rounded once."""
    q, k, v, dout = inputs(B, H, G, n, n, d, BF16)
    options = mask_options(which, B, H, n, (q, k, v, dout))
    ref = reference(q, k, v, dout, **options)
    out, saved = native.masked_attention(q, k, v, save=True, **options)
    close(out, ref[0], TOL_OUT[BF16], "out")
    grads = native.masked_attention_backward(dout, q, k, v, out, saved, **options)
    for name, got, want in zip(("dq", "dk", "dv"), grads, ref[1:]):
        close(got, want, TOL_GRAD[BF16], name)


@pytest.mark.parametrize("length", [2, 3, 37])
@pytest.mark.parametrize("causal", [False, True])
def test_gradients_of_short_documents_in_long_rows(length, causal):
    q, k, v, dout = inputs(1, 4, 2, 1300, 1300, 64, BF16)
    ids = (torch.arange(1300, device=DEV) // length).int()[None]
    options = dict(causal=causal, documents=(ids, ids))
    ref = reference(q, k, v, dout, **options)
    out, saved = native.masked_attention(q, k, v, save=True, **options)
    grads = native.masked_attention_backward(dout, q, k, v, out, saved, **options)
    for name, got, want in zip(("dq", "dk", "dv"), grads, ref[1:]):
        close(got, want, TOL_GRAD[BF16], name)


@pytest.mark.parametrize("nq,nk", [(1, 2000), (5, 700), (700, 90), (130, 1500)])
@pytest.mark.parametrize("d", [64, 128])
def test_gradients_in_one_part_of_queries_over_a_cache(nq, nk, d):
    q, k, v, dout = inputs(2, 8, 2, nq, nk, d, BF16)
    options = dict(causal=True, softcap=5.0, slopes=torch.tensor(SLOPES[:8], device=DEV))
    ref = reference(q, k, v, dout, **options)
    out, saved = native.masked_attention(q, k, v, save=True, **options)
    grads = native.masked_attention_backward(dout, q, k, v, out, saved, **options)
    for name, got, want in zip(("dq", "dk", "dv"), grads, ref[1:]):
        close(got, want, TOL_GRAD[BF16], name)
