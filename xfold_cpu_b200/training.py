"""Differentiable forms of the training operators, for torch's autograd.

masked_attention, rotary and layer_norm are the functions of the same names in `native`
(layer_norm: layer_norm_forward) with their hand-written backward passes behind
torch.autograd.Function; linear is a projection on the library's bf16 GEMM with its gradients.
Their results carry gradients to q, k, v, x, weight and bias; masks, positions, slopes and
frequencies are constants, and must not be changed in place before the backward pass.  Where no
gradient is wanted (torch.no_grad, or no input requires one) nothing is saved.  Gradients of
gradients are refused.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import native


def _masks(slopes, prefix, documents, key_documents):
    """native.masked_attention's masks; without key documents the others serve for both."""
    return dict(slopes=slopes, prefix=prefix, documents=documents if key_documents is None
                else (documents, key_documents))


class _MaskedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, prefix, documents, key_documents, options):
        masks = _masks(slopes, prefix, documents, key_documents)
        out, (lse, low) = native.masked_attention(q, k, v, save=True, **masks, **options)
        ctx.options = options
        # the masks too: the backward pass makes the scores again, and a mask that was changed in
        # place since would give gradients of another function
        ctx.save_for_backward(q, k, v, out, lse, low, slopes, prefix, documents, key_documents)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, low, *masks = ctx.saved_tensors
        dq, dk, dv = native.masked_attention_backward(dout, q, k, v, out, (lse, low),
                                                      **_masks(*masks), **ctx.options)
        return dq, dk, dv, None, None, None, None, None


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, frequencies, positions, options):
        ctx.save_for_backward(frequencies, positions)
        ctx.options = options
        return native.rotary(q, k, frequencies, positions=positions, **options)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        frequencies, positions = ctx.saved_tensors
        dq, dk = native.rotary_backward(dq, dk, frequencies, positions=positions, **ctx.options)
        return dq, dk, None, None, None


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = native.layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = native.layer_norm_backward(dy, x, weight, mean, rstd)
        return (dx, None if weight is None else dw.to(weight.dtype),
                None if ctx.bias_dtype is None else db.to(ctx.bias_dtype), None)


def _linear(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    return native.linear(x, weight, out_dtype=torch.bfloat16).to(x.dtype)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight):
        ctx.save_for_backward(x, weight)
        return _linear(x, weight)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        n, k = weight.shape
        dy2, x2 = dy.reshape(-1, n), x.reshape(-1, k)
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = native.linear(dy2, weight.t(), out_dtype=torch.bfloat16).to(x.dtype).view(x.shape)
        rows = x2.shape[0]
        if ctx.needs_input_grad[1] and rows == 0:
            dw = torch.zeros_like(weight)
        elif ctx.needs_input_grad[1]:
            pad = -rows % 8  # the GEMM reads 16-byte rows along its reduction too
            a, b = dy2.to(torch.bfloat16), x2.to(torch.bfloat16)
            if pad:
                a = torch.cat((a, a.new_zeros(pad, n)))
                b = torch.cat((b, b.new_zeros(pad, k)))
            dw = native.gemm(a.unsqueeze(0), b.unsqueeze(0), mn_major=True)[0].to(weight.dtype)
        return dx, dw


def _records(*inputs: torch.Tensor | None) -> bool:
    """Whether autograd is to record a call; inside a Function it cannot be seen any more."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in inputs)


def _constant(what: str, t: torch.Tensor | None) -> None:
    if t is not None and t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what} get no gradient here; pass them detached")


def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                     scale: float | None = None, softcap: float = 0.0,
                     slopes: torch.Tensor | None = None, causal: bool = False,
                     prefix: torch.Tensor | None = None, documents=None) -> torch.Tensor:
    """native.masked_attention with gradients to q, k and v."""
    _constant("slopes", slopes)
    if not _records(q, k, v):
        return native.masked_attention(q, k, v, scale=scale, softcap=softcap, slopes=slopes,
                                       causal=causal, prefix=prefix, documents=documents)
    documents, key_documents = native._document_pair(documents)
    if key_documents is documents:
        key_documents = None
    return _MaskedAttention.apply(q, k, v, slopes, prefix, documents, key_documents,
                                  dict(scale=scale, softcap=softcap, causal=causal))


def rotary(q: torch.Tensor, k: torch.Tensor, frequencies: torch.Tensor, *,
           positions: torch.Tensor | None = None, offset: int = 0, interleaved: bool = False,
           magnitude: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """native.rotary with gradients to q and k."""
    _constant("frequencies", frequencies)
    if not _records(q, k):
        return native.rotary(q, k, frequencies, positions=positions, offset=offset,
                             interleaved=interleaved, magnitude=magnitude)
    return _Rotary.apply(q, k, frequencies, positions,
                         dict(offset=offset, interleaved=interleaved, magnitude=magnitude))


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """LayerNorm over the last dimension with gradients to x, weight and bias."""
    if not _records(x, weight, bias):
        return native.layer_norm_forward(x, weight, bias, eps)[0]
    return _LayerNorm.apply(x, weight, bias, eps)


def linear(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """x @ weight^T in bf16 with f32 accumulation (both dimensions of weight multiples of 8)."""
    if not _records(x, weight):
        return _linear(x, weight)
    return _Linear.apply(x, weight)
