"""What torch's autograd asks of the differentiable operators beside the gradients' values."""

import pytest
import torch

from xfold_cpu_b200 import native, training

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda")


def tensors(*shape, count=3, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(0)
    return [torch.randn(*shape, generator=g).to(dtype).to(DEV).requires_grad_()
            for _ in range(count)]


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("name,mask", [
    ("documents", lambda: ints(*[0] * 9 + [1] * 11)),
    ("slopes", lambda: torch.tensor([0.5, 0.25], device=DEV)),
    ("prefix", lambda: ints(3))])
def test_a_mask_changed_before_the_backward_pass(name, mask):
    q, k, v = tensors(1, 2, 20, 16)
    mask = mask()
    options = {name: mask, "causal": True}
    out = training.masked_attention(q, k, v, **options)
    mask += 1
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()


@pytest.mark.parametrize("which", [0, 1])
def test_documents_of_queries_or_keys_changed_before_the_backward_pass(which):
    q, k, v = tensors(1, 2, 20, 16)
    documents = ints(*[0] * 20), ints(*[0] * 15 + [1] * 5)
    out = training.masked_attention(q, k, v, documents=documents)
    documents[which].fill_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()


@pytest.mark.parametrize("which", [0, 1])
def test_positions_or_frequencies_changed_before_the_backward_pass(which):
    q, k = tensors(1, 2, 20, 16, count=2)
    constants = native.rotary_frequencies(16).to(DEV), torch.arange(20, device=DEV)
    out = training.rotary(q, k, constants[0], positions=constants[1])
    constants[which].mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        (out[0].sum() + out[1].sum()).backward()


def test_forms_of_documents_give_the_same_gradients():
    ids = ints(*[0] * 9 + [1] * 11)
    grads = []
    for documents in (ids, ids.long(), (ids, ids), (ids, ids.clone()), [ids, ids.long()]):
        q, k, v = tensors(1, 2, 20, 16)
        training.masked_attention(q, k, v, documents=documents, causal=True).sum().backward()
        grads.append((q.grad, k.grad, v.grad))
    for other in grads[1:]:
        for a, b in zip(grads[0], other):
            assert torch.equal(a, b)


def test_constants_that_want_a_gradient_are_refused():
    q, k, v = tensors(1, 2, 20, 16)
    slopes = torch.tensor([0.5, 0.25], device=DEV, requires_grad=True)
    frequencies = native.rotary_frequencies(16).to(DEV).requires_grad_()
    with pytest.raises(RuntimeError, match="slopes"):
        training.masked_attention(q, k, v, slopes=slopes)
    with pytest.raises(RuntimeError, match="frequencies"):
        training.rotary(q, k, frequencies)
    training.masked_attention(q, k, v, slopes=slopes.detach()).sum().backward()
    with torch.no_grad():
        training.masked_attention(q, k, v, slopes=slopes)
        training.rotary(q, k, frequencies)


@pytest.mark.parametrize("grad_mode", [False, True])
def test_calls_that_need_no_gradient_save_nothing(monkeypatch, grad_mode):
    """Under no_grad on inputs that require a gradient, and with gradients on for inputs that do
    not, nothing goes through autograd and the attention keeps no statistics."""
    calls = []
    whole = native.masked_attention
    monkeypatch.setattr(native, "masked_attention",
                        lambda *a, **o: calls.append(o.get("save", False)) or whole(*a, **o))
    for name in ("_MaskedAttention", "_Rotary", "_LayerNorm", "_Linear"):
        monkeypatch.setattr(getattr(training, name), "apply", None)
    q, k, v = tensors(1, 2, 24, 16)
    x, w = tensors(24, 16, count=2)
    frequencies = native.rotary_frequencies(16).to(DEV)
    if grad_mode:
        q, k, v, x, w = (t.detach() for t in (q, k, v, x, w))
    with torch.set_grad_enabled(grad_mode):
        results = [training.masked_attention(q, k, v), training.layer_norm(x, w[0], w[1]),
                   training.linear(x, w), *training.rotary(q, k, frequencies)]
    assert calls == [False]
    assert not any(t.requires_grad for t in results)


@pytest.mark.parametrize("call,count", [
    (lambda a, b: training.linear(a, b), 2),
    (lambda a, b: training.layer_norm(a, b[0], b[1]), 2),
    (lambda a, b: training.rotary(a[None, None], b[None, None],
                                  native.rotary_frequencies(16).to(DEV))[0], 1),
    (lambda a, b: training.masked_attention(a[None, None], b[None, None], b[None, None]), 2)])
def test_gradients_of_gradients_are_refused(call, count):
    """Not left out: what a second backward pass would get through these is missing."""
    inputs = tensors(24, 16, count=2)
    w = torch.randn(24, 1, device=DEV).bfloat16().requires_grad_()
    out = (call(*inputs) * w).float().square().sum()
    grads = torch.autograd.grad(out, inputs[:count], create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        sum(g.float().square().sum() for g in grads).backward()


def test_linear_of_no_rows():
    w, = tensors(16, 24, count=1)
    x = torch.zeros(2, 0, 24, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = training.linear(x, w)
    assert y.shape == (2, 0, 16)
    y.sum().backward()
    assert x.grad.shape == x.shape and torch.equal(w.grad, torch.zeros_like(w))


@pytest.mark.parametrize("given", [(True, False), (False, True)])
def test_documents_of_one_side_are_refused(given):
    """Not taken for no documents, nor for those of the other side."""
    q, k, v = tensors(1, 2, 20, 16)
    documents = tuple(ints(*[0] * 20) if side else None for side in given)
    for call in (lambda: training.masked_attention(q, k, v, documents=documents),
                 lambda: native.masked_attention(q.detach(), k.detach(), v.detach(),
                                                 documents=documents)):
        with pytest.raises(ValueError, match="documents"):
            call()
    assert torch.equal(training.masked_attention(q, k, v, documents=(None, None)),
                       training.masked_attention(q, k, v))
