"""The operators bound as an autograd rule: a linear layer that keeps its input
in 8 bits, with its gradients, and an error for a second derivative, of which
the operators know nothing."""

import pytest
import torch
from torch.autograd.function import once_differentiable

pytestmark = pytest.mark.gpu


class Linear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w):
        import rollfast_b200 as rf

        ctx.saved_x = rf.save_activation(x)
        ctx.save_for_backward(w)
        return x @ w

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        import rollfast_b200 as rf

        w, = ctx.saved_tensors
        dw = rf.weight_gradient(ctx.saved_x, dy, layout="io")
        return dy @ w.t(), dw.to(w.dtype)


def _leaves():
    g = torch.Generator("cuda").manual_seed(1)
    # Whole numbers up to 127 with a 127 in each block: the 8-bit copy is x.
    x = torch.randint(-126, 127, (3, 50, 96), generator=g, device="cuda").float()
    x[..., ::32] = 127.0
    w = torch.randint(-4, 5, (96, 40), generator=g, device="cuda").float()
    return x.requires_grad_(), w.requires_grad_()


def test_gradients_of_a_linear_layer():
    x, w = _leaves()
    y = Linear8.apply(x, w)
    y.sum().backward()  # the incoming gradient is a broadcast one
    assert torch.equal(x.grad, w.sum(1).expand_as(x))
    assert torch.equal(w.grad, x.sum((0, 1))[:, None].expand_as(w))
    # A difference: the loss is linear in w.
    step = torch.zeros_like(w)
    step[5, 7] = 1.0
    with torch.no_grad():
        diff = Linear8.apply(x, w + step).double().sum() - Linear8.apply(x, w).double().sum()
    assert diff == w.grad[5, 7]


def test_a_second_derivative_is_an_error():
    x, w = _leaves()
    weights = torch.ones(3, 50, 40, device="cuda", requires_grad=True)
    # Without the mark, x's gradient keeps its history and w's loses it: the sum's derivative would lack a part.
    dx, dw = torch.autograd.grad((Linear8.apply(x, w) * weights).sum(), (x, w), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum() + dw.sum(), weights, retain_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (dx.sum() + dw.sum()).backward()
