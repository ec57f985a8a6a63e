"""What needs no GPU of the sequence operators' unusual cases."""
import pytest
import torch


def test_waits_are_made_to_run_out_only_on_request():
    from dwconv_b200 import _lib
    expire = _lib.lib.dwconv_b200_debug_expire
    assert expire(1) == 0 and expire(2) == 1 and expire(5) == 2 and expire(0) == 0


def test_first_order_gradients_refuse_to_be_constants():
    """y = x^2 w by a function whose backward is first-order: the gradient of a penalty on dx would lose 2 x w."""
    from dwconv_b200.sequence import _first_order

    class Square(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            ctx.save_for_backward(x, w)
            return x * x * w

        @staticmethod
        @_first_order
        def backward(ctx, grad):
            x, w = ctx.saved_tensors
            return 2 * x * w * grad, None

    x, w = torch.tensor([3.0], requires_grad=True), torch.tensor([2.0])
    dx, = torch.autograd.grad(Square.apply(x, w).sum(), x)
    assert dx.item() == 12 and not dx.requires_grad
    dx, = torch.autograd.grad(Square.apply(x, w).sum(), x, create_graph=True)
    assert dx.item() == 12
    with pytest.raises(RuntimeError, match="once_differentiable"):
        ((dx * dx).sum() + (x * x).sum()).backward()
