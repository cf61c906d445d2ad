"""What the operators' backward passes share."""

import torch


class _FirstOrder(torch.autograd.Function):
    @staticmethod
    def forward(ctx, what, output, *grads):
        ctx.what = what
        return tuple(None if g is None else g.detach() for g in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.what} has no second derivative: its gradients come from kernels without a backward "
                           "pass of their own")


def first_order(what, output, *grads):
    """``grads`` as they are; where a graph of the backward pass is being made (``create_graph``),
    such that differentiating them raises. ``output``, a saved output of the operator, ties them to
    all of its inputs. (torch's once_differentiable leaves gradients of a cotangent that needs none, a
    plain sum's, as constants, and ties the others to no input.)"""
    if not torch.is_grad_enabled():
        return grads
    return _FirstOrder.apply(what, output, *grads)
