"""The linear layer on invariant channels with what follows it: bias, activation and residual in the epilogue of the matrix product.
SO3weights' matrices are the equivariant form of its matrix; there is no counterpart in the reference, whose users take it from torch."""
import torch

from gelib_amd.gelib_common import backend
from gelib_amd.group_norm_act import graph_grads


def _differentiable(x, w, b, act):
    F = torch.nn.functional
    z = torch.matmul(x.float(), w.float())
    z = z if b is None else z + b.float()
    return {"none": lambda t: t, "relu": F.relu, "silu": F.silu, "gelu": F.gelu}[act](z).to(x.dtype)


class LinearActFn(torch.autograd.Function):
    """Keeps act'(x w + b) for the backward pass: the product is not formed again, and nothing else of its size is kept."""

    @staticmethod
    def forward(ctx, x, w, b, r, act):
        y, slope = backend().linear_act_fwd(x, w, b, r, act, True)
        ctx.save_for_backward(x, w, b, slope)
        ctx.act = act
        return y

    @staticmethod
    def backward(ctx, g):
        x, w, b, slope = ctx.saved_tensors
        need = ctx.needs_input_grad
        if torch.is_grad_enabled():   # a graph of the gradients is wanted
            grads = graph_grads(lambda x, w, b: _differentiable(x, w, b, ctx.act), (x, w, b), g) if any(need[:3]) else (None,) * 3
        else:
            grads = backend().linear_act_bwd(g, slope, x, w, need[0], need[1], need[2]) if any(need[:3]) else (None,) * 3
        return (*grads, g if need[3] else None, None)


def linear_act(x, w, bias=None, residual=None, act="none"):
    """act(x w + bias) + residual for x (..., n_in) and w (n_in, n_out), float32, bfloat16 or float16 tensors of one type on the GPU.

    act: "none", "relu", "silu" or "gelu" (with the error function); bias (n_out), residual (..., n_out).  The product is summed in
    float32 and the result rounded once.  Differentiable in all four tensors; in 16-bit layers the gradient that enters the two
    products of the backward pass is rounded to the layer's type."""
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        return LinearActFn.apply(x, w, bias, residual, act)
    return backend().linear_act_fwd(x, w, bias, residual, act, False)[0]
