"""The linear layer on invariant channels with what follows it: bias, activation and residual in the epilogue of the matrix product.
SO3weights' matrices are the equivariant form of its matrix; there is no counterpart in the reference, whose users take it from torch."""
from gelib_amd.gelib_common import backend


def linear_act(x, w, bias=None, residual=None, act="none"):
    """act(x w + bias) + residual for x (..., n_in) and w (n_in, n_out), float32, bfloat16 or float16 tensors of one type on the GPU.

    act: "none", "relu", "silu" or "gelu" (with the error function); bias (n_out), residual (..., n_out).  The product is summed in
    float32 and the result rounded once.  Differentiable in all four tensors, twice by torch's own operations; the forward pass keeps
    act'(x w + bias) for it, and in 16-bit layers the gradient that enters the two products of the backward pass is rounded to the
    layer's type.  Forward-mode derivatives, function transforms, tracing and dispatch modes get torch's own operations."""
    return backend().linear_act(x, w, bias, residual, act)
