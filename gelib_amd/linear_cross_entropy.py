"""The loss of a linear layer's classes: elements of masked atoms, rotations of a grid.  linear_act's matrix product with the softmax's sums in
its epilogue; no counterpart in the reference, whose users take it from torch."""
from gelib_amd.gelib_common import backend


def linear_cross_entropy(x, w, targets, bias=None):
    """log(sum_c exp(z_c)) - z_target of z = x w + bias for every row of x: float32 losses (...) from x (..., n_in), w (n_in, n_out),
    bias (n_out), float32, bfloat16 or float16 tensors of one type on the GPU, and int64 targets (...).

    A target below zero leaves its row out: its loss and its gradients are zero, whatever the row and w hold.  One that is n_out or more makes its loss and the gradients
    that it enters NaN: targets are read on the GPU only.  Logits are formed tile by tile, in float32, and not kept; the backward pass forms them
    again, for some classes after the other.  In 16-bit types the gradient of the logits is rounded to the type for the two products of the
    backward pass.  Differentiable in x, w and bias, twice by torch's own operations, which forward-mode derivatives, function
    transforms, tracing and dispatch modes get from the start."""
    return backend().linear_cross_entropy(x, w, targets, bias)
