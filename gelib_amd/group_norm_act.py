"""Group norm with an activation on channels-last tensors: the normalisation between layers on invariant channels.  No counterpart
in the reference, whose users take it from torch with the channels moved to the front and back."""
from gelib_amd.gelib_common import backend


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act="none", lengths=None):
    """act(group_norm(x) * weight + bias) of a tensor (batch, [positions...], channels) of float32, bfloat16 or float16 values on the GPU,
    in one or two passes over it.

    A group is channels / groups neighbouring channels over all positions of a sample; with lengths (int32, one a sample: atoms of a
    padded molecule, cells of a smaller grid) over its first lengths[n] positions, counted through all dimensions between the first
    and the last: the others are not read, and are zero in the result and in the gradient of x.  act: "none", "relu", "silu" or
    "gelu" (with the error function).  weight and bias: one value a channel, of x's type.  Statistics are formed in float32 around
    the mean; results are rounded to x's type once.  Differentiable in x, weight and bias, twice by torch's own operations, which
    forward-mode derivatives, function transforms, tracing and dispatch modes get from the start."""
    return backend().group_norm_act(x, groups, weight, bias, eps, act, lengths)
