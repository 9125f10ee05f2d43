"""Group norm with an activation on channels-last tensors: the normalisation between layers on invariant channels.  No counterpart
in the reference, whose users take it from torch with the channels moved to the front and back."""
import torch

from gelib_amd.gelib_common import backend


def _differentiable(x, groups, w, b, eps, act, lengths):
    """The same from torch's own operations, for gradients of gradients."""
    F = torch.nn.functional
    n, c = x.shape[0], x.shape[-1]
    t = x.reshape(n, -1, groups, c // groups)
    live = torch.ones((), dtype=torch.bool, device=x.device)
    count = t.shape[1] * t.shape[3]
    if lengths is not None:
        held = lengths.clamp(0, t.shape[1])
        live = (torch.arange(t.shape[1], device=x.device) < held[:, None])[:, :, None, None]
        count = (held.clamp(min=1) * t.shape[3])[:, None, None, None]
    t = torch.where(live, t.float(), 0.)
    d = torch.where(live, t - t.sum((1, 3), keepdim=True) / count, 0.)
    t = (d * torch.rsqrt((d * d).sum((1, 3), keepdim=True) / count + eps)).reshape(x.shape)
    t = t if w is None else t * w.float()
    t = t if b is None else t + b.float()
    t = {"none": lambda z: z, "relu": F.relu, "silu": F.silu, "gelu": F.gelu}[act](t)
    return torch.where(live, t.reshape(n, -1, groups, c // groups), 0.).reshape(x.shape).to(x.dtype)


def graph_grads(fn, tensors, g):
    """Gradients of fn(*tensors) with a graph of their own; None where a tensor is None or needs none."""
    with torch.enable_grad():
        views = [t if t is None else t.view_as(t) for t in tensors]   # (one tensor may stand in two places)
        wanted = [v for v, t in zip(views, tensors) if t is not None and t.requires_grad]
        got = iter(torch.autograd.grad(fn(*views), wanted, g, create_graph=True))
        return [next(got) if t is not None and t.requires_grad else None for t in tensors]


class GroupNormActFn(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, w, b, groups, eps, act, lengths):
        y, mean, rstd = backend().group_norm_act_fwd(x, groups, w, b, eps, act, lengths, True)
        ctx.save_for_backward(x, w, b, lengths, mean, rstd)
        ctx.how = groups, eps, act
        return y

    @staticmethod
    def backward(ctx, g):
        x, w, b, lengths, mean, rstd = ctx.saved_tensors
        groups, eps, act = ctx.how
        if torch.is_grad_enabled():   # a graph of the gradients is wanted
            grads = graph_grads(lambda x, w, b: _differentiable(x, groups, w, b, eps, act, lengths), (x, w, b), g)
        else:
            need = ctx.needs_input_grad
            grads = backend().group_norm_act_bwd(g, mean, rstd, x, groups, w, b, act, lengths, need[0], need[1], need[2])
        return (*grads, None, None, None, None)


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act="none", lengths=None):
    """act(group_norm(x) * weight + bias) of a tensor (batch, [positions...], channels) of float32, bfloat16 or float16 values on the GPU,
    in one or two passes over it.

    A group is channels / groups neighbouring channels over all positions of a sample; with lengths (int32, one a sample: atoms of a
    padded molecule, cells of a smaller grid) over its first lengths[n] positions, counted through all dimensions between the first
    and the last: the others are not read, and are zero in the result and in the gradient of x.  act: "none", "relu", "silu" or
    "gelu" (with the error function).  weight and bias: one value a channel, of x's type.  Statistics are formed in float32 around
    the mean; results are rounded to x's type once.  Differentiable in x, weight and bias."""
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        return GroupNormActFn.apply(x, weight, bias, groups, eps, act, lengths)
    return backend().group_norm_act_fwd(x, groups, weight, bias, eps, act, lengths, False)[0]
