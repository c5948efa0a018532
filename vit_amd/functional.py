"""Operators beside the model's own layers, as functions of tensors with gradients.

Each checks its arguments, launches the HIP kernels of libvitk on the current stream of its inputs' device, and raises
VitkError for what they do not take; there is no CPU path.
"""
import torch

from . import ops
from .autograd import GroupNormFn
from .lib import VitkError


def _on_device(x):
    """The context in which x's device is the current one."""
    if not x.is_cuda:
        raise VitkError("expected CUDA/HIP tensors: these operators have no CPU fallback")
    return ops._NULL if x.get_device() == torch.cuda.current_device() else torch.cuda.device(x.device)


def _needs_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def group_norm(x, num_groups, weight=None, bias=None, eps=1e-5, activation="none"):
    """act(GroupNorm(x)) for channels-last x [batch, ..., channels] (bf16 or f32, contiguous): tokens [B, N, C] as they
    are, a feature map in torch's channels_last format as `x.permute(0, 2, 3, 1)`, which is a view.

    Statistics over all positions of channels / num_groups neighbouring channels per sample, in f32; weight and bias f32
    [channels] or None; activation "none", "relu", "gelu" (exact erf) or "silu".  Returns x's shape and type.
    Differentiable once in x, weight and bias."""
    with _on_device(x):
        if _needs_grad(x, weight, bias):
            return GroupNormFn.apply(x, weight, bias, num_groups, eps, activation)
        return ops.group_norm(x, num_groups, weight, bias, eps, activation)[0]
