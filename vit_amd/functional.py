"""Operators beside the model's own layers, as functions of tensors with gradients.

Each checks its arguments, launches the HIP kernels of libvitk on the current stream of its inputs' device, and raises
VitkError for what they do not take; there is no CPU path.  Gradients are those of reverse mode: an input with a forward-mode
tangent is refused.
"""
import torch
from torch.autograd import forward_ad

from . import ops
from .autograd import DiffAttentionFn, GroupNormFn
from .lib import VitkError


def _on_device(x):
    """The context in which x's device is the current one."""
    if not x.is_cuda:
        raise VitkError("expected CUDA/HIP tensors: these operators have no CPU fallback")
    return ops._NULL if x.get_device() == torch.cuda.current_device() else torch.cuda.device(x.device)


def _needs_grad(*tensors):
    if getattr(forward_ad, "_current_level", 0) >= 0:          # inside a dual level: tangents would be dropped
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise VitkError("these operators have no forward-mode derivative")
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def group_norm(x, num_groups, weight=None, bias=None, eps=1e-5, activation="none"):
    """act(GroupNorm(x)) for channels-last x [batch, ..., channels] (bf16 or f32, contiguous): tokens [B, N, C] as they
    are, a feature map in torch's channels_last format as `x.permute(0, 2, 3, 1)`, which is a view.

    Statistics over all positions of channels / num_groups neighbouring channels per sample, in f32; weight and bias f32
    [channels] or None; activation "none", "relu", "gelu" (nn.GELU()'s z Phi(z): Phi to f32's rounding in
    f32, from an erf good to 1.5e-7 in bf16) or "silu".  Returns x's shape and type.
    Differentiable once in x, weight and bias."""
    with _on_device(x):
        if _needs_grad(x, weight, bias):
            return GroupNormFn.apply(x, weight, bias, num_groups, eps, activation)
        return ops.group_norm(x, num_groups, weight, bias, eps, activation)[0]


def diff_attention(q, k, v, lam, lambda_init=0.8, scale=None, key_lens=None, causal=False):
    """Differential attention: per head h the difference of two softmax maps with a learned weight,

        out[:, :, h] = (softmax(scale q_1 k_1^T) - w_h softmax(scale q_2 k_2^T)) v
        w_h = exp(lam[0] . lam[1]) - exp(lam[2] . lam[3]) + lambda_init

    q [B, Nq, H, 2, d], k [B, Nk, K, 2, d], v [B, Nk, K, 2d] (bf16 or f32; d a multiple of 8 up to 64; H a multiple of K,
    query heads h * H / K ... share key head h), out [B, Nq, H, 2d].  Any strides in multiples of 16 bytes with a dense last
    dimension: the fused projection's qkv [3, B, H, N, 2d] goes in as `qkv[i].view(B, H, N, 2, d).permute(0, 2, 1, 3, 4)`.
    q, k and v start at multiples of 16 bytes too.  lam f32 [4, H, d], or [4, d] for all heads, contiguous; scale defaults to d ** -0.5 and must be positive.
    key_lens (int32 [B] on the device) hides the keys from key_lens[b] on: they are never read and get no gradient.  causal:
    query t sees keys up to t + Nk - Nq (the last query all of them); keys and values that only some queries see have to be
    finite, since a probability of 0 still multiplies them.  A row without a visible key gives 0 and no gradient.
    Single query tokens against a long cache take a form that splits the keys.  Differentiable once in q, k, v and lam.

    Scores, softmax statistics and sums are f32; in bf16 the probabilities are rounded to bf16 for the product with v.  Without
    gradients the denominators add those rounded values, with gradients the f32 ones, so the two may differ by the output's
    rounding.  A scaled score's own f32 rounding, 2^-24 of it, enters the exponent: probabilities lose accuracy from some
    thousands on, gradients have none left from 2^22 on, and scores of 2^30 and more may give NaN."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if lam.data_ptr() % 16:                      # a view into something larger: the kernels load 16 bytes at a time
        lam = lam.clone()
    with _on_device(q):
        if _needs_grad(q, k, v, lam):
            return DiffAttentionFn.apply(q, k, v, lam, lambda_init, scale, key_lens, causal)
        return ops.diff_attention(q, k, v, lam, lambda_init, scale, key_lens, causal)[0]
