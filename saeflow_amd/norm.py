"""Layer norm of activations around a dictionary, differentiable (kernels/norm.py; no reference counterpart).

    z = layer_norm(x, weight, bias)                           # what a transcoder reads, trained through
    z = layer_norm(x, weight, bias, hold=torch.float8_e4m3fn) # 8 bits of x - mean kept for the backward pass, not x

    z, mean, rstd = layer_norm(x, return_stats=True)
    x_hat = denormalize(forward(sae, z), mean, rstd)          # the reconstruction in the tokens' own space

An SAE with input_norm="layer_norm" (sae.py) does the last two lines by itself.
"""

import torch
from torch.autograd.function import once_differentiable

from .kernels import norm as _k
from .kernels.fp8 import Fp8Rows

HOLD = (None, torch.float8_e4m3fn)


def check_hold(hold):
    if hold not in HOLD:
        raise ValueError(f"hold must be one of {list(HOLD)}, got {hold!r}")
    return hold is not None


class LayerNormFunction(torch.autograd.Function):
    """(x [M, D], weight, bias, eps, held) -> (y, mean, rstd)."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, held):
        y, rows8, stats = _k._forward(x, weight, bias, eps, None, True, held)
        mean, rstd = stats[0], stats[1]
        ctx.held, ctx.x_dtype, ctx.d = held, x.dtype, x.shape[1]
        kept = (rows8.q, rows8.scale) if held else (x, None)
        ctx.save_for_backward(*kept, mean, rstd, weight, bias)
        ctx.set_materialize_grads(False)
        return y, mean, rstd

    @staticmethod
    @once_differentiable
    def backward(ctx, g_y, g_mean, g_rstd):
        x, scale, mean, rstd, weight, bias = ctx.saved_tensors
        need = ctx.needs_input_grad
        if g_y is None and g_mean is None and g_rstd is None:
            return (None,) * 5
        if ctx.held:
            x = Fp8Rows(x, scale, ctx.d)
        if g_y is None:
            g_y = torch.zeros((rstd.shape[0], ctx.d), dtype=ctx.x_dtype, device=rstd.device)
        gr = _k.layer_norm_backward(g_y, x, mean, rstd, weight, bias if need[2] else None, need_grad_x=need[0],
                                    need_grad_weight=need[1], grad_mean=g_mean, grad_rstd=g_rstd, out_dtype=ctx.x_dtype)
        return gr.x, gr.weight, gr.bias, None, None


class DenormalizeFunction(torch.autograd.Function):
    """(h [M, D], mean, rstd) -> h / rstd + mean."""

    @staticmethod
    def forward(ctx, h, mean, rstd):
        stats = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        ctx.save_for_backward(h if stats else None, rstd)
        ctx.h_dtype = h.dtype
        return _k.denormalize(h, mean, rstd)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        h, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        dh, dmean, drstd = _k.denormalize_backward(g, h, rstd, need_grad_stats=need[1] or need[2], out_dtype=ctx.h_dtype)
        return dh if need[0] else None, dmean if need[1] else None, drstd if need[2] else None


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, hold=None, return_stats=False):
    """Layer norm over the last dimension of x [..., D], in x's type; with return_stats (y, mean, rstd), the last two
    float32 [...]. Differentiable with respect to x, weight and bias (and through mean and rstd).

    hold: None, or torch.float8_e4m3fn: the backward pass keeps x - mean in 8 bits (a power-of-two scale for each
      block of 128) in place of x: for the gradients each element is off by at most 2^-4 of itself, or 2^-10 of its
      block's scale; y is not touched.
    """
    held = check_hold(hold)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x needs a dimension to be normed over, got {list(x.shape)}")
    lead = x.shape[:-1]
    rows = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        y, mean, rstd = LayerNormFunction.apply(rows, weight, bias, eps, held)
    else:
        y, _, stats = _k._forward(rows, weight, bias, eps, None, return_stats, False)
        mean, rstd = (None, None) if stats is None else (stats[0], stats[1])
    if x.dim() != 2:
        y = y.view(x.shape)
        if return_stats:
            mean, rstd = mean.view(lead), rstd.view(lead)
    return (y, mean, rstd) if return_stats else y


def denormalize(h, mean, rstd):
    """h / rstd + mean over the rows of h [..., D], mean and rstd float32 [...] as layer_norm returned them, in h's type.
    Differentiable with respect to all three."""
    if h.dim() < 1 or h.shape[-1] < 1 or mean.shape != h.shape[:-1] or rstd.shape != h.shape[:-1]:
        raise ValueError(f"h {list(h.shape)} needs mean and rstd of its rows, got {list(mean.shape)} and {list(rstd.shape)}")
    rows, m, r = (h, mean, rstd) if h.dim() == 2 else (h.reshape(-1, h.shape[-1]), mean.reshape(-1), rstd.reshape(-1))
    if torch.is_grad_enabled() and (h.requires_grad or mean.requires_grad or rstd.requires_grad):
        out = DenormalizeFunction.apply(rows, m, r)
    else:
        out = _k.denormalize(rows, m, r)
    return out if h.dim() == 2 else out.view(h.shape)
