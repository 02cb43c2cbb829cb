"""Training through the sparse path: the forward of saeflow_amd.forward (encode_sparse then
decode_sparse, ops.py:29-49 in the reference) as a torch.autograd.Function whose backward runs
the gfx950 backward kernels (kernels/backward.py). The reference has these on its roadmap
(saeflow README.md:244); the dense [tokens, d_sae] features exist in neither direction.

    x_hat, (indptr, indices, values) = forward_train(sae, x)
    loss = (x_hat - x).pow(2).sum(-1).mean() + lam * values.float().abs().sum() / len(x)
    loss.backward()      # fills sae.W_enc.grad, b_enc.grad, W_dec.grad, b_dec.grad (and x.grad)

values is differentiable too, so a sparsity penalty on the feature activations (optionally
weighted by W_dec row norms gathered with `indices`) flows back through the encoder.
"""

from types import SimpleNamespace

import torch

from . import norm, ops
from .kernels import Fp8Rows, quantize_rows
from .kernels.backward import sparse_backward


class SparseSAEFunction(torch.autograd.Function):
    """(x, W_enc, b_enc, W_dec, b_dec, threshold, activation, k, held) -> (x_hat, indptr, indices, values).

    indptr and indices are not differentiable. The threshold gets no gradient (jumprelu's is
    zero almost everywhere; training it needs a pseudo-derivative, which is a modelling choice
    outside the path)."""

    @staticmethod
    def forward(ctx, x, W_enc, b_enc, W_dec, b_dec, threshold, activation, k, held=False):
        sae = SimpleNamespace(W_enc=W_enc, b_enc=b_enc, W_dec=W_dec, b_dec=b_dec, threshold=threshold,
                              activation=activation, k=k)
        indptr, indices, values = ops.encode_sparse(sae, x)  # (no input norm: forward_train has applied it)
        x_hat = ops.decode_sparse(sae, (indptr, indices, values))
        ctx.held, ctx.x_dtype = held, x.dtype
        kept = (x, None)
        if held:  # what the backward pass needs of x is x - b_dec, for dW_enc
            rows8 = quantize_rows(x, shift=b_dec)
            kept = (rows8.q, rows8.scale)
        ctx.save_for_backward(*kept, W_enc, b_enc, W_dec, b_dec, indptr, indices, values)
        ctx.mark_non_differentiable(indptr, indices)
        # absent gradients arrive as None, not as zeros filled for indptr, indices and an unused output
        ctx.set_materialize_grads(False)
        return x_hat, indptr, indices, values

    @staticmethod
    def backward(ctx, g_xhat, _g_indptr, _g_indices, g_values):
        x, scale, W_enc, b_enc, W_dec, b_dec, indptr, indices, values = ctx.saved_tensors
        need = ctx.needs_input_grad
        if not any(need[:5]):
            return (None,) * 9
        if ctx.held:
            x = Fp8Rows(x, scale, W_enc.shape[0])
        gr = sparse_backward(x, W_enc, b_enc, W_dec, b_dec, (indptr, indices, values), g_xhat, g_values,
                             need_grad_x=need[0])
        return (gr.x.to(ctx.x_dtype) if need[0] else None, gr.W_enc if need[1] else None,
                gr.b_enc if need[2] else None, gr.W_dec if need[3] else None, gr.b_dec if need[4] else None,
                None, None, None, None)


def forward_train(sae, x, *, hold=None):
    """x_hat and the CSR features (indptr, indices, values) of `sae` on x, differentiable with
    respect to x, W_enc, b_enc, W_dec and b_dec (and through `values`).

    hold: None, or torch.float8_e4m3fn: what the backward pass needs of the activations is kept in 8 bits (x - b_dec,
      and x - mean of an input norm, each element off by at most 2^-4 of itself or 2^-10 of its block's scale) in
      place of x. dW_enc sums those, and the gradient of x goes through an input norm by them; the features, x_hat and
      the other gradients are not touched."""
    held = norm.check_hold(hold)
    normed = ops.input_norm(sae) is not None
    if normed:
        x, mean, rstd = norm.layer_norm(x, eps=ops.norm_eps(sae), hold=hold, return_stats=True)
    x_hat, indptr, indices, values = SparseSAEFunction.apply(x, sae.W_enc, sae.b_enc, sae.W_dec, sae.b_dec,
                                                             sae.threshold, sae.activation, sae.k, held)
    if normed:
        x_hat = norm.denormalize(x_hat, mean, rstd)
    return x_hat, (indptr, indices, values)
