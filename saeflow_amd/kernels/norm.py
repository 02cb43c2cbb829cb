"""Layer norm of activations on gfx950, forward, backward and undone (C ABI, include/saeflow_hip.h).

The reference has no counterpart: its dictionaries read activations as they come. Per row of D elements:

    mean = sum x / D,  rstd = 1 / sqrt(sum (x - mean)^2 / D + eps),  xh = (x - mean) rstd,  y = xh weight + bias

The mean is summed in 64 bits, all else in 32; results are rounded once to their type. What the backward pass needs of
x is x itself or, from layer_norm_held, x - mean as 8-bit rows (kernels.Fp8Rows), a little over a byte an element.
"""

from types import SimpleNamespace

import torch

from .. import _lib
from .encode import _vector
from .fp8 import Fp8Rows


def _matrix(t, name):
    """t [M, D] with unit column stride (a copy only where it has another)."""
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions, got {list(t.shape)}")
    if t.shape[1] < 1:
        raise ValueError(f"{name} has rows of no elements")
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _param(t, n, name):
    """(tensor or None, address, dtype code) of a parameter vector."""
    if t is None:
        return None, None, 0
    t = _vector(t, n, name)
    return t, t.data_ptr(), _lib.dtype_code(t, name)


def _row_stat(t, M, name):
    if t.dtype != torch.float32 or t.dim() != 1 or t.numel() != M:
        raise ValueError(f"{name} must be a float32 tensor of shape [{M}], got {t.dtype} {list(t.shape)}")
    return t.contiguous()


def _forward(x, weight, bias, eps, out_dtype, stats, hold):
    x = _matrix(x, "x")
    M, D = x.shape
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    w, w_ptr, w_code = _param(weight, D, "weight")
    b, b_ptr, b_code = _param(bias, D, "bias")
    dev = _lib.require_gpu(("x", x), ("weight", w), ("bias", b))
    x_code = _lib.dtype_code(x, "x")
    y = torch.empty((M, D), dtype=out_dtype or x.dtype, device=dev)
    y_code = _lib.dtype_code(y, "out_dtype")
    both = torch.empty((2, M), dtype=torch.float32, device=dev) if stats else None
    held = Fp8Rows.empty(M, D, dev) if hold else None
    if M:
        at = None if both is None else both.data_ptr()
        q = held._args() if hold else (None, 0, None, 0)
        with _lib.device(dev):
            rc = _lib.load().sf_layer_norm(x.data_ptr(), x.stride(0), x_code, w_ptr, w_code, b_ptr, b_code, eps, M, D,
                                           y.data_ptr(), D, y_code, at, None if at is None else at + 4 * M, *q,
                                           _lib.stream(dev))
        if rc:
            _lib.check(rc)
    return y, held, both


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, out_dtype=None):
    """(y, mean, rstd) of the rows of x [M, D] in fp32, bf16 or fp16: y in out_dtype (x's own by default), mean and
    rstd float32 [M]. weight and bias [D], either None, in any of the three types."""
    y, _, stats = _forward(x, weight, bias, eps, out_dtype, True, False)
    return y, stats[0], stats[1]


def layer_norm_held(x, weight=None, bias=None, eps=1e-5, *, out_dtype=None):
    """(y, held, mean, rstd): layer_norm that also leaves x - mean in 8 bits (Fp8Rows), written in the same pass,
    which layer_norm_backward takes in place of x."""
    y, held, stats = _forward(x, weight, bias, eps, out_dtype, True, True)
    return y, held, stats[0], stats[1]


def layer_norm_backward(grad_y, x, mean, rstd, weight=None, bias=None, *, need_grad_x=True, grad_mean=None,
                        grad_rstd=None, out_dtype=None):
    """Gradients of a loss through layer_norm, from grad_y = dL/dy [M, D]: a namespace of x [M, D], weight and bias
    (each in its parameter's type, None for one that is not given), x None without need_grad_x.

    x: what layer_norm was given, or the Fp8Rows of layer_norm_held (then mean is not read and may be None).
    grad_mean, grad_rstd: float32 [M], gradients of the mean and rstd that the forward pass returned, if they were
      used. out_dtype: of the gradient of x; x's own by default, grad_y's for Fp8Rows.
    fp32 sums in a fixed order: repeated calls give identical bits. Nothing waits for the GPU.
    """
    g = _matrix(grad_y, "grad_y")
    M, D = g.shape
    held = isinstance(x, Fp8Rows)
    if tuple(x.shape) != (M, D):
        raise ValueError(f"grad_y has shape {[M, D]}, x {list(x.shape)}")
    if not held:
        x = _matrix(x, "x")
    rstd = _row_stat(rstd, M, "rstd")
    mean = None if held else _row_stat(mean, M, "mean")
    grad_mean = None if grad_mean is None else _row_stat(grad_mean, M, "grad_mean")
    grad_rstd = None if grad_rstd is None else _row_stat(grad_rstd, M, "grad_rstd")
    w, w_ptr, w_code = _param(weight, D, "weight")
    if bias is not None and (bias.dim() != 1 or bias.numel() != D):
        raise ValueError(f"bias must have shape [{D}], got {list(bias.shape)}")
    dev = _lib.require_gpu(("grad_y", g), ("x", x.q if held else x), ("mean", mean), ("rstd", rstd), ("weight", w),
                           ("bias", bias), ("grad_mean", grad_mean), ("grad_rstd", grad_rstd))
    g_code = _lib.dtype_code(g, "grad_y")
    x_args = (None, 0, 0, *x._args()) if held else (x.data_ptr(), x.stride(0), _lib.dtype_code(x, "x"), None, 0, None, 0)
    dx = dx_ptr = dw = dw_ptr = db = db_ptr = None
    dx_code = db_code = 0
    if need_grad_x:
        dx = torch.empty((M, D), dtype=out_dtype or (g.dtype if held else x.dtype), device=dev)
        dx_ptr, dx_code = dx.data_ptr(), _lib.dtype_code(dx, "out_dtype")
    if w is not None:
        dw = torch.empty(D, dtype=w.dtype, device=dev)
        dw_ptr = dw.data_ptr()
    if bias is not None:
        db = torch.empty(D, dtype=bias.dtype, device=dev)
        db_ptr, db_code = db.data_ptr(), _lib.dtype_code(db, "bias")
    with _lib.device(dev):
        ws = None
        if dw is not None or db is not None:
            ws = torch.empty(_lib.layer_norm_workspace_bytes(M, D), dtype=torch.uint8, device=dev)
        rc = _lib.load().sf_layer_norm_backward(
            g.data_ptr(), g.stride(0), g_code, *x_args, _lib.ptr(mean), rstd.data_ptr(), w_ptr, w_code,
            _lib.ptr(grad_mean), _lib.ptr(grad_rstd), M, D, dx_ptr, D, dx_code, dw_ptr, w_code, db_ptr, db_code,
            _lib.ptr(ws), 0 if ws is None else ws.numel(), _lib.stream(dev))
    if rc:
        _lib.check(rc)
    return SimpleNamespace(x=dx, weight=dw, bias=db)


def denormalize(h, mean, rstd, *, out_dtype=None):
    """h / rstd + mean per row of h [M, D]: layer_norm (without weight and bias) undone, which carries a reconstruction
    of normed rows back to the rows' own space. In fp32, rounded once to out_dtype (h's own by default)."""
    h = _matrix(h, "h")
    M, D = h.shape
    mean, rstd = _row_stat(mean, M, "mean"), _row_stat(rstd, M, "rstd")
    dev = _lib.require_gpu(("h", h), ("mean", mean), ("rstd", rstd))
    h_code = _lib.dtype_code(h, "h")
    out = torch.empty((M, D), dtype=out_dtype or h.dtype, device=dev)
    out_code = _lib.dtype_code(out, "out_dtype")
    with _lib.device(dev):
        rc = _lib.load().sf_denormalize(h.data_ptr(), h.stride(0), h_code, mean.data_ptr(), rstd.data_ptr(), M, D,
                                        out.data_ptr(), D, out_code, _lib.stream(dev))
    if rc:
        _lib.check(rc)
    return out


def denormalize_backward(grad, h, rstd, *, need_grad_stats=True, out_dtype=None):
    """(dh, dmean, drstd) of denormalize from grad [M, D]: dh in out_dtype (h's own by default), the other two float32
    [M], or None without need_grad_stats (then h is not read and may be None, dh in grad's type by default)."""
    g = _matrix(grad, "grad")
    M, D = g.shape
    if h is None and need_grad_stats:
        raise ValueError("the gradients of mean and rstd need h")
    h = None if h is None else _matrix(h, "h")
    if h is not None and tuple(h.shape) != (M, D):
        raise ValueError(f"grad has shape {[M, D]}, h {list(h.shape)}")
    rstd = _row_stat(rstd, M, "rstd")
    dev = _lib.require_gpu(("grad", g), ("h", h), ("rstd", rstd))
    g_code = _lib.dtype_code(g, "grad")
    h_args = (None, 0, 0) if h is None else (h.data_ptr(), h.stride(0), _lib.dtype_code(h, "h"))
    dh = torch.empty((M, D), dtype=out_dtype or (g if h is None else h).dtype, device=dev)
    dh_code = _lib.dtype_code(dh, "out_dtype")
    stats = torch.empty((2, M), dtype=torch.float32, device=dev) if need_grad_stats else None
    at = None if stats is None else stats.data_ptr()
    with _lib.device(dev):
        rc = _lib.load().sf_denormalize_backward(g.data_ptr(), g.stride(0), g_code, *h_args, rstd.data_ptr(), M, D,
                                                 dh.data_ptr(), D, dh_code, at, None if at is None else at + 4 * M, _lib.stream(dev))
    if rc:
        _lib.check(rc)
    return (dh, None, None) if stats is None else (dh, stats[0], stats[1])
