"""Layer norm of activations on gfx950, forward, backward and undone (C ABI, include/saeflow_hip.h).

The reference has no counterpart: its dictionaries read activations as they come. Per row of D elements:

    mean = sum x / D,  rstd = 1 / sqrt(sum (x - mean)^2 / D + eps),  xh = (x - mean) rstd,  y = xh weight + bias

The mean is summed in 64 bits, all else in 32; results are rounded once to their type. What the backward pass needs of
x is x itself or, from layer_norm_held, x - mean as 8-bit rows (kernels.Fp8Rows), a little over a byte an element.

A call on few rows is bound by the host (a launch takes 3 us, a tensor made 1 to 1.4), so the wrappers make few objects.
"""

from types import SimpleNamespace

import torch

from .. import _lib
from .encode import _vector
from .fp8 import Fp8Rows

_DTYPE = _lib.DTYPE


def _matrix(t, name):
    """t [M, D] with unit column stride (a copy only where it has another), M, D and the row stride."""
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions, got {list(t.shape)}")
    M, D = t.shape
    if D < 1:
        raise ValueError(f"{name} has rows of no elements")
    row, col = t.stride()
    if col != 1 and D > 1:
        t = t.contiguous()
        row = D
    return t, M, D, row


def _param(t, n, name):
    """(tensor or None, address, dtype code) of a parameter vector."""
    if t is None:
        return None, None, 0
    t = _vector(t, n, name)
    code = _DTYPE.get(t.dtype)
    return t, t.data_ptr(), _lib.dtype_code(t, name) if code is None else code


def _code(t, name):
    code = _DTYPE.get(t.dtype)
    return _lib.dtype_code(t, name) if code is None else code


def _row_stat(t, M, name):
    if t is None:
        raise ValueError(f"{name} is needed")
    if t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != M:
        raise ValueError(f"{name} must be a float32 tensor of shape [{M}], got {t.dtype} {list(t.shape)}")
    return t.contiguous()


def _gpu(first, *named):
    """first's device number, which the other tensors (or None) have to share; require_gpu's errors."""
    at = first.get_device()
    if at >= 0:
        for _, t in named:
            if t is not None and t.get_device() != at:
                break
        else:
            return at
    _lib.require_gpu(("rows", first), *named)
    raise ValueError("the tensors are on different devices")


def _result(like, M, D, dtype):
    """Room for [M, D], contiguous."""
    return torch.empty_like(like) if like.dtype == dtype and like.is_contiguous() else like.new_empty((M, D), dtype=dtype)


def _run(fn, at, *args):
    """The C call on torch's current stream, with GPU `at` current."""
    stream = torch._C._cuda_getCurrentRawStream(at)
    if torch._C._cuda_getDevice() == at:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(at):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc)


def _forward(x, weight, bias, eps, out_dtype, stats, hold):
    x, M, D, row = _matrix(x, "x")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    w, w_ptr, w_code = _param(weight, D, "weight")
    b, b_ptr, b_code = _param(bias, D, "bias")
    at = _gpu(x, ("weight", w), ("bias", b))
    x_code = _code(x, "x")
    y = _result(x, M, D, out_dtype or x.dtype)
    y_code = _code(y, "out_dtype")
    both, mean, rstd = None, None, None
    if stats:
        both = x.new_empty((2, M), dtype=torch.float32)
        mean = both.data_ptr()
        rstd = mean + 4 * M
    held, q = None, (None, 0, None, 0)
    if hold:
        held = Fp8Rows.empty(M, D, x.device, normed=False)
        q = held._args()
    if M:
        _run(_lib.load().sf_layer_norm, at, x.data_ptr(), row, x_code, w_ptr, w_code, b_ptr, b_code, eps, M, D,
             y.data_ptr(), D, y_code, mean, rstd, *q)
    return y, held, both


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, out_dtype=None):
    """(y, mean, rstd) of the rows of x [M, D] in fp32, bf16 or fp16: y in out_dtype (x's own by default), mean and
    rstd float32 [M]. weight and bias [D], either None, in any of the three types."""
    y, _, stats = _forward(x, weight, bias, eps, out_dtype, True, False)
    return y, *stats.unbind()


def layer_norm_held(x, weight=None, bias=None, eps=1e-5, *, out_dtype=None):
    """(y, held, mean, rstd): layer_norm that also leaves x - mean in 8 bits (Fp8Rows), written in the same pass,
    which layer_norm_backward takes in place of x."""
    y, held, stats = _forward(x, weight, bias, eps, out_dtype, True, True)
    return y, held, *stats.unbind()


def layer_norm_backward(grad_y, x, mean, rstd, weight=None, bias=None, *, need_grad_x=True, need_grad_weight=True,
                        grad_mean=None, grad_rstd=None, out_dtype=None):
    """Gradients of a loss through layer_norm, from grad_y = dL/dy [M, D]: a namespace of x [M, D], weight and bias
    (each in its parameter's type, None for one that is not given), x None without need_grad_x, weight without
    need_grad_weight.

    x: what layer_norm was given, or the Fp8Rows of layer_norm_held (then mean is not read and may be None).
    grad_mean, grad_rstd: float32 [M], gradients of the mean and rstd that the forward pass returned, if they were
      used. out_dtype: of the gradient of x; x's own by default, grad_y's for Fp8Rows.
    fp32 sums in a fixed order: repeated calls give identical bits. Nothing waits for the GPU.
    """
    g, M, D, g_row = _matrix(grad_y, "grad_y")
    held = isinstance(x, Fp8Rows)
    if tuple(x.shape) != (M, D):
        raise ValueError(f"grad_y has shape {[M, D]}, x {list(x.shape)}")
    if held:
        mean = mean_ptr = None
        x_args, first = (None, 0, 0, *x._args()), x.q
    else:
        x, _, _, x_row = _matrix(x, "x")
        mean = _row_stat(mean, M, "mean")
        mean_ptr = mean.data_ptr()
        x_args, first = (x.data_ptr(), x_row, _code(x, "x"), None, 0, None, 0), x
    rstd = _row_stat(rstd, M, "rstd")
    gm = gr = gm_ptr = gr_ptr = None
    if grad_mean is not None:
        gm = _row_stat(grad_mean, M, "grad_mean")
        gm_ptr = gm.data_ptr()
    if grad_rstd is not None:
        gr = _row_stat(grad_rstd, M, "grad_rstd")
        gr_ptr = gr.data_ptr()
    w, w_ptr, w_code = _param(weight, D, "weight")
    b, _, b_code = _param(bias, D, "bias")
    at = _gpu(g, ("x", first), ("mean", mean), ("rstd", rstd), ("weight", w), ("bias", b), ("grad_mean", gm),
              ("grad_rstd", gr))
    g_code = _code(g, "grad_y")
    dx = dx_ptr = dw = dw_ptr = db = db_ptr = ws = ws_ptr = None
    dx_code = nbytes = 0
    if need_grad_x:
        dx = _result(g if held else x, M, D, out_dtype or (g if held else x).dtype)
        dx_ptr, dx_code = dx.data_ptr(), _code(dx, "out_dtype")
    if w is not None and need_grad_weight:
        dw = torch.empty_like(w)
        dw_ptr = dw.data_ptr()
    if b is not None:
        db = torch.empty_like(b)
        db_ptr = db.data_ptr()
    if dw is not None or db is not None:
        nbytes = _lib.layer_norm_workspace_bytes(M, D)
        if nbytes:
            ws = rstd.new_empty(nbytes // 4)
            ws_ptr = ws.data_ptr()
    _run(_lib.load().sf_layer_norm_backward, at, g.data_ptr(), g_row, g_code, *x_args, mean_ptr, rstd.data_ptr(),
         w_ptr, w_code, gm_ptr, gr_ptr, M, D, dx_ptr, D, dx_code, dw_ptr, w_code, db_ptr, b_code, ws_ptr, nbytes)
    return SimpleNamespace(x=dx, weight=dw, bias=db)


def denormalize(h, mean, rstd, *, out_dtype=None):
    """h / rstd + mean per row of h [M, D]: layer_norm (without weight and bias) undone, which carries a reconstruction
    of normed rows back to the rows' own space. In fp32, rounded once to out_dtype (h's own by default)."""
    h, M, D, row = _matrix(h, "h")
    mean, rstd = _row_stat(mean, M, "mean"), _row_stat(rstd, M, "rstd")
    at = _gpu(h, ("mean", mean), ("rstd", rstd))
    h_code = _code(h, "h")
    out = _result(h, M, D, out_dtype or h.dtype)
    _run(_lib.load().sf_denormalize, at, h.data_ptr(), row, h_code, mean.data_ptr(), rstd.data_ptr(), M, D,
         out.data_ptr(), D, _code(out, "out_dtype"))
    return out


def denormalize_backward(grad, h, rstd, *, need_grad_stats=True, out_dtype=None):
    """(dh, dmean, drstd) of denormalize from grad [M, D]: dh in out_dtype (h's own by default), the other two float32
    [M], or None without need_grad_stats (then h is not read and may be None, dh in grad's type by default)."""
    g, M, D, g_row = _matrix(grad, "grad")
    if h is None and need_grad_stats:
        raise ValueError("the gradients of mean and rstd need h")
    h_args = (None, 0, 0)
    if h is not None:
        if tuple(h.shape) != (M, D):
            raise ValueError(f"grad has shape {[M, D]}, h {list(h.shape)}")
        h, _, _, h_row = _matrix(h, "h")
        h_args = (h.data_ptr(), h_row, _code(h, "h"))
    rstd = _row_stat(rstd, M, "rstd")
    at = _gpu(g, ("h", h), ("rstd", rstd))
    g_code = _code(g, "grad")
    dh = _result(g, M, D, out_dtype or (g if h is None else h).dtype)
    stats = dmean = drstd = None
    if need_grad_stats:
        stats = g.new_empty((2, M), dtype=torch.float32)
        dmean = stats.data_ptr()
        drstd = dmean + 4 * M
    _run(_lib.load().sf_denormalize_backward, at, g.data_ptr(), g_row, g_code, *h_args, rstd.data_ptr(), M, D,
         dh.data_ptr(), D, _code(dh, "out_dtype"), dmean, drstd)
    return (dh, None, None) if stats is None else (dh, *stats.unbind())
