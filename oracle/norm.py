"""Layer norm and its gradients in 64-bit arithmetic on the CPU (no reference counterpart).

    mean = sum x / D,  rstd = 1 / sqrt(sum (x - mean)^2 / D + eps),  xh = (x - mean) rstd,  y = xh w + b

backward takes the centred rows d (x - mean, or the values that 8-bit rows hold for it) and rstd, and gives, next to
the gradients, the sums of magnitudes that an error bound of them is made of. Pinned in tests/test_norm.py by float64
autograd and by finite differences.
"""

from types import SimpleNamespace

import torch


def _d(t):
    return None if t is None else t.detach().to("cpu", torch.float64)


def forward(x, w=None, b=None, eps=1e-5):
    """(y, mean, rstd, xh) in float64."""
    x, w, b = _d(x), _d(w), _d(b)
    mean = x.sum(1) / x.shape[1]
    d = x - mean[:, None]
    rstd = 1.0 / torch.sqrt((d * d).sum(1) / x.shape[1] + eps)
    xh = d * rstd[:, None]
    y = xh if w is None else xh * w
    return (y if b is None else y + b), mean, rstd, xh


def backward(g, d, rstd, w=None, g_mean=None, g_rstd=None):
    """x, weight, bias: the gradients; q, c1, c2 and the means of magnitudes mq = mean |q|, mqx = mean |q xh|, and
    column sums aw = sum |g xh|, ab = sum |g|."""
    g, d, rstd, w, g_mean, g_rstd = map(_d, (g, d, rstd, w, g_mean, g_rstd))
    D = g.shape[1]
    xh = d * rstd[:, None]
    q = g if w is None else g * w
    c1, c2 = q.sum(1, keepdim=True) / D, (q * xh).sum(1, keepdim=True) / D
    dx = rstd[:, None] * (q - c1 - xh * c2)
    if g_mean is not None:
        dx = dx + g_mean[:, None] / D
    if g_rstd is not None:
        dx = dx - (g_rstd * rstd * rstd)[:, None] * xh / D
    return SimpleNamespace(x=dx, weight=(g * xh).sum(0), bias=g.sum(0), xh=xh, q=q, c1=c1, c2=c2,
                           mq=q.abs().mean(1, keepdim=True), mqx=(q * xh).abs().mean(1, keepdim=True),
                           aw=(g * xh).abs().sum(0), ab=g.abs().sum(0))


def undone(h, mean, rstd):
    return _d(h) / _d(rstd)[:, None] + _d(mean)[:, None]


def undone_backward(g, h, rstd):
    """(dh, dmean, drstd)."""
    g, h, rstd = _d(g), _d(h), _d(rstd)
    return g / rstd[:, None], g.sum(1), -(g * h).sum(1) / rstd ** 2
