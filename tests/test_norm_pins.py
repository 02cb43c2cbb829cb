"""CPU: what the pin of the layer norm oracle and the bounds of the GPU tests reject: small wrong coefficients, a dropped
row, a missing term, planted in the oracle's own result."""

from types import SimpleNamespace

import pytest
import torch

from oracle import norm as onorm
from test_gpu_norm import check_backward


def inputs(M=24, D=96, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, w, b = r(M, D) * 2 + 0.5, 1 + 0.3 * r(D), r(D)
    _, mean, rstd, xh = onorm.forward(x)
    return x, w, b, xh + 0.5 * r(M, D), r(M), r(M), mean, rstd  # (gradients along xh: c2 is about one)


def planted(o, rstd, g, gm, gr, D):
    """The oracle's gradients with one mistake each."""
    rs, xh = rstd[:, None], o.xh
    worse = lambda **kw: SimpleNamespace(**{"x": o.x, "weight": o.weight, "bias": o.bias, **kw})  # noqa: E731
    return {"c2 off by one percent": worse(x=o.x - 0.01 * rs * xh * o.c2),
            "c1 off by one percent": worse(x=o.x - 0.01 * rs * o.c1),
            "the gradient of rstd off by one percent": worse(x=o.x - 0.01 * (gr * rstd ** 2)[:, None] * xh / D),
            "the gradient of rstd with one rstd": worse(x=o.x + ((gr * rstd ** 2) - (gr * rstd))[:, None] * xh / D),
            "no gradient of the mean": worse(x=o.x - gm[:, None] / D),
            "a row missing from dw": worse(weight=o.weight - g[-1] * xh[-1]),
            "a row twice in db": worse(bias=o.bias + g[0])}


def autograd(x, w, b, g, gm, gr):
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    X, W, B = leaves
    mean = X.mean(1)
    rstd = ((X - mean[:, None]) ** 2).mean(1).add(1e-5).rsqrt()
    y = (X - mean[:, None]) * rstd[:, None] * W + B
    ((y * g).sum() + (mean * gm).sum() + (rstd * gr).sum()).backward()
    return [t.grad for t in leaves]


def pin(got, want):
    """The oracle's pin: equal to autograd in 64 bits."""
    for name, leaf in zip(("x", "weight", "bias"), want):
        torch.testing.assert_close(getattr(got, name), leaf, atol=1e-12, rtol=1e-12)


def test_the_pin_rejects_planted_mistakes():
    x, w, b, g, gm, gr, mean, rstd = inputs()
    o = onorm.backward(g, x - mean[:, None], rstd, w, gm, gr)
    want = autograd(x, w, b, g, gm, gr)
    pin(o, want)
    for what, bad in planted(o, rstd, g, gm, gr, x.shape[1]).items():
        with pytest.raises(AssertionError):
            pin(bad, want)
            pytest.fail(what)  # (not an AssertionError)


@pytest.mark.parametrize("exact_input", [False, True])
def test_the_bounds_of_the_gpu_tests_reject_planted_mistakes(exact_input):
    """The oracle's result rounded to fp32 stands for the kernels'."""
    x, w, b, g, gm, gr, _, _ = inputs()
    x, w, b, g, gm, gr = (t.float() for t in (x, w, b, g, gm, gr))
    _, mean, rstd, _ = onorm.forward(x)
    d = x.double() - mean[:, None]
    o = onorm.backward(g, d, rstd, w, gm, gr)

    def check(result):
        got = SimpleNamespace(**{n: getattr(result, n).float() for n in ("x", "weight", "bias")})
        check_backward(g, d, rstd, w, b, got, mean, gm, gr, exact_input=exact_input)

    check(o)
    for what, bad in planted(o, rstd, g.double(), gm.double(), gr.double(), x.shape[1]).items():
        with pytest.raises(AssertionError):
            check(bad)
            pytest.fail(what)


def test_the_bounds_for_16_bits_reject_planted_mistakes():
    x, w, b, g, gm, gr, _, _ = inputs(seed=1)
    x, g = x.bfloat16(), g.bfloat16()
    _, mean, rstd, _ = onorm.forward(x)
    d = x.double() - mean[:, None]
    o = onorm.backward(g, d, rstd, w.float(), gm.float(), gr.float())

    def check(result):
        got = SimpleNamespace(x=result.x.bfloat16(), weight=result.weight.float(), bias=result.bias.float())
        check_backward(g, d, rstd, w.float(), b.float(), got, mean, gm.float(), gr.float())

    check(o)
    bad = planted(o, rstd, g.double(), gm, gr, x.shape[1])
    for what in ("c2 off by one percent", "the gradient of rstd with one rstd", "a row missing from dw", "a row twice in db"):
        with pytest.raises(AssertionError):
            check(bad[what])
            pytest.fail(what)
