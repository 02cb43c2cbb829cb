"""CPU: the layer norm oracle against float64 autograd and finite differences, and what the entry points refuse
(nothing here reaches a kernel)."""

import ctypes
import inspect

import pytest
import torch

import saeflow_amd
from oracle import norm as onorm
from saeflow_amd import SAE, Fp8Encoder, _lib, kernels


def _inputs(M=5, D=37, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    return r(M, D) * 2 + 0.5, 1 + 0.3 * r(D), r(D), r(M, D), r(M), r(M)


def test_oracle_forward_is_torchs_layer_norm():
    x, w, b, *_ = _inputs()
    want = torch.nn.functional.layer_norm(x, (x.shape[1],), w, b, 1e-5)
    torch.testing.assert_close(onorm.forward(x, w, b)[0], want, atol=1e-13, rtol=1e-13)


def test_oracle_backward_matches_autograd_and_finite_differences():
    x, w, b, g, gm, gr = _inputs()
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]

    def loss(x, w, b):
        mean = x.mean(1)
        rstd = ((x - mean[:, None]) ** 2).mean(1).add(1e-5).rsqrt()
        y = (x - mean[:, None]) * rstd[:, None] * w + b
        return (y * g).sum() + (mean * gm).sum() + (rstd * gr).sum()

    loss(*leaves).backward()
    _, mean, rstd, _ = onorm.forward(x)
    got = onorm.backward(g, x - mean[:, None], rstd, w, gm, gr)
    for name, leaf in zip(("x", "weight", "bias"), leaves):
        torch.testing.assert_close(getattr(got, name), leaf.grad, atol=1e-12, rtol=1e-12)
    for at in ((0, 0), (3, 17), (4, 36)):
        step = torch.zeros_like(x)
        step[at] = 1e-5
        diff = (loss(x + step, w, b) - loss(x - step, w, b)) / 2e-5
        torch.testing.assert_close(got.x[at], diff, atol=1e-7, rtol=1e-7)


def test_oracle_undone_is_the_inverse_and_its_gradients_match_autograd():
    x, _, _, g, *_ = _inputs()
    _, mean, rstd, xh = onorm.forward(x)
    torch.testing.assert_close(onorm.undone(xh, mean, rstd), x, atol=1e-13, rtol=1e-13)
    leaves = [t.clone().requires_grad_(True) for t in (xh, mean, rstd)]
    (onorm_undone(*leaves) * g).sum().backward()
    for got, leaf in zip(onorm.undone_backward(g, xh, rstd), leaves):
        torch.testing.assert_close(got, leaf.grad, atol=1e-12, rtol=1e-12)


def onorm_undone(h, mean, rstd):
    return h / rstd[:, None] + mean[:, None]


def test_a_planted_mistake_fails_the_pin():
    x, w, b, g, *_ = _inputs()
    _, mean, rstd, _ = onorm.forward(x)
    good = onorm.backward(g, x - mean[:, None], rstd, w)
    bad = good.x + rstd[:, None] * good.xh * good.c2 * 1.01  # c2 off by one percent of itself twice over
    assert (bad - good.x).abs().max() > 1e-3


def test_cpu_tensors_are_refused():
    x, v, s = torch.zeros(4, 8), torch.zeros(8), torch.zeros(4)
    for call in (lambda: kernels.layer_norm(x), lambda: kernels.layer_norm_held(x, v, v),
                 lambda: kernels.layer_norm_backward(x, x, s, s, v, v), lambda: kernels.denormalize(x, s, s),
                 lambda: kernels.denormalize_backward(x, x, s), lambda: saeflow_amd.layer_norm(x),
                 lambda: saeflow_amd.denormalize(x, s, s)):
        with pytest.raises(ValueError, match="GPU only"):
            call()


def test_shapes_and_values_are_refused():
    x, s = torch.zeros(4, 8), torch.zeros(4)
    for call, match in ((lambda: kernels.layer_norm(torch.zeros(8)), "two dimensions"),
                        (lambda: kernels.layer_norm(torch.zeros(4, 0)), "no elements"),
                        (lambda: kernels.layer_norm(x, torch.zeros(7)), "weight must have shape"),
                        (lambda: kernels.layer_norm(x, None, torch.zeros(2, 4)), "bias must have shape"),
                        (lambda: kernels.layer_norm(x, eps=-1e-5), "eps"),
                        (lambda: kernels.layer_norm(x, eps=float("nan")), "eps"),
                        (lambda: kernels.layer_norm_backward(x, torch.zeros(4, 7), s, s), "x"),
                        (lambda: kernels.layer_norm_backward(x, x, s, s.double()), "rstd"),
                        (lambda: kernels.layer_norm_backward(x, x, torch.zeros(5), s), "mean"),
                        (lambda: kernels.layer_norm_backward(x, x, s, s, bias=torch.zeros(9)), "bias"),
                        (lambda: kernels.layer_norm_backward(x, x, s, s, grad_rstd=torch.zeros(3)), "grad_rstd"),
                        (lambda: kernels.denormalize(x, s, torch.zeros(3)), "rstd"),
                        (lambda: kernels.denormalize_backward(x, None, s), "need h"),
                        (lambda: kernels.denormalize_backward(x, torch.zeros(4, 9), s), "h"),
                        (lambda: kernels.layer_norm_backward(x, x, None, s), "mean"),
                        (lambda: kernels.layer_norm_backward(x, x, s, None), "rstd"),
                        (lambda: saeflow_amd.layer_norm(torch.zeros(3, 0)), "dimension"),
                        (lambda: saeflow_amd.denormalize(torch.zeros(3, 0), torch.zeros(3), torch.zeros(3)), "mean and rstd"),
                        (lambda: saeflow_amd.layer_norm(x, hold=torch.int8), "hold"),
                        (lambda: saeflow_amd.layer_norm(torch.tensor(1.0)), "dimension"),
                        (lambda: saeflow_amd.denormalize(x, torch.zeros(4, 1), s), "needs mean and rstd"),
                        (lambda: saeflow_amd.forward_train(SAE(8, 16), x, hold="fp8"), "hold"),
                        (lambda: SAE(8, 16, input_norm="batch"), "input_norm"),
                        (lambda: Fp8Encoder(torch.zeros(8, 16), torch.zeros(16), torch.zeros(8), input_norm="rms"),
                         "input_norm")):
        with pytest.raises(ValueError, match=match):
            call()


def test_a_duck_typed_sae_needs_no_input_norm_and_a_wrong_one_is_refused():
    from saeflow_amd import ops

    class Duck:
        pass

    assert ops.input_norm(Duck()) is None
    duck = Duck()
    duck.input_norm = "group_norm"
    with pytest.raises(ValueError, match="input_norm"):
        ops.encode_sparse(duck, torch.zeros(2, 8))
    assert list(inspect.signature(SAE.__init__).parameters)[:7] == ["self", "d_in", "d_sae", "activation", "k", "device",
                                                                    "dtype"]


def test_c_abi_refuses_bad_arguments_without_touching_the_gpu():
    lib = _lib.load()

    def norm(M=4, D=8, x=16, dt=1, y=16, sym=8, eps=1e-5, q=None, sq=0, scale=None, ss=0, w=None, w_dt=0):
        return lib.sf_layer_norm(x, D, dt, w, w_dt, None, 0, eps, M, D, y, sym, 1, None, None, q, sq, scale, ss, None)

    def refused(rc, text):
        assert rc == _lib.SF_EINVAL and text in lib.sf_last_error(), lib.sf_last_error()

    refused(norm(M=-1), b"shape")
    refused(norm(D=0), b"shape")
    refused(norm(D=(1 << 24) + 1), b"shape")
    refused(norm(dt=7), b"dtype")
    refused(norm(w=16, w_dt=5), b"dtype")
    refused(norm(eps=-1.0), b"eps")
    refused(norm(eps=float("nan")), b"eps")
    refused(norm(x=None), b"x must not be NULL")
    refused(norm(x=17), b"aligned")
    refused(norm(y=None), b"y must not be NULL")
    refused(norm(sym=7), b"overlap")
    refused(norm(q=16, sq=128), b"NULL")
    refused(norm(scale=16, ss=4), b"NULL")
    refused(norm(q=24, sq=128, scale=16, ss=4), b"16-B")
    refused(norm(q=16, sq=112, scale=16, ss=4), b"too short")
    refused(norm(q=16, sq=128, scale=16, ss=3), b"4-B")
    assert norm(M=0) == _lib.SF_OK

    def back(M=4, D=8, g=16, x=16, q=None, sq=0, scale=None, ss=0, mean=16, rstd=16, dx=16, dw=None, ws=None, wsb=0):
        return lib.sf_layer_norm_backward(g, D, 1, x, D, 1, q, sq, scale, ss, mean, rstd, None, 0, None, None, M, D, dx,
                                          D, 1, dw, 0, None, 0, ws, wsb, None)

    refused(back(g=None), b"g must not be NULL")
    refused(back(x=None), b"not both")
    refused(back(q=16, sq=128, scale=16, ss=4), b"not both")
    refused(back(mean=None), b"mean")
    refused(back(rstd=None), b"rstd")
    refused(back(x=None, q=16, sq=64, scale=16, ss=4), b"too short")
    need = ctypes.c_int64()
    assert lib.sf_layer_norm_backward_workspace_size(4000, 2304, ctypes.byref(need)) == _lib.SF_OK and need.value > 0
    refused(back(M=4000, D=2304, dw=16, ws=16, wsb=need.value - 1), b"workspace")
    refused(lib.sf_layer_norm_backward_workspace_size(4, 0, ctypes.byref(need)), b"shape")
    assert back(M=0) == _lib.SF_OK
    assert back(dx=None) == _lib.SF_OK  # nothing asked for
    refused(lib.sf_denormalize(16, 8, 1, None, 16, 4, 8, 16, 8, 1, None), b"mean and rstd")
    refused(lib.sf_denormalize(16, 8, 3, 16, 16, 4, 8, 16, 8, 1, None), b"dtype")
    refused(lib.sf_denormalize_backward(16, 8, 1, None, 8, 1, 16, 4, 8, 16, 8, 1, 16, 16, None), b"h must not be NULL")
    refused(lib.sf_denormalize_backward(16, 8, 1, 16, 8, 1, None, 4, 8, 16, 8, 1, None, None, None), b"rstd")
    P = 16
    refused(lib.sf_backward_biases(P, 4, 8, 8, 5, P, 4, 4, 1, 1, P, None, 0, P, 0, P, 64, None), b"dtype")
    refused(lib.sf_backward_biases(P, 4, 8, 8, 1, P, 4, 4, 1, 1, None, None, 0, P, 0, P, 64, None), b"NULL")
    refused(lib.sf_backward_biases(P, 4, 8, 8, 1, P, 4, 4, 1, 1, P, None, 0, P, 0, P, 63, None), b"workspace")
    refused(lib.sf_backward_biases(P, -4, 8, 8, 1, P, 4, 4, 1, 1, P, None, 0, P, 0, P, 64, None), b"size")

    def held(q=P, sq=128, scale=P, ss=4):
        return lib.sf_backward_columns_held(P, P, P, P, P, P, P, 1, 1, P, 1, None, 0, P, 8, q, sq, scale, ss, P, 8, 1, 4, 4, 8,
                                            4, P, P, P, P, P, P, 64, None)

    refused(held(q=None), b"NULL codes")
    refused(held(q=24), b"16-B")
    refused(held(sq=64), b"too short")
    refused(held(ss=2), b"4-B")
