"""GPU: layer norm of rows whose squares leave fp32, against the formulas in float64 (tolerances as in test_gpu_norm.py)."""

import pytest
import torch

from oracle import norm as onorm
from saeflow_amd import SAE, kernels
from test_gpu_norm import U, check_backward, check_forward, check_held, cuda, held_values, make, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [6, 40, 1000, 5000, 8500])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-30, 1e-22, 1e20, 1e30])
def test_rows_whose_squares_leave_fp32(size, dtype, D):
    """Sums of squares over the largest number of fp32, and (with no eps) under its smallest normal one."""
    x, w, b, g = make(9, D, dtype, seed=D)
    x = x * size
    assert torch.isfinite(x).all() and (x != 0).any(1).all()
    xg, wg, bg, gg = cuda(x, w, b, g)
    for eps in (0.0, 1e-5) if size > 1 else (0.0,):
        y, held, mean, rstd = kernels.layer_norm_held(xg, wg, bg, eps=eps)
        check_forward(x, w, b, y, mean, rstd, eps=eps)
        check_held(x, held)
        if dtype != torch.float32:  # y of another type than x: another kernel
            y32, _, _ = kernels.layer_norm(xg, wg, bg, eps=eps, out_dtype=torch.float32)
            check_forward(x, w, b, y32, mean, rstd, eps=eps)
    _, mean64, rstd64, _ = onorm.forward(x, eps=eps)
    if dtype == torch.float32 or 1e-22 <= size <= 1e20:  # (gradients of the rows go with 1 / size)
        check_backward(g, x.double() - mean64[:, None], rstd64, w, b, kernels.layer_norm_backward(gg, xg, mean, rstd, wg, bg), mean64)
        check_backward(g, held_values(held), rstd.cpu(), w, b, kernels.layer_norm_backward(gg, held, None, rstd, wg, bg), mean64, exact_input=True)


@pytest.mark.parametrize("D", [7, 96, 2304, 4097, 9000])
def test_rows_up_to_the_largest_number(D):
    x, w, b, _ = make(5, D, torch.float32, seed=D)
    x = x * 1e36
    x[2] = torch.linspace(-1, 1, D) * 3e38
    x[3] = torch.randn(D)  # an ordinary row among them
    xg, wg, bg = cuda(x, w, b)
    y, held, mean, rstd = kernels.layer_norm_held(xg, wg, bg)
    assert torch.isfinite(y).all() and (rstd > 0).all()
    ordinary = [0, 1, 3, 4]
    check_forward(x[ordinary], w, b, y[ordinary], mean[ordinary], rstd[ordinary])
    # a rstd of 2^-127 has 22 bits
    want, _, rstd64, xh = onorm.forward(x[2:3], w, b)
    within(rstd[2:3], rstd64, U * (D / 128 + 16) * rstd64 + 2.0 ** -149, "rstd")
    within(y[2:3], want, U * (D / 128 + 32) * (want.abs() + (xh * w.double()).abs() + b.double().abs()) + 2.0 ** -149 * (xh * w.double() / rstd64[:, None]).abs(), "y")
    check_held(x, held)


@pytest.mark.parametrize("D", [7, 96, 1000, 5000, 9000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_whose_deviations_are_infinite_are_not_numbers(dtype, D):
    """All of the row, not the element whose deviation is; gradients too."""
    x, w, b, g = make(5, D, dtype, seed=D)
    x[1], x[3] = -3e38, 3e38
    x[1, D - 1], x[3, 0] = 3e38, -3e38
    xg, wg, bg, gg = cuda(x, w, b, g)
    y, held, mean, rstd = kernels.layer_norm_held(xg, wg, bg)
    y32, _, _ = kernels.layer_norm(xg, wg, bg, out_dtype=torch.float32)
    clean = [0, 2, 4]
    assert torch.isnan(y[[1, 3]]).all() and torch.isnan(y32[[1, 3]]).all() and torch.isfinite(mean).all()
    check_forward(x[clean], w, b, y[clean], mean[clean], rstd[clean])
    for source in (xg, held):
        gr = kernels.layer_norm_backward(gg, source, mean, rstd, wg, bg)
        assert torch.isnan(gr.x[[1, 3]]).all() and torch.isfinite(gr.x[clean]).all()


def test_a_dictionary_over_rows_whose_squares_leave_fp32():
    """The reconstruction in the rows' own space goes with their size."""
    torch.manual_seed(0)
    sae = SAE(96, 256, "relu", input_norm="layer_norm", norm_eps=0.0).cuda()
    x = torch.randn(20, 96, device="cuda") + 0.5
    small, size = sae(x), 2.0 ** 67
    big = sae(x * size)
    assert torch.isfinite(big).all()
    # each side's rstd is off by D / 128 + 16 units (z by as much), the products' sums by D and by the features a row has
    torch.testing.assert_close(big / size, small, atol=1e-4, rtol=1e-4)
