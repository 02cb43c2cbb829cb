"""GPU: the norm undone where its input is infinite, and where the inverse of rstd is near the largest number, against the
formulas in float64 (tolerances as in test_gpu_norm.py)."""

import pytest
import torch

from oracle import norm as onorm
from saeflow_amd import kernels
from test_gpu_norm import U, cuda, half, tiny, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_infinities_through_the_norm_undone_stay_infinities(dtype):
    M, D = 64, 130
    g = torch.Generator().manual_seed(0)
    h, gr = torch.randn(M, D, generator=g), torch.randn(M, D, generator=g)
    mean, rstd = torch.randn(M, generator=g), torch.exp(0.5 * torch.randn(M, generator=g))
    rstd[0] = 1.0  # 1 / rstd without a remainder
    h[:, 3], h[:, 129], gr[:, 64] = float("inf"), -float("inf"), float("inf")
    h[5, 7], gr[6, 8] = float("nan"), float("nan")
    h, gr = h.to(dtype), gr.to(dtype)
    hg, gg, mg, rg = cuda(h, gr, mean, rstd)
    out = kernels.denormalize(hg, mg, rg).cpu()
    want = onorm.undone(h, mean, rstd)
    assert torch.equal(torch.isinf(out), torch.isinf(want)) and torch.equal(torch.isnan(out), torch.isnan(want))
    on = torch.isinf(want)
    assert torch.equal(out[on].double(), want[on])
    dh, dmean, _ = kernels.denormalize_backward(gg, hg, rg)
    dh = dh.cpu()
    want_dh, want_dm, _ = onorm.undone_backward(gr, h, rstd)
    assert torch.equal(torch.isinf(dh), torch.isinf(want_dh)) and torch.equal(torch.isnan(dh), torch.isnan(want_dh))
    assert torch.equal(torch.isinf(dmean.cpu()), torch.isinf(want_dm))
    on = torch.isfinite(want)
    mags = h.double().abs() / rstd.double()[:, None] + mean.double().abs()[:, None]
    within(out[on], want[on], (1.01 * half(dtype) * want.abs() + tiny(dtype) + 2 * U * mags)[on], "out")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_undone_where_the_inverse_is_near_the_largest_number(dtype):
    """1 / rstd of 1e37 to 3e38, of rows that small: as exact as elsewhere."""
    g = torch.Generator().manual_seed(1)
    h = (torch.rand(16, 200, generator=g) - 0.5).to(dtype)
    rstd = 1.0 / (10.0 ** torch.linspace(37, 38.4, 16, dtype=torch.float64))
    rstd = rstd.float()
    mean = 1e37 * torch.randn(16, generator=g)
    hg, mg, rg = cuda(h, mean, rstd)
    out, want = kernels.denormalize(hg, mg, rg), onorm.undone(h, mean, rstd)
    mags = h.double().abs() / rstd.double()[:, None] + mean.double().abs()[:, None]
    within(out, want, 1.01 * half(dtype) * want.abs() + 2 * U * mags, "out")


def test_undone_far_past_the_largest_number_is_infinite():
    """Both parts of h / rstd overflow, of whatever signs."""
    g = torch.Generator().manual_seed(2)
    h, mean = 1e12 * torch.randn(40, 100, generator=g), torch.randn(40, generator=g)
    rstd = (1.0 / (1e37 * (1 + 3 * torch.rand(40, generator=g)))).float()
    h[0] = 0.0
    hg, mg, rg = cuda(h, mean, rstd)
    want = onorm.undone(h, mean, rstd).float()
    assert torch.isinf(want[1:]).all()
    assert torch.equal(kernels.denormalize(hg, mg, rg).cpu(), want)
    assert torch.equal(kernels.denormalize_backward(hg, None, rg, need_grad_stats=False)[0].cpu(), (h.double() / rstd.double()[:, None]).float())
