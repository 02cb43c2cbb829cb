"""GPU: sparse_backward takes the column indices that sparse_decode takes."""

import pytest
import torch

from saeflow_amd.kernels import csr_transpose, quantize_rows, sparse_backward
from test_gpu_held import cuda, problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("held", [False, True])
def test_indices_of_any_integer_type(held):
    x, W_enc, b_enc, W_dec, b_dec, csr, _, G, H = problem(40, 96, 120, torch.bfloat16)
    xg, We, be, Wd, bd, ip, ix, va, Gg, Hg = cuda(x, W_enc, b_enc, W_dec, b_dec, *csr, G, H)
    rows = quantize_rows(xg, shift=bd) if held else xg
    want = sparse_backward(rows, We, be, Wd, bd, (ip, ix, va), Gg, Hg)
    for dtype in (torch.int64, torch.int16, torch.uint8):
        got = sparse_backward(rows, We, be, Wd, bd, (ip, ix.to(dtype), va), Gg, Hg)
        for name in ("W_enc", "b_enc", "W_dec", "b_dec", "pre", "x"):
            assert torch.equal(getattr(got, name), getattr(want, name)), (dtype, name)


def test_transposes_of_indices_of_any_integer_type():
    *_, csr, _, _, _ = problem(40, 8, 120, torch.bfloat16)
    ip, ix = cuda(*csr[:2])
    want = csr_transpose(ip, ix, 120)
    for dtype in (torch.int64, torch.int16, torch.uint8):
        assert all(torch.equal(a, b) for a, b in zip(csr_transpose(ip, ix.to(dtype), 120), want))
    with pytest.raises(ValueError, match="int64"):
        csr_transpose(ip.int(), ix, 120)
