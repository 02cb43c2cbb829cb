"""GPU: sparse_backward takes the column indices that sparse_decode takes."""

import pytest
import torch

from saeflow_amd import _lib
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_8_bit_rows_of_no_elements(dtype):
    """At the C entry d_in may be zero, and then nothing is said of codes and scales: db_enc comes from the values' gradients."""
    *_, csr, _, _, H = problem(40, 8, 120, dtype)
    ip, ix, va, Hg = cuda(*csr, H)
    N, nnz, lib, dev = 120, ix.numel(), _lib.load(), ip.device
    colptr, rows, pos = csr_transpose(ip, ix, N)
    _, items, slots, floats = _lib.backward_sizes(40, N, nnz, 0, _lib.DTYPE[dtype])
    i32 = lambda n: torch.empty(max(n, 1), dtype=torch.int32, device=dev)  # noqa: E731
    plan, item_col, multi_col, slot_item = torch.empty(3 * (N + 1), dtype=torch.int64, device=dev), i32(items), i32(N), i32(slots)
    s = _lib.stream(dev)
    _lib.check(lib.sf_backward_plan(colptr.data_ptr(), N, nnz, plan.data_ptr(), item_col.data_ptr(), multi_col.data_ptr(),
                                    slot_item.data_ptr(), s))
    f32 = lambda n: torch.zeros(max(n, 1), dtype=torch.float32, device=dev)  # noqa: E731
    g_pre, d_wdec, d_benc, partials, work = f32(nnz), f32(N), f32(N), f32(slots), f32(floats)
    code = _lib.DTYPE[dtype]
    codes = torch.empty(16, dtype=torch.uint8, device=dev)
    _lib.check(lib.sf_backward_columns_held(
        colptr.data_ptr(), rows.data_ptr(), pos.data_ptr(), plan.data_ptr(), item_col.data_ptr(), multi_col.data_ptr(),
        slot_item.data_ptr(), items, slots, va.data_ptr(), code, Hg.data_ptr(), code, None, 0, codes.data_ptr(), 0, None, 0, None,
        0, code, N, 40, 0, nnz, g_pre.data_ptr(), d_wdec.data_ptr(), None, d_benc.data_ptr(), partials.data_ptr(),
        work.data_ptr(), floats, s))
    assert torch.equal(g_pre, Hg.float())
    want = torch.zeros(N, dtype=torch.float64).index_add_(0, csr[1].long(), H.double())
    sizes = torch.zeros(N, dtype=torch.float64).index_add_(0, csr[1].long(), H.double().abs())
    assert ((d_benc.double().cpu() - want).abs() <= 2.0 ** -24 * 50 * sizes).all()
