"""CPU: what sparse_backward refuses before anything reaches a kernel, from tokens and from 8-bit rows."""

import pytest
import torch

from saeflow_amd.kernels import Fp8Rows, sparse_backward

M, D, N, NNZ = 6, 64, 32, 20


@pytest.mark.parametrize("held", [False, True])
@pytest.mark.parametrize("what,match", [("b_enc", "b_enc"), ("b_dec", "b_dec"),
                                        ("grad_x_hat of fewer rows", "grad_x_hat"), ("grad_x_hat of other columns", "grad_x_hat"),
                                        ("grad_x_hat of one dimension", "grad_x_hat"), ("values", "values"), ("indptr", "int64"),
                                        ("indices", "integer"), (None, "GPU only")])
def test_shapes_and_types_that_do_not_fit_are_refused(what, match, held):
    x = Fp8Rows.empty(M, D, "cpu") if held else torch.zeros(M, D)
    b_enc, b_dec, g, values = torch.zeros(N), torch.zeros(D), torch.zeros(M, D), torch.zeros(NNZ)
    indptr, indices = torch.zeros(M + 1, dtype=torch.int64), torch.zeros(NNZ, dtype=torch.int32)
    if what == "b_enc":
        b_enc = torch.zeros(N - 1)
    elif what == "b_dec":
        b_dec = torch.zeros(D - 1)
    elif what == "grad_x_hat of fewer rows":
        g = g[1:]
    elif what == "grad_x_hat of other columns":
        g = g[:, :60]
    elif what == "grad_x_hat of one dimension":
        g = g.flatten()
    elif what == "values":
        values = values[1:]
    elif what == "indptr":
        indptr = indptr.int()
    elif what == "indices":
        indices = indices.float()
    with pytest.raises(ValueError, match=match):
        sparse_backward(x, torch.zeros(D, N), b_enc, torch.zeros(N, D), b_dec, (indptr, indices, values), g)
