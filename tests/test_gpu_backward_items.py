"""GPU: the sparse backward where four work items share a wave, over types, rows that take element loads, several slabs, and
columns of over 64 and over 256 entries among the short ones, against the formulas in float64.

Tolerances, with u = 2^-24 and e / 2 the half step of a result's type: dL/dpre of an entry is a dot product of D terms (at most
D / 64 + 24 additions to a lane's sum, and one for each slab) plus a given gradient; a feature's sum over n entries adds them
one after the other (n + 8 with the parts of long columns). Each is bounded by u times that number times the sum of
magnitudes.
"""

import re
from pathlib import Path

import pytest
import torch

from saeflow_amd import _lib
from saeflow_amd.kernels import quantize_rows, sparse_backward
from test_gpu_norm import U, cuda, half, held_values, tiny, within

pytestmark = pytest.mark.gpu


def least_waves():
    """From how many waves on four items share one: the rule of units_per_wave."""
    source = (Path(_lib.__file__).parent / "csrc" / "backward.hip").read_text()
    return int(re.search(r"nnz < 4 \* N && waves >= (\d+) \? 4 : 1", source).group(1))


@pytest.mark.parametrize("held", [False, True])
@pytest.mark.parametrize("dtype,D", [(torch.float32, 600), (torch.float32, 601), (torch.bfloat16, 1000), (torch.bfloat16, 1003),
                                     (torch.float16, 1000), (torch.float16, 1003)])
def test_sparse_backward_four_items_a_wave(dtype, D, held):
    M, slabs = 320, -(-D * dtype.itemsize // 1024)
    N = least_waves() // slabs + 10
    g = torch.Generator().manual_seed(D)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    on = torch.rand(M, N, generator=g) < 1.4 / M
    on[:, 100::4001] = True                          # over 256 entries
    on[:90, 101::2003] = True                        # over 64
    on[5] = False                                    # a token without features
    on[:, 7:40] = False                              # features that no token has
    f = (n(M, N).abs() + 0.1) * on
    x, G = (n(M, D) + 0.2).to(dtype), (0.1 * n(M, D)).to(dtype)
    W_enc, W_dec = (n(D, N) / D ** 0.5).to(dtype), (n(N, D) / D ** 0.5).to(dtype)
    b_enc, b_dec, f = (0.1 * n(N)).to(dtype), (0.1 * n(D)).to(dtype), f.to(dtype)
    indptr = torch.cat([torch.zeros(1, dtype=torch.int64), on.sum(1).cumsum(0)])
    indices, values = on.nonzero()[:, 1].int(), f[on]
    nnz = indices.numel()
    H = (0.05 * n(nnz)).to(dtype)
    _, items, _, floats = _lib.backward_sizes(M, N, nnz, D, _lib.DTYPE[dtype])
    assert floats == (slabs + 1) * nnz and items * slabs >= least_waves() and nnz < 4 * N
    xg, We, be, Wd, bd, ip, ix, va, Gg, Hg = cuda(x, W_enc, b_enc, W_dec, b_dec, indptr, indices, values, G, H)
    rows = quantize_rows(xg, shift=bd) if held else xg
    got = sparse_backward(rows, We, be, Wd, bd, (ip, ix, va), Gg, Hg)
    again = sparse_backward(rows, We, be, Wd, bd, (ip, ix, va), Gg, Hg)
    for name in ("W_enc", "W_dec", "b_enc", "b_dec", "pre", "x"):
        assert torch.equal(getattr(got, name), getattr(again, name)), name

    xs = held_values(rows) if held else (x.float() - b_dec.float()).to(dtype).double()
    Gd, Wdd, fd = G.double(), W_dec.double(), f.double()
    Hd = torch.zeros(M, N, dtype=torch.float64)
    Hd[on] = H.double()
    p, pa = (Gd @ Wdd.T + Hd) * on, (Gd.abs() @ Wdd.abs().T + Hd.abs()) * on
    dot, entries = D / 64 + 24 + slabs, on.sum(0).double()
    within(got.pre, p[on], U * dot * pa[on], "pre")

    def check(name, want, tol):
        result = getattr(got, name)
        assert result.dtype == dtype
        within(result, want, 1.01 * half(dtype) * want.abs() + tiny(dtype) + 1.01 * tol, name)

    check("W_enc", xs.T @ p, U * (entries + 8) * (xs.abs().T @ p.abs()) + U * dot * (xs.abs().T @ pa))
    check("W_dec", fd.T @ Gd, U * (entries[:, None] + 8) * (fd.abs().T @ Gd.abs()))
    check("b_enc", p.sum(0), U * (entries + 8) * p.abs().sum(0) + U * dot * pa.sum(0))
    assert (got.W_dec.cpu()[7:40] == 0).all() and (got.W_enc.cpu()[:, 7:40] == 0).all() and (got.b_enc.cpu()[7:40] == 0).all()
