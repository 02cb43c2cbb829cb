"""CPU: the 64-bit definition of 8-bit rows against torch's own e4m3, Fp8Rows on the host, and what the
wrappers and the C ABI refuse before anything reaches a GPU."""

import copy
import ctypes
import pickle

import numpy as np
import pytest
import torch

import saeflow_amd
from oracle import fp8 as ofp8
from saeflow_amd import _lib
from saeflow_amd.cache import cache_activations
from saeflow_amd.kernels import Fp8Rows, dequantize_rows, fused_encode_fp8, quantize_rows


def test_oracle_code_values_are_torchs():
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(ofp8.CODES, want)


def test_oracle_rounding_is_torchs_within_a_block():
    x = torch.randn(40, 300) * 2.0 ** torch.randint(-12, 3, (40, 300)).float()
    codes, scale = ofp8.quantize(x.numpy())
    two = torch.from_numpy(np.repeat(2.0 ** (scale.astype(np.float64) - 127), 128, axis=1)[:, :300])
    want = (x.double() / two).float().to(torch.float8_e4m3fn).double()
    np.testing.assert_array_equal(codes, want.numpy())
    assert (np.abs(codes) <= 448).all()
    # the scale is the smallest: half of it would not hold the largest element
    top = np.abs(x.double().numpy()).reshape(40, -1)[:, :128].max(1)
    assert (top > 448 * 2.0 ** (scale[:, 0].astype(np.float64) - 128)).all()


@pytest.mark.parametrize("a,e", [(0.0, -127), (448.0, 0), (448.0000001, 1), (447.0, 0), (224.0, -1), (1.0, -8),
                                 (2.0 ** -149, -127), (3.4028234663852886e38, 120)])
def test_oracle_exponent(a, e):
    assert ofp8.exponent(a) == e


def host_rows(R, d):
    return Fp8Rows.from_parts(torch.zeros(R, d).to(torch.float8_e4m3fn), torch.zeros(R, -(-d // 128), dtype=torch.uint8))


@pytest.mark.parametrize("d", [1, 127, 128, 129, 600])
def test_rows_on_the_host(d):
    r = host_rows(5, d)
    assert r.shape == (5, d) and len(r) == 5 and r.device.type == "cpu"
    assert r.q.shape[1] % 128 == 0 and r.q.shape[1] - d < 128 and r.scale.shape[1] % 4 == 0
    assert r.nbytes == r.q.numel() + r.scale.numel()
    part = r[1:4]
    assert len(part) == 3 and part.q.data_ptr() == r.q[1:].data_ptr()
    assert len(Fp8Rows.empty(0, d, "cpu")) == 0 and "x" in repr(r)


def test_copies_and_pickles_hold_their_own_memory():
    r = Fp8Rows(torch.randn(5, 256).to(torch.float8_e4m3fn), torch.randint(120, 130, (5, 4), dtype=torch.uint8), 200)
    for other in (copy.deepcopy(r), pickle.loads(pickle.dumps(r))):
        assert other.shape == r.shape and other.q.data_ptr() != r.q.data_ptr()
        assert torch.equal(other.q.view(torch.uint8), r.q.view(torch.uint8)) and torch.equal(other.scale, r.scale)
        assert other._args() == (other.q.data_ptr(), 256, other.scale.data_ptr(), 4)
    for name, value in (("q", r.q[:3]), ("scale", r.scale[:3]), ("d", 100)):
        with pytest.raises(AttributeError):
            setattr(r, name, value)
    assert len(r) == 5 and r.d == 200


def test_bad_rows_are_refused():
    q, s = torch.zeros(4, 256).to(torch.float8_e4m3fn), torch.zeros(4, 4, dtype=torch.uint8)
    Fp8Rows(q, s, 200)
    for bad in (lambda: Fp8Rows(q.view(torch.uint8), s, 200), lambda: Fp8Rows(q, s.int(), 200), lambda: Fp8Rows(q, s, 0),
                lambda: Fp8Rows(q, s, 128), lambda: Fp8Rows(q, s, 257), lambda: Fp8Rows(q[:3], s, 200),
                lambda: Fp8Rows(q, s[:, :2], 200), lambda: Fp8Rows(q[0], s, 200),
                lambda: Fp8Rows(torch.zeros(256, 4).to(torch.float8_e4m3fn).T, s, 200),
                lambda: Fp8Rows.from_parts(q, s), lambda: Fp8Rows.from_parts(q.float(), s[:, :2])):
        with pytest.raises(ValueError):
            bad()


def test_host_tensors_are_refused(tmp_path):
    x, r = torch.randn(5, 200), host_rows(5, 200)
    for call in (lambda: quantize_rows(x), lambda: quantize_rows(x, out=r), lambda: dequantize_rows(r),
                 lambda: fused_encode_fp8(x, r), lambda: fused_encode_fp8(r, r),
                 lambda: saeflow_amd.ActivationBuffer(4, 8, device="cpu"),
                 lambda: saeflow_amd.Fp8Encoder(x, x[0], x[:, 0])):
        with pytest.raises(ValueError, match="GPU only"):
            call()


def test_cache_refuses_other_types(tmp_path):
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        cache_activations(None, torch.zeros(1, 1, dtype=torch.long), [], tmp_path, dtype=torch.float8_e5m2)


def test_c_abi_refuses_before_any_launch():
    """Every argument that the kernels rely on: types, strides, alignment, shapes, workspaces."""
    lib, p = _lib.load(), 4096  # (an address that is never used)

    def refused(rc, text):
        assert rc == _lib.SF_EINVAL and text in lib.sf_last_error(), lib.sf_last_error()

    def quant(x=p, xdt=1, shift=None, sdt=0, M=4, K=200, q=p, sq=256, s=p, ss=4, row0=0, R=8):
        return lib.sf_quantize_rows(x, K, 1, xdt, shift, sdt, M, K, q, sq, s, ss, row0, R, None)

    assert quant(M=0) == _lib.SF_OK
    refused(quant(xdt=7), b"dtype")
    refused(quant(shift=p, sdt=9), b"dtype")
    refused(quant(M=-1), b"shape")
    refused(quant(K=0), b"shape")
    refused(quant(x=None), b"NULL")
    refused(quant(q=None), b"NULL")
    refused(quant(q=p + 8), b"aligned")
    refused(quant(sq=264), b"aligned")
    refused(quant(sq=128), b"needed")
    refused(quant(s=p + 2), b"aligned")
    refused(quant(ss=2), b"aligned")
    refused(quant(K=600, sq=640, ss=4), b"needed")
    refused(quant(M=9), b"fit")
    refused(quant(row0=8), b"outside")
    refused(quant(row0=-1), b"outside")

    def deq(q=p, sq=256, s=p, ss=4, R=8, rows=None, row0=0, M=4, K=200, out=p, som=200, odt=1):
        return lib.sf_dequantize_rows(q, sq, s, ss, R, rows, row0, None, 0, M, K, out, som, odt, None)

    assert deq(M=0) == _lib.SF_OK
    refused(deq(odt=3), b"dtype")
    refused(deq(out=None), b"NULL")
    refused(deq(som=199), b"overlap")
    refused(deq(M=9), b"asked")
    refused(deq(row0=8), b"outside")
    refused(deq(sq=250), b"aligned")
    refused(deq(R=0, rows=p), b"no rows")

    def enc(xq=p, sxq=256, xs=p, sxs=4, wq=p, swq=256, ws=p, sws=4, b=None, bdt=0, thr=None, tdt=0, out=p, som=10, odt=1,
            M=4, N=10, K=200, act=0, work=p, nbytes=1 << 20):
        return lib.sf_encode_fp8_rows(xq, sxq, xs, sxs, wq, swq, ws, sws, b, bdt, thr, tdt, out, som, odt, None, M, N, K,
                                      act, work, nbytes, None)

    assert enc(M=0) == _lib.SF_OK and enc(N=0) == _lib.SF_OK
    refused(enc(odt=5), b"dtype")
    refused(enc(b=p, bdt=5), b"dtype")
    refused(enc(act=3), b"activation")
    refused(enc(act=1), b"threshold")
    refused(enc(K=0), b"size")
    refused(enc(K=1 << 23), b"large")
    refused(enc(out=None), b"NULL")
    refused(enc(som=9), b"overlap")
    refused(enc(work=None), b"workspace")
    refused(enc(work=p + 4), b"workspace")
    refused(enc(nbytes=16), b"workspace")
    refused(enc(xq=None), b"x: codes")
    refused(enc(wq=p + 4), b"w: rows of codes")
    refused(enc(swq=128), b"w: rows of codes")
    refused(enc(sxq=1 << 23), b"x: rows of codes")
    refused(enc(sws=2), b"w: rows of scales")

    size = ctypes.c_int64()
    assert lib.sf_encode_fp8_workspace_size(10, 200, ctypes.byref(size)) == _lib.SF_OK
    assert size.value >= 10 * (256 + 4) and size.value % 64 == 0
    refused(lib.sf_encode_fp8_workspace_size(-1, 200, ctypes.byref(size)), b"size")
    refused(lib.sf_encode_fp8_workspace_size(1, 200, None), b"NULL")

    def tok(x=p, xdt=1, bd=None, bdt=0, work=p, nbytes=1 << 20, M=100):
        return lib.sf_encode_fp8(x, 200, 1, xdt, bd, bdt, p, 256, p, 4, None, 0, None, 0, p, 10, 1, None, M, 10, 200, 0,
                                 work, nbytes, None)

    refused(tok(xdt=4), b"dtype")
    refused(tok(bd=p, bdt=4), b"dtype")
    refused(tok(x=None), b"NULL")
    refused(tok(nbytes=100 * 260), b"workspace")


@pytest.mark.parametrize("M,N", [(4, 10), (0, 10), (4, 0)])
def test_counts_without_an_activation_are_refused(M, N):
    """Bare pre-activations have no nonzeros to count: refused as sf_encode refuses it, before any launch."""
    lib, p = _lib.load(), 4096  # (an address that is never used)

    def tail(act):
        return (p, 256, p, 4, None, 0, None, 0, p, 10, 1, p, M, N, 200, act, p, 1 << 20, None)

    for call, x in ((lib.sf_encode_fp8_rows, (p, 256, p, 4)), (lib.sf_encode_fp8, (p, 200, 1, 1, None, 0))):
        assert call(*x, *tail(_lib.ACT["none"])) == _lib.SF_EINVAL
        assert b"row counts need relu or jumprelu" in lib.sf_last_error()
    x, W, nnz = torch.randn(M, 200), host_rows(N, 200), torch.zeros(M, dtype=torch.int32)
    for rows in (x, host_rows(M, 200)):
        with pytest.raises(ValueError, match="row counts need relu or jumprelu"):
            fused_encode_fp8(rows, W, activation="none", row_nnz=nnz)
