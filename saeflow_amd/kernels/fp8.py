"""Rows in 8 bits on gfx950: written, read back, and multiplied (C ABI, include/saeflow_hip.h).

The reference has no counterpart. A row is held as e4m3 codes with one power-of-two scale for each
block of 128 elements (the last block may be short): element = code * 2^(byte - 127), the byte's 2^e
the smallest, e >= -127, that brings the block's largest finite magnitude to 448 or less. Codes round
to nearest even, so an element keeps four significant bits down to 2^-6 of its scale and an absolute
2^-10 of it below; NaN and infinities become NaN. 16-bit rows take half the memory, fp32 a quarter.
"""

import torch

from .. import _lib
from .encode import _vector

BLOCK = 128
ACTIVATIONS = {"none": _lib.ACT["none"], "relu": _lib.ACT["relu"], "jumprelu": _lib.ACT["jumprelu"]}


def _up(n, m):
    return -(-n // m) * m


def _rows_of_bytes(q, scale, d):
    return Fp8Rows(q.view(torch.float8_e4m3fn), scale, d)


class Fp8Rows:
    """R rows of d elements in 8 bits: `q` [R, d rounded up to 128] float8_e4m3fn, zeros behind d, and
    `scale` [R, ceil(d / 128) rounded up to 4] uint8. Slicing rows gives a view. The three belong together, so
    they are not assigned to; copies and pickles are made of them alone."""

    __slots__ = ("q", "scale", "d", "_strides")

    def __init__(self, q, scale, d):
        if q.dtype != torch.float8_e4m3fn or scale.dtype != torch.uint8:
            raise ValueError(f"8-bit rows are float8_e4m3fn codes and uint8 scales, got {q.dtype} and {scale.dtype}")
        if d < 1 or q.dim() != 2 or scale.dim() != 2 or q.shape[0] != scale.shape[0]:
            raise ValueError(f"bad shapes for rows of {d}: codes {tuple(q.shape)}, scales {tuple(scale.shape)}")
        if q.shape[1] != _up(d, BLOCK) or scale.shape[1] != _up(_up(d, BLOCK) // BLOCK, 4):
            raise ValueError(f"rows of {d} are padded to {_up(d, BLOCK)} codes and {_up(_up(d, BLOCK) // BLOCK, 4)} "
                             f"scales, got {q.shape[1]} and {scale.shape[1]}")
        if q.stride(1) != 1 or scale.stride(1) != 1:
            raise ValueError("codes and scales must be contiguous along a row")
        if q.device != scale.device:
            raise ValueError(f"codes are on {q.device}, scales on {scale.device}")
        # a lone row's stride is not used and may be anything
        strides = (q.stride(0), scale.stride(0)) if q.shape[0] > 1 else (q.shape[1], scale.shape[1])
        for name, value in (("q", q), ("scale", scale), ("d", d), ("_strides", strides)):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError(f"{name} of 8-bit rows is not assigned to; make new Fp8Rows")

    def __reduce__(self):
        # (the codes as bytes: torch has no plain pickles of float8 tensors)
        return _rows_of_bytes, (self.q.view(torch.uint8), self.scale, self.d)

    def _args(self):
        """The C ABI's (codes, their stride, scales, their stride)."""
        sq, ss = self._strides
        return self.q.data_ptr(), sq, self.scale.data_ptr(), ss

    @classmethod
    def empty(cls, rows, d, device="cuda"):
        """Room for `rows` rows, uninitialised."""
        kp = _up(d, BLOCK)
        return cls(torch.empty(rows, kp, dtype=torch.float8_e4m3fn, device=device),
                   torch.empty(rows, _up(kp // BLOCK, 4), dtype=torch.uint8, device=device), d)

    @classmethod
    def from_parts(cls, codes, scale):
        """Rows from codes [R, d] (float8_e4m3fn) and scale bytes [R, ceil(d / 128)], copied where they are
        not padded and aligned as rows are held."""
        if codes.dtype != torch.float8_e4m3fn or codes.dim() != 2:
            raise ValueError(f"codes must be a float8_e4m3fn matrix, got {codes.dtype} {list(codes.shape)}")
        R, d = codes.shape
        kp, sp = _up(d, BLOCK), _up(_up(d, BLOCK) // BLOCK, 4)
        if scale.shape != (R, kp // BLOCK):
            raise ValueError(f"codes {tuple(codes.shape)} need scales of shape {(R, kp // BLOCK)}, got {tuple(scale.shape)}")
        if kp != d or codes.stride(1) != 1 or codes.stride(0) % 16 or codes.data_ptr() % 16:
            padded = torch.zeros(R, kp, dtype=torch.uint8, device=codes.device)
            padded[:, :d] = codes.view(torch.uint8)
            codes = padded.view(torch.float8_e4m3fn)
        scales = torch.zeros(R, sp, dtype=scale.dtype, device=scale.device)
        scales[:, :kp // BLOCK] = scale
        return cls(codes, scales, d)

    @property
    def shape(self):
        return torch.Size((self.q.shape[0], self.d))

    @property
    def device(self):
        return self.q.device

    @property
    def nbytes(self):
        return self.q.nbytes + self.scale.nbytes

    def __len__(self):
        return self.q.shape[0]

    def __getitem__(self, rows):
        if not isinstance(rows, slice):
            raise TypeError("8-bit rows are sliced; dequantize_rows takes row ids")
        return Fp8Rows(self.q[rows], self.scale[rows], self.d)

    def to(self, device, non_blocking=False):
        return Fp8Rows(self.q.to(device, non_blocking=non_blocking), self.scale.to(device, non_blocking=non_blocking), self.d)

    def __repr__(self):
        return f"Fp8Rows({len(self)} x {self.d}, {self.device})"


def _shift(t, n, name):
    return None if t is None else _vector(t, n, name)


def _device(first, *named):
    """first's device, which the other tensors (or None) have to share; require_gpu's errors."""
    dev = first.device
    if dev.type == "cuda":
        for _, t in named:
            if t is not None and t.device != dev:
                break
        else:
            return dev
    return _lib.require_gpu(("rows", first), *named)


def quantize_rows(x, *, shift=None, out=None, row0=0):
    """x [M, d] in fp32, bf16 or fp16 (any strides; a transposed matrix is read along its own rows) as
    8-bit rows, minus `shift` [d] if given (the difference in fp32).

    out: Fp8Rows to write into, rows (row0 + m) % len(out); a new Fp8Rows of M rows if None.
    """
    if x.dim() != 2:
        raise ValueError(f"x must have two dimensions, got {list(x.shape)}")
    M, d = x.shape
    if d < 1:
        raise ValueError("rows of no elements have no 8-bit form")
    shift = _shift(shift, d, "shift")
    if out is None:
        if row0:
            raise ValueError("row0 is a row of `out`, which is not given")
        out = Fp8Rows.empty(M, d, _device(x))
    elif out.d != d:
        raise ValueError(f"out holds rows of {out.d}, x has {d}")
    dev = _device(x, ("out", out.q), ("shift", shift))
    if M == 0:
        return out
    sxm, sxk = x.stride()
    with _lib.device(dev):
        rc = _lib.load().sf_quantize_rows(
            x.data_ptr(), sxm, sxk, _lib.dtype_code(x, "x"), None if shift is None else shift.data_ptr(),
            0 if shift is None else _lib.dtype_code(shift, "shift"), M, d, *out._args(), row0, out.q.shape[0],
            _lib.stream(dev))
    if rc:
        _lib.check(rc)
    return out


def dequantize_rows(rows8, rows=None, *, row0=0, count=None, shift=None, out_dtype=torch.bfloat16):
    """Rows read back, plus `shift` [d] if given (the sum in fp32, then rounded to out_dtype): those with
    the ids `rows` (int64, in any order; an id outside the store gives zeros), or `count` rows from row0 on,
    going on at row 0 behind the last (all of them by default)."""
    return read_rows(rows8, rows8.q.shape[0], rows, row0, count, shift, out_dtype)


def read_rows(rows8, R, rows, row0, count, shift, out_dtype):
    """dequantize_rows of a store of which only the first R rows have been written."""
    d = rows8.d
    if rows is not None:
        if rows.dtype != torch.int64 or rows.dim() != 1:
            raise ValueError(f"rows must be a one-dimensional int64 tensor, got {rows.dtype} {list(rows.shape)}")
        if row0 or count is not None:
            raise ValueError("rows are named by ids or by row0 and count, not by both")
        rows = rows.contiguous()
        M, ids = rows.shape[0], rows.data_ptr()
    else:
        M, ids = R if count is None else count, None
        if M < 0 or M > R:
            raise ValueError(f"count must lie in [0, {R}], got {M}")
    at, code = None, 0
    if shift is not None:
        shift = _vector(shift, d, "shift")
        at, code = shift.data_ptr(), _lib.dtype_code(shift, "shift")
    dev = _device(rows8.q, ("rows", rows), ("shift", shift))
    out = torch.empty((M, d), dtype=out_dtype, device=dev)
    out_code = _lib.dtype_code(out, "out_dtype")
    if M == 0:
        return out
    if R == 0:  # no id has a row
        return out.zero_()
    with _lib.device(dev):
        rc = _lib.load().sf_dequantize_rows(*rows8._args(), R, ids, row0, at, code, M, d, out.data_ptr(), d, out_code,
                                            _lib.stream(dev))
    if rc:
        _lib.check(rc)
    return out


def fused_encode_fp8(x, W, b_enc=None, threshold=None, activation="relu", *, b_dec=None, out_dtype=None, row_nnz=None):
    """fused_encode on 8-bit rows: act(x W^T + b_enc) [M, d_sae] on the matrix cores.

    float32 results are as good as fp32 sums (16-bit matrix instruction). bfloat16 and float16 results take the
    8-bit one, at twice the rate, which sums in fp32 but drops, of each eight products, what lies below 2^-13 of
    the largest: at most 7 * 2^-13 of sum |x w|, 5.5e-5 of the result in the root mean square for normal operands.

    x: Fp8Rows [M, d_in], or tokens [M, d_in] in fp32, bf16 or fp16, which are quantised on the way
      (minus `b_dec` if given).
    W: Fp8Rows [d_sae, d_in], a row a feature (quantize_rows(W_enc.T)).
    activation: "relu", "none", or "jumprelu" with a per-feature `threshold` [d_sae].
    out_dtype: x's own, bfloat16 for Fp8Rows. row_nnz: as in fused_encode; not with "none".
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"fused_encode_fp8 supports {list(ACTIVATIONS)}, got {activation!r}")
    if activation == "jumprelu" and threshold is None:
        raise ValueError("jumprelu needs a threshold")
    if activation == "none" and row_nnz is not None:
        raise ValueError("row counts need relu or jumprelu")
    held = isinstance(x, Fp8Rows)
    if not isinstance(W, Fp8Rows):
        raise ValueError("W must be Fp8Rows, a row a feature: quantize_rows(W_enc.T)")
    if held and b_dec is not None:
        raise ValueError("b_dec is subtracted before tokens are quantised; 8-bit rows are taken as they are")
    if not held and x.dim() != 2:
        raise ValueError(f"x must have two dimensions, got {list(x.shape)}")
    (M, d), N, d_w = x.shape, W.q.shape[0], W.d
    if d != d_w:
        raise ValueError(f"x has d_in={d} but W has d_in={d_w}")
    if out_dtype is None:
        out_dtype = torch.bfloat16 if held else x.dtype
    dev = _device(x.q if held else x, ("W", W.q), ("b_enc", b_enc), ("b_dec", b_dec), ("threshold", threshold),
                  ("row_nnz", row_nnz))
    b_enc, b_dec = _shift(b_enc, N, "b_enc"), _shift(b_dec, d, "b_dec")
    threshold = _vector(threshold, N, "threshold") if activation == "jumprelu" else None
    if row_nnz is not None:
        if row_nnz.dtype != torch.int32 or row_nnz.dim() != 1 or row_nnz.numel() != M or not row_nnz.is_contiguous():
            raise ValueError(f"row_nnz must be a contiguous int32 tensor of shape [{M}]")
    out = torch.empty((M, N), dtype=out_dtype, device=dev)
    code = _lib.dtype_code(out, "out_dtype")
    if M == 0 or N == 0:
        return out
    lib = _lib.load()
    tail = (*W._args(), _lib.ptr(b_enc), 0 if b_enc is None else _lib.dtype_code(b_enc, "b_enc"), _lib.ptr(threshold),
            0 if threshold is None else _lib.dtype_code(threshold, "threshold"), out.data_ptr(), N, code,
            _lib.ptr(row_nnz), M, N, d, ACTIVATIONS[activation])
    with _lib.device(dev):
        ws = torch.empty(_lib.fp8_workspace_bytes(0 if held else M, d), dtype=torch.uint8, device=dev)
        if held:
            _lib.check(lib.sf_encode_fp8_rows(*x._args(), *tail, ws.data_ptr(), ws.numel(), _lib.stream(dev)))
        else:
            x_code = _lib.dtype_code(x, "x")
            _lib.check(lib.sf_encode_fp8(x.data_ptr(), x.stride(0), x.stride(1), x_code, _lib.ptr(b_dec),
                                         0 if b_dec is None else _lib.dtype_code(b_dec, "b_dec"), *tail, ws.data_ptr(),
                                         ws.numel(), _lib.stream(dev)))
    return out
