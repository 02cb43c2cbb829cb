"""A dictionary and an activation cache in 8 bits (kernels/fp8.py; no reference counterpart).

ActivationBuffer holds activations in HBM at one byte an element, for training on shuffled rows or
for encoding what a model has produced: twice the rows of a 16-bit cache. Fp8Encoder applies a
trained SAE's encoder on the 8-bit matrix cores, to tokens or to the buffer's rows as they lie.

    buf = ActivationBuffer(1 << 21, sae.W_enc.shape[0], center=sae.b_dec)
    buf.write(acts)                               # as the model produces them
    x = buf.read(torch.randint(len(buf), (8192,), device="cuda"))     # a training batch

    enc = Fp8Encoder.from_sae(sae)
    csr = enc.encode_sparse(x)                    # tokens in hand
    csr = enc.encode_sparse(buf.rows(0, 4096))    # rows of the buffer
    x_hat = saeflow_amd.decode_sparse(sae, csr)
"""

import torch

from . import _lib
from .kernels import dense_to_csr, fixed_width_to_dense, layer_norm, topk_rows
from .kernels.fp8 import Fp8Rows, _vector, dequantize_rows, fused_encode_fp8, quantize_rows, read_rows
from .ops import INPUT_NORMS, input_norm, norm_eps
from .sae import ACTIVATIONS


class ActivationBuffer:
    """A ring of `rows` activations [d] in 8 bits on the GPU, written in order and read in any.

    center: optional [d] (a dictionary's b_dec, or the activations' mean); the buffer holds x - center,
    which spends the codes on what differs between tokens, and adds it back on reading.
    normed: whether what is written has been through a dictionary's input norm; its rows say so to an Fp8Encoder.
    len(buffer) is the number of rows written so far, at most `rows`.
    """

    def __init__(self, rows, d, *, center=None, device="cuda", normed=False):
        if rows < 1 or d < 1:
            raise ValueError(f"a buffer needs rows and a width, got {rows} x {d}")
        self.center = None if center is None else _vector(center.detach(), d, "center").clone()
        self.store = Fp8Rows.empty(rows, d, device, normed=bool(normed))
        self._device = _lib.require_gpu(("the buffer", self.store.q), ("center", self.center))
        self._next, self._filled = 0, 0

    @property
    def capacity(self):
        return len(self.store)

    @property
    def d(self):
        return self.store.d

    def __len__(self):
        return self._filled

    def write(self, x):
        """Appends x [M, d], M <= capacity, over the oldest rows once the ring is full. Returns (first
        row, M), which read takes. Not while a graph is captured: the ring's place is kept on the host."""
        M = x.shape[0]
        if M > self.capacity:
            raise ValueError(f"{M} rows do not fit a buffer of {self.capacity}")
        with _lib.device(self._device):
            # (replays would write the same rows over and over, and rows only captured would count as written)
            if torch._C._cuda_isCurrentStreamCapturing():
                raise RuntimeError("ActivationBuffer.write cannot be captured in a graph; quantize_rows(out=, row0=) "
                                   "writes to fixed rows")
        at = self._next
        quantize_rows(x, shift=self.center, out=self.store, row0=at)
        self._next = (at + M) % self.capacity
        # in order from row 0 on, so the written rows are the first ones until the ring is full
        self._filled = min(self._filled + M, self.capacity)
        return at, M

    def read(self, rows=None, *, out_dtype=torch.bfloat16):
        """Rows as out_dtype [n, d]: those of an int64 tensor of ids on the GPU (which are not checked: one
        that no row has been written to reads as zeros), of a pair as write returns it, or, by default, all written.
        Captured in a graph, a read knows the rows that were written by then."""
        if torch.is_tensor(rows):
            return read_rows(self.store, self._filled, rows, 0, None, self.center, out_dtype)
        R, filled = self.capacity, self._filled
        row0, count = (0, filled) if rows is None else rows
        if count < 0 or not 0 <= row0 < R or count > filled or (row0 + count > filled < R):
            raise ValueError(f"{count} rows from {row0} on are not among the {filled} written")
        return read_rows(self.store, R, None, row0, count, self.center, out_dtype)

    def rows(self, start, stop):
        """Written rows [start, stop) as they lie (a view): what Fp8Encoder and fused_encode_fp8 take."""
        if not 0 <= start <= stop <= len(self):
            raise ValueError(f"rows [{start}, {stop}) are not among the {len(self)} written")
        return self.store[start:stop]


class Fp8Encoder:
    """A trained SAE's encoder with its dictionary in 8 bits, in the form in which it is applied; its
    parameters are copied, so it is made again when they change.

    Tokens are quantised minus b_dec, in blocks of 128, on the way into the product. 8-bit rows (an
    ActivationBuffer's) are taken as they are: they hold x - center, `center` by default b_dec.
    input_norm="layer_norm": tokens are normed first, as the SAE's are. 8-bit rows hold normed tokens then: those of a buffer or
    a cache that were not normed are refused.
    """

    def __init__(self, W_enc, b_enc, b_dec, threshold=None, activation="relu", k=None, *, center=None, input_norm=None,
                 norm_eps=1e-5):
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {ACTIVATIONS}, got {activation!r}")
        if activation == "jumprelu" and threshold is None:
            raise ValueError("jumprelu needs a threshold")
        if activation == "topk" and not k:
            raise ValueError("topk activation needs k")
        if input_norm not in INPUT_NORMS:
            raise ValueError(f"input_norm must be one of {INPUT_NORMS}, got {input_norm!r}")
        self.input_norm, self.norm_eps = input_norm, norm_eps
        d_in, d_sae = W_enc.shape
        self.activation, self.k = activation, k
        self.b_enc = _vector(b_enc.detach(), d_sae, "b_enc").clone()
        self.b_dec = _vector(b_dec.detach(), d_in, "b_dec").clone()
        self.threshold = None if activation != "jumprelu" else _vector(threshold.detach(), d_sae, "threshold").clone()
        self.W = quantize_rows(W_enc.detach().T)
        self.rows_bias = self.b_enc
        if center is not None:
            self.rows_bias = self._moved_bias(_vector(center.detach(), d_in, "center"))

    @classmethod
    def from_sae(cls, sae, *, center=None):
        """Of a saeflow_amd.SAE, or anything with its attributes."""
        return cls(sae.W_enc, sae.b_enc, sae.b_dec, sae.threshold, sae.activation, sae.k, center=center,
                   input_norm=input_norm(sae), norm_eps=norm_eps(sae))

    def _moved_bias(self, center):
        """b_enc + W (center - b_dec) in fp32, W as it is held: the bias for rows that hold x - center."""
        N, d = self.W.shape
        by = center.float() - self.b_dec.float()
        out = self.b_enc.float().clone()
        lib, dev = _lib.load(), _lib.require_gpu(("W_enc", self.W.q), ("center", by))
        step = max(1, (1 << 28) // d)
        with _lib.device(dev):
            for n in range(0, N, step):
                part = dequantize_rows(self.W[n:n + step], out_dtype=torch.float32)
                ws = torch.empty(len(part) * min(256, d), dtype=torch.float32, device=dev)
                _lib.check(lib.sf_matvec(part.data_ptr(), len(part), d, d, 1, _lib.DTYPE[torch.float32], by.data_ptr(),
                                         1.0, 1, out[n:].data_ptr(), ws.data_ptr(), ws.numel(), _lib.stream(dev)))
        return out

    def _features(self, x, activation, row_nnz=None, out_dtype=None):
        if isinstance(x, Fp8Rows):
            if self.input_norm is not None and x.normed is False:
                raise ValueError("the encoder norms its tokens, and these 8-bit rows hold tokens that were not normed: pass them "
                                 "read back, or, if they were, say normed=True to the ActivationBuffer or iter_batches")
            return fused_encode_fp8(x, self.W, self.rows_bias, self.threshold, activation, out_dtype=out_dtype,
                                    row_nnz=row_nnz)
        if self.input_norm is not None:
            x = layer_norm(x, eps=self.norm_eps)[0]
        return fused_encode_fp8(x, self.W, self.b_enc, self.threshold, activation, b_dec=self.b_dec,
                                out_dtype=out_dtype, row_nnz=row_nnz)

    def encode(self, x, *, out_dtype=None):
        """The features of every token, or 8-bit row, as a dense [M, d_sae] tensor (x's type; bfloat16 for
        8-bit rows)."""
        if self.activation == "topk":
            values, indices = topk_rows(self._features(x, "relu", out_dtype=out_dtype), self.k)
            return fixed_width_to_dense(indices, values, self.W.shape[0])
        return self._features(x, self.activation, out_dtype=out_dtype)

    def encode_sparse(self, x, *, out_dtype=None):
        """The same in the CSR contract, as saeflow_amd.encode_sparse gives it."""
        M = x.shape[0]
        if self.activation == "topk":
            values, indices = topk_rows(self._features(x, "relu", out_dtype=out_dtype), self.k)
            indptr = torch.arange(0, M * self.k + 1, self.k, device=x.device, dtype=torch.int64)
            return indptr, indices.flatten(), values.flatten()
        row_nnz = torch.zeros(M, device=x.device, dtype=torch.int32)
        return dense_to_csr(self._features(x, self.activation, row_nnz, out_dtype), row_nnz)
