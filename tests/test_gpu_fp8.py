"""8-bit rows on the GPU: codes, scales and values bit for bit against the definition in 64 bits; the
product exactly where its sums are exact in fp32, and within a bound derived from fp32 sums elsewhere."""

import numpy as np
import pytest
import torch

import saeflow_amd
from oracle import fp8 as ofp8
from oracle import reference as oref
from saeflow_amd.kernels import (Fp8Rows, csr_to_dense, dense_to_csr, dequantize_rows, fused_encode,
                                 fused_encode_fp8, quantize_rows, topk_rows)

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def wide(M, d, dtype, seed=0):
    """Elements over many binades: blocks of very different size, small elements beside large ones."""
    g = torch.Generator().manual_seed(seed)
    lo, hi = (-9, 8) if dtype == F16 else (-40, 40)
    x = torch.randn(M, d, generator=g) * 2.0 ** torch.empty(M, d).uniform_(-12, 0, generator=g)
    nb = -(-d // 128)
    block = 2.0 ** torch.randint(lo, hi, (M, nb), generator=g).float().repeat_interleave(128, 1)[:, :d]
    return (x * block).to(dtype)


def code_values(rows8):
    """Values of the codes before scaling, and the scale bytes, on the host, padding left out."""
    nb = -(-rows8.d // 128)
    return (ofp8.CODES[rows8.q.view(torch.uint8).cpu().numpy()][:, :rows8.d], rows8.scale.cpu().numpy()[:, :nb])


def check_rows(rows8, v):
    """rows8 holds exactly what the definition gives for the fp32 rows v, and zeros behind them."""
    want, byte = ofp8.quantize(v.cpu().numpy())
    got, scale = code_values(rows8)
    np.testing.assert_array_equal(scale, byte)
    np.testing.assert_array_equal(got, want)
    assert not rows8.q.view(torch.uint8)[:, rows8.d:].any() and not rows8.scale[:, byte.shape[1]:].any()


def layouts(x):
    """x in memory in several ways: itself, its transpose's, every second element, off 16 B, one element apart."""
    M, d = x.shape
    yield "rows", x.cuda()
    yield "columns", x.T.contiguous().cuda().T
    wide_ = torch.full((M, 2 * d + 6), 7.0, dtype=x.dtype, device="cuda")
    wide_[:, 0:2 * d:2] = x.cuda()
    yield "strided", wide_[:, 0:2 * d:2]
    off = torch.full((M, d + 3), 7.0, dtype=x.dtype, device="cuda")
    off[:, 1:d + 1] = x.cuda()
    yield "off 16 B", off[:, 1:d + 1]
    cols = torch.full((d, M + 5), 7.0, dtype=x.dtype, device="cuda")
    cols[:, 1:M + 1] = x.T.cuda()
    yield "columns off 16 B", cols[:, 1:M + 1].T


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,d", [(1, 1), (3, 127), (17, 128), (64, 129), (130, 768), (65, 1000), (5, 2304)])
def test_codes_and_scales_are_those_of_the_definition(dtype, M, d):
    x = wide(M, d, dtype, seed=M + d)
    for name, t in layouts(x):
        check_rows(quantize_rows(t), x.float())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("c_dtype", [F32, BF16, F16])
def test_the_shift_is_subtracted_in_fp32(dtype, c_dtype):
    x = torch.randn(20, 300).to(dtype)
    c = torch.randn(304).to(c_dtype)[3:303]  # (off 16 B)
    for shift in (c, c.clone()):
        for name, t in layouts(x):
            check_rows(quantize_rows(t, shift=shift.cuda()), x.float() - c.float())


def test_edges_of_the_scale_and_of_the_codes():
    rows = [torch.zeros(128)]
    for e in (-149, -140, -128, -127, -126, -120, -8, 0, 100):
        top = torch.tensor(448.0).double() * 2.0 ** e
        for a in (top, top * (1 + 2.0 ** -20), top * (1 - 2.0 ** -20), top / 2):
            r = torch.linspace(-1, 1, 128).double() * a
            rows.append(r.float())
    rows.append(torch.full((128,), torch.finfo(F32).max))
    rows.append(torch.tensor([2.0 ** -149] * 127 + [-0.0]))
    # every midpoint between neighbouring codes, and just beside it (the block's scale is 1)
    codes = np.unique(ofp8.CODES[np.isfinite(ofp8.CODES)])
    mid = torch.from_numpy((codes[1:] + codes[:-1]) / 2).float()
    for m in (mid, torch.nextafter(mid, torch.tensor(1e9)), torch.nextafter(mid, torch.tensor(-1e9))):
        for part in m.split(127):
            r = torch.zeros(128)
            r[0], r[1:1 + len(part)] = 448.0, part
            rows.append(r)
    x = torch.stack(rows)
    check_rows(quantize_rows(x.cuda()), x)
    check_rows(quantize_rows(x.T.contiguous().cuda().T), x)


def test_nan_and_infinities_become_nan_and_leave_the_scale_alone():
    x = torch.randn(6, 260)
    x[0, 3], x[1, 200], x[2, 259], x[3, :128] = float("nan"), float("inf"), float("-inf"), float("nan")
    x[4, :] = float("inf")
    for t in (x.cuda(), x.T.contiguous().cuda().T, x.to(BF16).cuda()):
        check_rows(quantize_rows(t), t.cpu().float())
    back = dequantize_rows(quantize_rows(x.cuda()), out_dtype=F32).cpu()
    assert torch.equal(back.isnan(), ~x.isfinite())


@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d", [1, 64, 129, 768, 1000, 1001])
def test_reading_back_is_exact(out_dtype, d):
    x = wide(50, d, F16, seed=d)
    c = torch.randn(d).to(BF16)
    rows8 = quantize_rows(x.cuda())
    v = torch.from_numpy(ofp8.values(rows8.q.view(torch.uint8).cpu().numpy()[:, :d],
                                     rows8.scale.cpu().numpy()[:, :-(-d // 128)])).float()
    assert torch.equal(dequantize_rows(rows8, out_dtype=out_dtype).cpu(), v.to(out_dtype))
    ids = torch.tensor([49, 0, 7, 7, 50, -1, 1 << 40, 3])
    want = (v[ids.clamp(0, 49)] + c.float())
    want[[4, 5, 6]] = 0
    got = dequantize_rows(rows8, ids.cuda(), shift=c.cuda(), out_dtype=out_dtype)
    assert torch.equal(got.cpu(), want.to(out_dtype))
    got = dequantize_rows(rows8, row0=45, count=11, shift=c.cuda().to(out_dtype), out_dtype=out_dtype)
    want = v[torch.arange(45, 56) % 50] + c.to(out_dtype).float()
    assert torch.equal(got.cpu(), want.to(out_dtype))


def test_every_code_and_every_scale_reads_back():
    codes = torch.arange(256, dtype=torch.uint8)[None].repeat(255, 1)
    scale = torch.arange(255, dtype=torch.uint8)[:, None].repeat(1, 2)
    rows8 = Fp8Rows.from_parts(codes.view(torch.float8_e4m3fn).cuda(), scale.cuda())
    want = torch.from_numpy(ofp8.values(codes.numpy(), scale.numpy())).float()  # (overflows to infinity at the top)
    got = dequantize_rows(rows8, out_dtype=F32).cpu()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(0.0, 1e39, -1e39), want.nan_to_num(0.0, 1e39, -1e39))


def test_rows_behind_four_gigabytes():
    R, d = (1 << 25) + 40, 128  # 4.3 GB of codes
    store = Fp8Rows.empty(R, d)
    x = wide(100, d, BF16)
    quantize_rows(x.cuda(), out=store, row0=R - 60)  # 60 rows at the end, 40 from row 0 on
    ids = (torch.arange(100) + R - 60) % R
    tail = store[R - 60:]
    check_rows(tail, x[:60].float())
    check_rows(store[:40], x[60:].float())
    want = dequantize_rows(quantize_rows(x.cuda()), out_dtype=F32)
    assert torch.equal(dequantize_rows(store, ids.cuda(), out_dtype=F32), want)
    assert torch.equal(dequantize_rows(store, row0=R - 60, count=100, out_dtype=F32), want)
    W = quantize_rows(torch.randn(96, d, device="cuda"))
    assert torch.equal(fused_encode_fp8(tail, W, out_dtype=F32),
                       fused_encode_fp8(quantize_rows(x[:60].cuda()), W, out_dtype=F32))


# ----------------------------------------------------------------------------- product
def whole(R, d, seed, top=3):
    """Rows of codes that are whole numbers up to `top`, scales 1/2 or 1: products are multiples of 1/4 and
    sums of up to 2^22 / top^2 of them exact in fp32, in any order. (rows, their values in 64 bits)"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    v = torch.randint(-top, top + 1, (R, d), generator=g, device="cuda").float()
    scale = torch.randint(126, 128, (R, -(-d // 128)), generator=g, device="cuda", dtype=torch.uint8)
    two = torch.exp2(scale.double() - 127).repeat_interleave(128, 1)[:, :d]
    return Fp8Rows.from_parts(v.to(torch.float8_e4m3fn), scale), v.double() * two


# few tokens and many, panels cut short, blocks cut short, more blocks than LDS holds scales for, odd d_sae
SHAPES = [(1, 64, 128), (1, 257, 2304), (7, 1000, 129), (32, 4099, 768), (33, 130, 4096), (100, 777, 1000),
          (137, 2048, 1), (128, 512, 4224), (250, 1001, 8320), (1000, 10007, 256), (16, 100, 8448), (515, 65536, 300),
          (2048, 16384, 130), (2000, 16391, 127), (4099, 8200, 4352), (200, 12291, 2304), (250, 12288, 4352)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_is_exact_where_sums_are(M, N, K):
    x, xv = whole(M, K, 1)
    W, wv = whole(N, K, 2)
    b = torch.randint(-50, 50, (N,), device="cuda").float()
    want = (xv @ wv.T.contiguous() + b.double()).float()
    assert torch.equal(fused_encode_fp8(x, W, b, activation="none", out_dtype=F32), want)
    for dtype in (BF16, F16):
        nnz = torch.zeros(M, dtype=torch.int32, device="cuda")
        f = fused_encode_fp8(x, W, b.to(BF16), out_dtype=dtype, row_nnz=nnz)
        assert torch.equal(f, want.clamp(min=0).to(dtype))
        assert torch.equal(nnz, (f != 0).sum(1, dtype=torch.int32))
    thr = torch.randint(0, 30, (N,), device="cuda").to(F16)
    f = fused_encode_fp8(x, W, b, thr, "jumprelu")
    assert f.dtype == BF16 and torch.equal(f, torch.where(want > thr.float(), want, 0.0).to(BF16))


@pytest.mark.parametrize("M,N,K", [(1, 1000, 2304), (60, 3000, 1000), (300, 4099, 768), (2100, 16384, 2304)])
def test_product_of_ordinary_rows(M, N, K):
    """Sums of K terms in fp32, each addition off by at most one unit in the last place (2^-23, whichever
    way the matrix cores round) of what it adds to: K * 2^-23 * sum |x w|; for 16-bit results, seven of
    each eight products lose at most 2^-13 of the largest: 7 * 2^-13 * sum |x w|; then one rounding to
    the output."""
    x = quantize_rows(torch.randn(M, K, device="cuda") * torch.exp(torch.randn(K, device="cuda")))
    W = quantize_rows(torch.randn(N, K, device="cuda") / K ** 0.5)
    xv, wv = (dequantize_rows(r, out_dtype=F32).double() for r in (x, W))
    want, size = xv @ wv.T.contiguous(), xv.abs() @ wv.abs().T.contiguous()
    for dtype, u in ((F32, 0.0), (BF16, 2.0 ** -8), (F16, 2.0 ** -11)):
        got = fused_encode_fp8(x, W, activation="none", out_dtype=dtype).double()
        err = (got - want).abs()
        sums = (K + 1) * 2.0 ** -23 + (7 * 2.0 ** -13 if u else 0.0)
        assert (err <= sums * size * (1 + u) + u * want.abs() + 2.0 ** -24).all()


def test_scales_of_every_block_and_size_reach_the_product():
    """Rows with one nonzero element each: the product is that element pair's, whatever the scales."""
    K, n = 4 * 128 + 60, 255
    x, W = torch.zeros(n, K), torch.zeros(n, K)
    byte = torch.arange(n)
    at = torch.arange(n) * 7 % K
    for r in range(n):
        x[r, at[r]] = 1.5
        W[r, at[r]] = -2.0
    ex = torch.where(byte % 2 == 0, byte % 100 - 40, 3 - byte % 90)
    x = x * 2.0 ** ex[:, None]
    W = W * 2.0 ** (-ex // 2)[:, None]
    want = x.double() @ W.double().T
    got = fused_encode_fp8(quantize_rows(x.cuda()), quantize_rows(W.cuda()), activation="none", out_dtype=F32)
    assert torch.equal(got.cpu().double(), want)


@pytest.mark.parametrize("out_dtype", [F32, BF16])
def test_smallest_and_largest_scales_in_the_product(out_dtype):
    """Blocks at 2^-119 and below (scale bytes 0 to 8) against features of 2^100, and the other way round."""
    g = torch.Generator().manual_seed(3)
    x = torch.randint(1, 4, (30, 128), generator=g).float() * 2.0 ** torch.randint(-119, -110, (30, 1), generator=g)
    W = torch.randint(1, 4, (70, 128), generator=g).float() * 2.0 ** torch.randint(90, 110, (70, 1), generator=g)
    want = x.double() @ W.double().T
    for a, b, w in ((x, W, want), (W, x, want.T)):
        got = fused_encode_fp8(quantize_rows(a.cuda()), quantize_rows(b.cuda()), activation="none", out_dtype=out_dtype)
        assert torch.equal(got.cpu(), w.to(F32).to(out_dtype))


def test_product_past_four_gigabytes():
    """Operands and results whose offsets pass 32 bits, through narrow and wide tiles."""
    R, d = (1 << 25) + 40, 128
    W = Fp8Rows.empty(R, d)  # 4.3 GB of codes
    W.q.view(torch.uint8).zero_()
    W.scale.fill_(127)
    tail, tv = whole(300, d, 5)
    W.q[R - 300:].view(torch.uint8).copy_(tail.q.view(torch.uint8))
    W.scale[R - 300:] = tail.scale
    x, xv = whole(300, d, 6)
    want = (xv @ tv.T.contiguous()).float()
    for M, dtype in ((1, BF16), (33, F32)):
        got = fused_encode_fp8(x[:M], W, activation="none", out_dtype=dtype)
        assert torch.equal(got[:, R - 300:], want[:M].to(dtype)) and not got[:, R - 900:R - 300].any()
        del got
    sparse = Fp8Rows(W.q.view(R // 8, 8 * 128)[:, :128], W.scale.view(R // 8, 32)[:, :4], d)  # rows 1 KB apart
    wide_rows = Fp8Rows(sparse.q[::16], sparse.scale[::16], d)  # and 16 KB
    n = len(wide_rows)
    wide_rows.q[n - 300:].view(torch.uint8).copy_(tail.q.view(torch.uint8))
    wide_rows.scale[n - 300:] = tail.scale
    for M in (1, 40, 100, 300):
        for dtype in (BF16, F32):
            got = fused_encode_fp8(x[:M], wide_rows, activation="none", out_dtype=dtype)
            assert torch.equal(got[:, n - 300:], want[:M].to(dtype))
            got = fused_encode_fp8(wide_rows[n - 300:], x[:M], activation="none", out_dtype=dtype)
            assert torch.equal(got, want[:M].T.to(dtype))
    del W, sparse, wide_rows, got
    x, xv = whole(9000, d, 7)
    W, wv = whole(131072, d, 8)  # 4.7 GB of fp32 results, 2.4 GB of bf16
    for dtype in (F32, BF16):
        got = fused_encode_fp8(x, W, activation="none", out_dtype=dtype)
        for m in (0, 4000, 8900):
            assert torch.equal(got[m:m + 100], (xv[m:m + 100] @ wv.T.contiguous()).to(dtype))


@pytest.mark.parametrize("M,N,out_dtype", [(16384, 16391, BF16), (16384, 16416, F16), (16384, 16384, BF16),
                                           (4096, 12936, BF16), (4096, 12921, F16), (2048, 12921, F32),
                                           (2048, 12928, F32), (300, 24640, F16), (300, 24600, BF16)])
def test_results_of_rows_on_and_off_whole_lines(M, N, out_dtype):
    """Rows that begin on cache lines and rows that do not, few bytes and many: small whole numbers, whose sums
    (at most 9 * 130) are exact in fp32 and rounded once."""
    g = torch.Generator(device="cuda").manual_seed(M + N)
    x = torch.randint(-3, 4, (M, 130), generator=g, device="cuda").float()
    W = torch.randint(-3, 4, (N, 130), generator=g, device="cuda").float()
    got = fused_encode_fp8(quantize_rows(x), quantize_rows(W), activation="none", out_dtype=out_dtype)
    assert torch.equal(got, (x @ W.T.contiguous()).to(out_dtype))


def test_one_row_of_any_stride():
    """A lone row's stride addresses nothing."""
    W, wv = whole(70, 256, 9)
    x, xv = whole(3, 256, 10)
    one = Fp8Rows(x.q.view(torch.uint8)[1].as_strided((1, 256), (1, 1)).view(torch.float8_e4m3fn),
                  x.scale[1].as_strided((1, 4), (3, 1)), 256)
    want = (xv[1:2] @ wv.T.contiguous()).float()
    assert torch.equal(fused_encode_fp8(one, W, activation="none", out_dtype=F32), want)
    assert torch.equal(dequantize_rows(one, out_dtype=F32).double(), xv[1:2])
    # codes that lie off 16 B are laid out anew
    codes = torch.zeros(3, 300, dtype=torch.uint8, device="cuda")
    codes[:, 7:263] = x.q.view(torch.uint8)
    moved = Fp8Rows.from_parts(codes[:, 7:263].view(torch.float8_e4m3fn), x.scale[:, :2])
    assert torch.equal(fused_encode_fp8(moved, W, activation="none", out_dtype=F32), (xv @ wv.T.contiguous()).float())


@pytest.mark.parametrize("M", [5, 300, 2048])
def test_biases_up_to_the_largest_and_with_every_bit(M):
    """A zero product plus a bias is the bias, whole, in fp32, at the largest finite and the smallest normal
    magnitudes too."""
    N = 16384
    x, W = quantize_rows(torch.zeros(M, 200, device="cuda")), quantize_rows(torch.zeros(N, 200, device="cuda"))
    g = torch.Generator().manual_seed(4)
    b = (torch.rand(N, generator=g) + 1) * 2.0 ** torch.randint(-100, 127, (N,), generator=g) * torch.randn(N, generator=g).sign()
    b[:4] = torch.tensor([torch.finfo(F32).max, -torch.finfo(F32).max, 0.0, float("inf")])
    b = b.cuda()
    got = fused_encode_fp8(x, W, b, activation="none", out_dtype=F32)
    assert torch.equal(got, b.expand(M, N))
    for dtype in (BF16, F16):
        assert torch.equal(fused_encode_fp8(x, W, b, activation="none", out_dtype=dtype), b.to(dtype).expand(M, N))


def test_fp32_results_are_as_good_as_fp32_sums():
    """Normal operands, K terms added one after the other in fp32: each of the K roundings is at most
    2^-24 of a partial sum no larger than a few standard deviations of the result, so the root mean
    square error is at most about sqrt(K) * 2^-24 of it; twice that for another rounding mode."""
    for M, N, K in ((1, 4096, 2304), (300, 2048, 768), (2048, 16384, 768)):
        x, W = quantize_rows(torch.randn(M, K, device="cuda")), quantize_rows(torch.randn(N, K, device="cuda"))
        want = dequantize_rows(x, out_dtype=F32).double() @ dequantize_rows(W, out_dtype=F32).double().T.contiguous()
        got = fused_encode_fp8(x, W, activation="none", out_dtype=F32).double()
        assert (got - want).norm() <= 2 * K ** 0.5 * 2.0 ** -24 * want.norm()


def test_nan_stays_in_its_row_and_padding_is_never_read():
    x, W = torch.randn(40, 200), torch.randn(300, 200)
    x[3, 190] = float("inf")
    W[7, 0] = float("nan")
    f = fused_encode_fp8(quantize_rows(x.cuda()), quantize_rows(W.cuda()), out_dtype=F32).cpu()
    bad = torch.zeros(40, 300, dtype=torch.bool)
    bad[3], bad[:, 7] = True, True
    assert torch.equal(f.isnan(), bad)
    # rows of a larger store, NaN all around them
    big = Fp8Rows.empty(50, 200)
    big.q.view(torch.uint8).fill_(0x7F)
    big.scale.fill_(200)
    quantize_rows(x[10:33].cuda(), out=big, row0=20)
    assert torch.equal(fused_encode_fp8(big[20:43], quantize_rows(W.cuda()), out_dtype=F32).cpu().nan_to_num(-1.0),
                       f[10:33].nan_to_num(-1.0))


@pytest.mark.parametrize("out_dtype", [F32, BF16])
def test_large_products_keep_nan_infinite_biases_and_thresholds(out_dtype):
    """The persistent tiles: NaN rows and features, biases that are infinite, NaN, tiny and huge, a NaN
    threshold (keeps nothing), counts; d_sae cuts the last tile."""
    x, xv = whole(2300, 640, 5)
    W, wv = whole(16200, 640, 6)
    x.q.view(torch.uint8)[77, 3] = 0x7F
    W.q.view(torch.uint8)[16199, 600] = 0xFF
    W.q.view(torch.uint8)[300, 0] = 0x7F
    xv[77], wv[16199], wv[300] = float("nan"), float("nan"), float("nan")
    b = torch.randint(-50, 50, (16200,), device="cuda").float()
    b[5], b[6], b[7], b[8], b[9] = float("inf"), float("-inf"), float("nan"), 1e-30, 3e38
    pre = (xv @ wv.T.contiguous()).float() + b
    pre[:, 9] = 3e38
    pre[77, 9] = float("nan")
    pre[:, 8] = (xv @ wv[8]).float() + torch.where(xv @ wv[8] == 0, 1e-30, 0.0).float()

    def same(got, want):
        return torch.equal(got.nan_to_num(-7.0, 1e38, -1e38), want.to(out_dtype).nan_to_num(-7.0, 1e38, -1e38))

    assert same(fused_encode_fp8(x, W, b, activation="none", out_dtype=out_dtype), pre)
    relu = torch.where(pre <= 0, 0.0, pre)
    assert same(fused_encode_fp8(x, W, b, out_dtype=out_dtype), relu)
    nnz = torch.zeros(2300, dtype=torch.int32, device="cuda")
    f = fused_encode_fp8(x, W, b, out_dtype=out_dtype, row_nnz=nnz)
    assert same(f, relu) and torch.equal(nnz, (f != 0).sum(1, dtype=torch.int32))
    thr = torch.randint(0, 30, (16200,), device="cuda").float()
    thr[100] = float("nan")
    want = torch.relu(pre) * (pre > thr)  # (a NaN stays one, whatever its threshold)
    nnz.zero_()
    f = fused_encode_fp8(x, W, b, thr, "jumprelu", out_dtype=out_dtype, row_nnz=nnz)
    assert same(f, want) and torch.equal(nnz, (f != 0).sum(1, dtype=torch.int32))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M", [0, 1, 5, 70, 300])
def test_tokens_are_quantised_on_the_way(dtype, M):
    x, b_dec = torch.randn(M, 500).to(dtype), torch.randn(500).to(dtype)
    W, b = quantize_rows(torch.randn(1000, 500, device="cuda")), torch.randn(1000, device="cuda")
    for name, t in layouts(x) if M else [("rows", x.cuda())]:
        got = fused_encode_fp8(t, W, b, b_dec=b_dec.cuda())
        want = fused_encode_fp8(quantize_rows(x.cuda(), shift=b_dec.cuda()), W, b, out_dtype=dtype)
        assert got.dtype == dtype and torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,d", [(1, 8), (3, 128), (8, 504), (1, 1000), (1, 2304), (4, 1024), (1, 4096), (2, 2300)])
def test_few_tokens_quantised_by_the_product_itself(dtype, M, d):
    x, W = wide(M, d, dtype, seed=d), quantize_rows(torch.randn(500, d, device="cuda"))
    x[0, d - 1] = float("nan") if M > 1 else 3.0
    b_dec = torch.randn(d + 1)
    for c in (None, b_dec[:d].to(dtype).cuda(), b_dec.to(dtype).cuda()[1:], b_dec[:d].to(F16 if dtype == BF16 else BF16).cuda()):
        rows8 = quantize_rows(x.cuda(), shift=c)
        for out_dtype in (F32, BF16):
            want = fused_encode_fp8(rows8, W, out_dtype=out_dtype)
            got = fused_encode_fp8(x.cuda(), W, b_dec=c, out_dtype=out_dtype)
            assert torch.equal(got.nan_to_num(-1.0), want.nan_to_num(-1.0))


def test_calls_repeat_bit_for_bit_on_another_stream_and_in_a_graph():
    x, W = torch.randn(90, 700, device="cuda"), quantize_rows(torch.randn(2000, 700, device="cuda"))
    want = fused_encode_fp8(x, W)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fused_encode_fp8(x, W)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph, inp = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        out = fused_encode_fp8(inp, W)
    for i in range(4):
        y = torch.randn(90, 700, device="cuda")
        inp.copy_(y)
        graph.replay()
        assert torch.equal(out, fused_encode_fp8(y, W))


# ----------------------------------------------------------------------------- encoder and buffer
def small_sae(activation, d_in=300, d_sae=2000, dtype=BF16):
    sae = saeflow_amd.SAE(d_in, d_sae, activation, k=16 if activation == "topk" else None, dtype=dtype, device="cuda")
    sae.b_enc.copy_(torch.randn(d_sae) * 0.1)
    sae.b_dec.copy_(torch.randn(d_in) * 0.5)
    if sae.threshold is not None:
        sae.threshold.copy_(torch.rand(d_sae) * 2)
    return sae


@pytest.mark.parametrize("activation", ["relu", "jumprelu", "topk"])
def test_encoder_dense_sparse_and_from_the_buffer(activation):
    sae = small_sae(activation)
    enc = saeflow_amd.Fp8Encoder.from_sae(sae)
    x = torch.randn(200, 300, device="cuda").to(BF16)
    f = enc.encode(x)
    act = "relu" if activation == "topk" else activation
    dense = fused_encode_fp8(x, quantize_rows(sae.W_enc.T), sae.b_enc, sae.threshold, act, b_dec=sae.b_dec)
    if activation == "topk":
        v, i = topk_rows(dense, 16)
        dense = torch.zeros_like(dense).scatter_(1, i.long(), v)
    assert torch.equal(f, dense)
    csr = enc.encode_sparse(x)
    assert torch.equal(csr_to_dense(*csr, 2000), f)
    assert saeflow_amd.decode_sparse(sae, csr).shape == x.shape
    buf = saeflow_amd.ActivationBuffer(256, 300, center=sae.b_dec)
    buf.write(x)
    assert torch.equal(enc.encode(buf.rows(0, 200)), f)
    assert torch.equal(enc.encode(buf.rows(50, 51)), f[50:51])
    got = enc.encode_sparse(buf.rows(0, 200))
    assert all(torch.equal(a, b) for a, b in zip(got, csr))


def test_encoder_is_near_the_unquantised_one():
    """Two operands rounded to within 2^-4 of themselves each, errors of zero mean: a product term is off by
    about sqrt(2) * 2^-4 / sqrt(3) (uniform) at most, so pre-activations of unit size by at most about 0.05."""
    sae = small_sae("relu", 2304, 4096)
    sae.b_enc.zero_()
    x = sae.b_dec + torch.randn(500, 2304, device="cuda").to(BF16)
    pre = oref.encode_pre(x.cpu(), sae.W_enc.cpu(), sae.b_enc.cpu(), sae.b_dec.cpu()).clamp(min=0)
    got = saeflow_amd.Fp8Encoder.from_sae(sae).encode(x, out_dtype=F32).cpu()
    assert (got - pre).pow(2).mean().sqrt() <= 0.05 * pre.pow(2).mean().sqrt() * 2 ** 0.5


@pytest.mark.parametrize("centered", [False, True])
def test_rows_with_another_center(centered):
    """x W + b with the center's share moved into the bias: the features of the values that the buffer
    holds, within fp32 sums (d_in terms) of both parts."""
    sae = small_sae("relu", dtype=F32)
    center = torch.randn(300, device="cuda") if centered else torch.zeros(300, device="cuda")
    buf = saeflow_amd.ActivationBuffer(64, 300, center=center if centered else None)
    x = torch.randn(64, 300, device="cuda")
    buf.write(x)
    enc = saeflow_amd.Fp8Encoder.from_sae(sae, center=center)
    W = dequantize_rows(enc.W, out_dtype=F32).double()
    held = dequantize_rows(buf.store, out_dtype=F32).double() + center.double() - sae.b_dec.double()
    want = held @ W.T.contiguous() + sae.b_enc.double()
    size = held.abs() @ W.abs().T.contiguous() + sae.b_enc.abs().double() + (center - sae.b_dec).abs().double() @ W.abs().T
    got = enc.encode(buf.rows(0, 64), out_dtype=F32).double()
    assert ((got - want.clamp(min=0)).abs() <= 3 * 302 * 2.0 ** -23 * size).all()


def test_buffer_wraps_and_knows_what_it_holds():
    buf = saeflow_amd.ActivationBuffer(100, 130)
    assert len(buf) == 0 and buf.capacity == 100 and buf.d == 130
    assert buf.read().shape == (0, 130)
    x = torch.randn(250, 130, device="cuda")
    held = dequantize_rows(quantize_rows(x), out_dtype=F32)
    assert buf.write(x[:70]) == (0, 70) and len(buf) == 70
    assert torch.equal(buf.read(out_dtype=F32), held[:70])
    with pytest.raises(ValueError):
        buf.read((60, 11))
    with pytest.raises(ValueError):
        buf.rows(0, 71)
    at = buf.write(x[70:130])
    assert at == (70, 60) and len(buf) == 100
    assert torch.equal(buf.read(at, out_dtype=F32), held[70:130])
    want = torch.cat([held[100:130], held[30:100]])
    assert torch.equal(buf.read(out_dtype=F32), want)
    assert buf.write(x[130:130]) == (30, 0) and buf.write(x[130:230]) == (30, 100)
    ids = torch.randperm(100, device="cuda")
    assert torch.equal(buf.read(ids, out_dtype=F32), torch.cat([held[200:230], held[130:200]])[ids])


def test_training_on_batches_from_the_buffer():
    """Batches read back go through forward_train: the gradients are those of the values read."""
    sae = small_sae("relu", 64, 512, F32)
    sae.requires_grad_(True)
    buf = saeflow_amd.ActivationBuffer(512, 64, center=sae.b_dec)
    buf.write(torch.randn(512, 64, device="cuda"))
    x = buf.read(torch.randperm(512, device="cuda")[:128], out_dtype=F32)
    x_hat, _ = saeflow_amd.forward_train(sae, x)
    (x_hat - x).pow(2).mean().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in (sae.W_enc, sae.b_enc, sae.W_dec, sae.b_dec))


# ----------------------------------------------------------------------------- refusals
def test_refusals():
    x, W = torch.randn(4, 200, device="cuda"), quantize_rows(torch.randn(10, 200, device="cuda"))
    for bad in (lambda: quantize_rows(x[0]), lambda: quantize_rows(x.int()), lambda: quantize_rows(x.cpu()),
                lambda: quantize_rows(x, shift=x[0, :100]), lambda: quantize_rows(x, row0=1),
                lambda: quantize_rows(x[:, :0]), lambda: quantize_rows(x, out=Fp8Rows.empty(4, 100)),
                lambda: quantize_rows(x, out=Fp8Rows.empty(3, 200)),
                lambda: quantize_rows(x, out=Fp8Rows.empty(8, 200), row0=8),
                lambda: quantize_rows(x, out=Fp8Rows.empty(8, 200), row0=-1),
                lambda: dequantize_rows(W, torch.zeros(3, dtype=torch.int32, device="cuda")),
                lambda: dequantize_rows(W, torch.zeros(3, dtype=torch.int64)), lambda: dequantize_rows(W, count=11),
                lambda: dequantize_rows(W, row0=10, count=1), lambda: dequantize_rows(W, out_dtype=torch.int32),
                lambda: dequantize_rows(W, torch.zeros(3, dtype=torch.int64, device="cuda"), count=3),
                lambda: fused_encode_fp8(x[:, :100], W), lambda: fused_encode_fp8(x, x),
                lambda: fused_encode_fp8(x, W, activation="gelu"), lambda: fused_encode_fp8(x, W, activation="jumprelu"),
                lambda: fused_encode_fp8(W, W, b_dec=x[0]), lambda: fused_encode_fp8(x, W, x[0]),
                lambda: fused_encode_fp8(x, W, row_nnz=torch.zeros(5, dtype=torch.int32, device="cuda")),
                lambda: fused_encode_fp8(x, W, out_dtype=torch.int8),
                lambda: Fp8Rows(W.q, W.scale, 300), lambda: Fp8Rows(W.q, W.scale[:5], 200),
                lambda: Fp8Rows.from_parts(W.q, W.scale), lambda: Fp8Rows.from_parts(x, W.scale),
                lambda: saeflow_amd.ActivationBuffer(0, 5), lambda: saeflow_amd.ActivationBuffer(2, 200).write(x),
                lambda: saeflow_amd.ActivationBuffer(9, 100).write(x),
                lambda: saeflow_amd.Fp8Encoder(x, x[:, 0], x[:, 0], activation="relu6"),
                lambda: saeflow_amd.Fp8Encoder(x, x[0], x[:, 0], activation="jumprelu"),
                lambda: saeflow_amd.Fp8Encoder(x, x[0], x[:, 0], activation="topk")):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        W[3]


@pytest.mark.parametrize("centered", [False, True])
def test_ids_of_rows_not_written_yet_read_as_zeros(centered):
    """An id between the rows written and the capacity has no row: zeros, as for an id past the capacity,
    whatever the memory behind it holds."""
    center = torch.randn(130, device="cuda") if centered else None
    buf = saeflow_amd.ActivationBuffer(100, 130, center=center)
    buf.store.q.view(torch.uint8).fill_(0x7F)  # NaN codes
    buf.store.scale.fill_(130)
    ids = torch.tensor([69, 70, 0, 99, 100, -1, 5], device="cuda")
    assert torch.equal(buf.read(ids, out_dtype=F32), torch.zeros(7, 130, device="cuda"))
    assert buf.read(ids[:0]).shape == (0, 130)
    for bad in (ids.int(), ids[None], ids.cpu()):
        with pytest.raises(ValueError):
            buf.read(bad)
    x = torch.randn(130, 130, device="cuda")
    held = dequantize_rows(quantize_rows(x, shift=center), shift=center, out_dtype=F32)
    buf.write(x[:70])
    want = held[ids.clamp(0, 69)]
    want[[1, 3, 4, 5]] = 0
    assert torch.equal(buf.read(ids, out_dtype=F32), want)
    assert torch.equal(buf.read(out_dtype=F32), held[:70])
    buf.write(x[70:100])  # full from here on
    want = held[ids.clamp(0, 99)]
    want[[4, 5]] = 0
    assert torch.equal(buf.read(ids, out_dtype=F32), want)
    buf.write(x[100:])
    assert torch.equal(buf.read(ids, out_dtype=F32)[2], held[100])


def test_a_write_is_refused_while_a_graph_is_captured():
    """The ring's place is the host's: replays would write the same rows over and over, and rows that were
    only captured would count as written. Reading may be captured."""
    buf = saeflow_amd.ActivationBuffer(50, 130)
    x = torch.randn(60, 130, device="cuda")
    held = dequantize_rows(quantize_rows(x), out_dtype=F32)
    buf.write(x[:20])
    ids = torch.arange(8, device="cuda")
    buf.read(ids, out_dtype=F32)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            buf.write(x[20:30])
        out = buf.read(ids, out_dtype=F32)
    assert len(buf) == 20 and buf.write(x.requires_grad_()[20:60]) == (20, 40) and len(buf) == 50
    for i in range(3):
        ids.copy_(torch.randperm(20, device="cuda")[:8])
        graph.replay()
        assert torch.equal(out, buf.read(ids, out_dtype=F32))
        assert torch.equal(out, torch.cat([held[50:60], held[10:20]])[ids])


@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M", [1, 20, 300, 2048])
def test_the_smallest_features_are_the_same_with_counts_and_without(M, out_dtype):
    """A zero product plus a bias down to the smallest subnormal: what the result's type holds of it is stored and
    counted, by every form alike."""
    N = 16384
    x, W = quantize_rows(torch.zeros(M, 200, device="cuda")), quantize_rows(torch.zeros(N, 200, device="cuda"))
    b = torch.zeros(N, dtype=torch.float64)
    b[:150] = 2.0 ** -torch.arange(150).double()
    b[150:300] = 2.0 ** -torch.arange(150).double() * 1.25
    b[300:450] = -b[:150]
    b = b.float().cuda()
    f = fused_encode_fp8(x, W, b, out_dtype=out_dtype)
    held = b.double() == b.to(BF16).double()  # (the largest tiles take a bias in bf16 pieces)
    assert torch.equal(f[:, held], b.clamp(min=0).to(out_dtype)[held].expand(M, -1))
    for thr, act in ((None, "relu"), (torch.zeros(N, device="cuda"), "jumprelu"), (b.abs(), "jumprelu")):
        nnz = torch.zeros(M, dtype=torch.int32, device="cuda")
        got = fused_encode_fp8(x, W, b, thr, act, out_dtype=out_dtype, row_nnz=nnz)
        want = torch.zeros_like(f) if thr is not None and thr.any() else f
        assert torch.equal(got, want) and torch.equal(nnz, (want != 0).sum(1, dtype=torch.int32))
        assert torch.equal(fused_encode_fp8(x, W, b, thr, act, out_dtype=out_dtype), want)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("activation", ["relu", "jumprelu", "topk"])
def test_sparse_features_of_large_products(activation, dtype):
    """CSR out of the persistent tiles: 2300 tokens x 16200 features, rows without features and rows of NaN among
    them, against the dense features of the same tiles and their nonzeros."""
    sae = small_sae(activation, 640, 16200, dtype)
    sae.b_enc.sub_(1.5)
    x = torch.randn(2300, 640, device="cuda").to(dtype)
    x[700:703] = sae.b_dec  # zeros once it is subtracted, and every bias below 0 drops them
    sae.b_enc.clamp_(max=-0.5)
    x[77, 5] = float("nan")
    enc = saeflow_amd.Fp8Encoder.from_sae(sae)
    f = enc.encode(x)
    indptr, indices, values = enc.encode_sparse(x)
    if activation == "topk":
        pre = fused_encode_fp8(x, enc.W, enc.b_enc, b_dec=enc.b_dec)
        v, i = topk_rows(pre, 16)
        assert torch.equal(indptr, torch.arange(0, 16 * 2300 + 1, 16, device="cuda"))
        assert torch.equal(indices.view(2300, 16), i) and torch.equal(values.nan_to_num(-7.0), v.nan_to_num(-7.0).flatten())
        return
    rows, cols = f.nonzero(as_tuple=True)
    assert torch.equal(indptr[1:], (f != 0).sum(1).cumsum(0)) and indptr[0] == 0
    assert torch.equal(indices, cols.int()) and torch.equal(values.nan_to_num(-7.0), f[rows, cols].nan_to_num(-7.0))
    assert not f[700:703].any() and f[77].isnan().all() and f[0].any()


@pytest.mark.parametrize("activation", ["relu", "jumprelu", "topk"])
def test_encoder_without_tokens(activation):
    enc = saeflow_amd.Fp8Encoder.from_sae(small_sae(activation))
    x = torch.empty(0, 300, dtype=BF16, device="cuda")
    for rows in (x, quantize_rows(x)):
        assert enc.encode(rows).shape == (0, 2000)
        indptr, indices, values = enc.encode_sparse(rows)
        assert indptr.tolist() == [0] and indices.numel() == 0 and values.numel() == 0


@pytest.mark.parametrize("times", [30, 3000])
def test_product_of_rows_with_outlying_dimensions(times):
    """Four dimensions `times` the others in size, biases that take most of what they add away again: the error
    stays below 7 * 2^-13 of sum |x w| (of each eight products, seven lose at most 2^-13 of the largest), fp32
    sums of K terms and one rounding."""
    M, N, K = 300, 4096, 768
    x = torch.randn(M, K, device="cuda")
    x[:, [5, 130, 131, 700]] = times * (1 + 0.1 * x[:, [5, 130, 131, 700]])
    x, W = quantize_rows(x), quantize_rows(torch.randn(N, K, device="cuda") / K ** 0.5)
    xv, wv = (dequantize_rows(r, out_dtype=F32).double() for r in (x, W))
    b = -(wv @ xv.mean(0)).float()
    want, size = xv @ wv.T.contiguous() + b.double(), xv.abs() @ wv.abs().T.contiguous() + b.double().abs()
    for dtype, u in ((F32, 0.0), (BF16, 2.0 ** -8), (F16, 2.0 ** -11)):
        err = (fused_encode_fp8(x, W, b, activation="none", out_dtype=dtype).double() - want).abs()
        sums = (K + 1) * 2.0 ** -23 + (7 * 2.0 ** -13 if u else 0.0)
        assert (err <= sums * size * (1 + u) + u * want.abs() + 2.0 ** -24).all()


def test_gradients_of_batches_from_the_buffer_are_those_of_the_values_read():
    """Batches are the definition's values in 64 bits, bit for bit, and the gradients of a step on them are float64
    autograd's at those values, to the tolerance of fp32 parameters (1e-4 of the largest, tests/test_gpu_backward.py)."""
    from oracle import backward as obwd

    sae = small_sae("relu", 200, 512, F32)
    sae.requires_grad_(True)
    data, b_dec = torch.randn(300, 200), sae.b_dec.detach().cpu()
    buf = saeflow_amd.ActivationBuffer(256, 200, center=sae.b_dec)
    buf.write(data[:200].cuda())
    buf.write(data[200:].cuda())  # over rows 0 to 43
    ids = torch.randperm(256)[:100]
    x = buf.read(ids.cuda(), out_dtype=F32)
    codes, scale = ofp8.quantize((torch.cat([data[256:], data[44:256]])[ids] - b_dec).numpy())
    held = torch.from_numpy(codes * np.repeat(2.0 ** (scale.astype(np.float64) - 127), 128, 1)[:, :200]).float()
    assert torch.equal(x.cpu(), held + b_dec)
    x_hat, (indptr, indices, values) = saeflow_amd.forward_train(sae, x)
    loss = (x_hat - x).pow(2).mean() + 0.01 * values.sum()
    loss.backward()
    G = (2 * (x_hat - x) / x.numel()).detach()
    active = csr_to_dense(indptr, indices, values.detach(), 512).cpu() > 0
    p = {name: getattr(sae, name).detach().cpu() for name in ("W_enc", "b_enc", "W_dec", "b_dec")}
    want = obwd.grads(held + b_dec, p["W_enc"], p["b_enc"], p["W_dec"], p["b_dec"], active, G.cpu(), torch.full((100, 512), 0.01))
    for name in p:
        got = getattr(sae, name).grad.double().cpu()
        torch.testing.assert_close(got, want[name], atol=1e-4 * float(want[name].abs().max()), rtol=1e-4, msg=name)


@pytest.mark.parametrize("M,N,K,out_dtype", [(16384, 16391, 1100, BF16), (16384, 18501, 300, F16), (18500, 18501, 120, BF16),
                                             (12000, 18500, 1030, F16)])
def test_many_results_of_rows_off_whole_lines(M, N, K, out_dtype):
    """Either kind of store, by d_in and the bytes of the results: whole numbers, whose sums (at most 9 * 1100) are
    exact in fp32 and rounded once."""
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    x = torch.randint(-3, 4, (M, K), generator=g, device="cuda").float()
    W = torch.randint(-3, 4, (N, K), generator=g, device="cuda").float()
    got = fused_encode_fp8(quantize_rows(x), quantize_rows(W), activation="none", out_dtype=out_dtype)
    assert torch.equal(got, (x @ W.T.contiguous()).to(out_dtype))
