"""GPU: layer norm forward, backward and undone against the formulas in float64 (oracle/norm.py).

Tolerances, with u = 2^-24 and e / 2 the half step of a result's type:
- a fp32 chain of n additions is off by at most n u of the sum of magnitudes; a wave adds D / 64 squares a lane, a block
  of 1024 threads D / 1024, then come six or ten levels, so rstd (half of its argument's relative error, and a root, a
  quotient and a product) is off by at most STAT = D / 128 + 16 units;
- mean is the rounded 64-bit sum, off by u |mean|, so x - mean by u (|mean| + |x - mean|), xh by u (STAT + 1) |xh| +
  u |mean| rstd;
- row sums of the backward pass add eight or D / 1024 elements a lane, six levels and up to sixteen waves: n = D / 1024 +
  48; column sums add at most M / 64 rows a lane, then blocks' parts: n = M / 64 + 64.
"""

import pytest
import torch

import saeflow_amd
from oracle import fp8 as ofp8
from oracle import norm as onorm
from saeflow_amd import kernels
from saeflow_amd.kernels import Fp8Rows

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# one element, inside a chunk, chunk and block edges, a wave, teams of waves, the longest row of a wave, of a team, longer
WIDTHS = [1, 2, 7, 8, 9, 64, 100, 127, 129, 511, 512, 513, 768, 1000, 1003, 1537, 2304, 4095, 4096, 4097, 6144, 8191, 8192, 8200, 20001]


def half(dtype):
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else U


def tiny(dtype):
    """Half of the smallest step (subnormal results)."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def stat_units(D):
    return D / 128 + 16


def make(M, D, dtype, seed=0, w_dtype=None, offset=0.3):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = ((n(M, D) * torch.exp(0.5 * n(D)) + offset) * torch.exp(0.3 * n(M, 1))).to(dtype)
    wd = w_dtype or dtype
    return x, (1 + 0.2 * n(D)).to(wd), (0.1 * n(D)).to(wd), (0.1 * n(M, D)).to(dtype)


def within(got, want, tol, what):
    got = got.detach().double().cpu()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol.clamp(min=1e-300)).max()):.3g} of the tolerance"


def check_forward(x, w, b, y, mean, rstd, eps=1e-5):
    D = x.shape[1]
    want, mean64, rstd64, xh = onorm.forward(x, w, b, eps)
    within(mean, mean64, 1.01 * U * mean64.abs() + 1e-300, "mean")
    within(rstd, rstd64, U * stat_units(D) * rstd64, "rstd")
    wa = torch.ones(D, dtype=torch.float64) if w is None else w.double().cpu().abs()
    tol = half(y.dtype) * want.abs() * 1.01 + tiny(y.dtype) + U * wa * ((stat_units(D) + 3) * xh.abs() + (mean64.abs() * rstd64)[:, None])
    if b is not None:
        tol = tol + U * (want.abs() + b.double().cpu().abs())
    within(y, want, tol, "y")


def check_backward(g, d, rstd, w, b, gr, mean, g_mean=None, g_rstd=None, exact_input=False, D=None):
    """d: the centred rows (float64); exact_input: they and rstd are what the kernel was given."""
    M, D = g.shape
    o = onorm.backward(g, d, rstd, w, g_mean, g_rstd)
    st, n = (2.0 if exact_input else stat_units(D) + 2), D / 1024 + 48
    r = rstd.double().cpu()[:, None]
    dxh = U * (st * o.xh.abs() + (0 if exact_input else (mean.double().cpu().abs()[:, None] * r)))
    if gr.x is not None:
        want = o.x
        tol = r * (U * ((4 + st) * (o.q.abs() + o.c1.abs()) + n * o.mq) + dxh * o.c2.abs()
                   + o.xh.abs() * (U * ((6 + st) * o.c2.abs() + n * o.mqx) + (o.q.abs() * dxh).mean(1, keepdim=True)))
        if g_mean is not None:
            tol = tol + 4 * U * g_mean.double().cpu().abs()[:, None] / D
        if g_rstd is not None:
            tol = tol + ((8 + 2 * st) * U * o.xh.abs() + dxh) * (g_rstd.double().cpu().abs()[:, None] * r * r / D)
        within(gr.x, want, 1.01 * half(gr.x.dtype) * want.abs() + tiny(gr.x.dtype) + 1.01 * tol, "dx")
    rows = M / 64 + 64
    if w is not None:
        tol = U * (rows + 3) * o.aw + (g.double().cpu().abs() * dxh).sum(0)
        within(gr.weight, o.weight, 1.01 * half(gr.weight.dtype) * o.weight.abs() + tiny(gr.weight.dtype) + 1.01 * tol, "dweight")
    if b is not None:
        within(gr.bias, o.bias, 1.01 * half(gr.bias.dtype) * o.bias.abs() + tiny(gr.bias.dtype) + U * rows * o.ab, "dbias")


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def held_values(rows8):
    return kernels.dequantize_rows(rows8, out_dtype=torch.float32).double().cpu()


def check_held(x, held):
    """The codes are those of fp32(x - mean), mean the 64-bit mean rounded to 32 bits, byte for byte."""
    mean = (x.double().cpu().sum(1) / x.shape[1]).float()
    d = (x.double().cpu() - mean.double()[:, None]).float()
    codes, scale = ofp8.quantize(d.numpy())
    nb = scale.shape[1]
    assert (held.scale.cpu().numpy()[:, :nb] == scale).all() and (held.scale.cpu().numpy()[:, nb:] == 0).all()
    q = held.q.view(torch.uint8).cpu().numpy()
    assert (ofp8.CODES[q[:, :x.shape[1]]] == codes).all() and (q[:, x.shape[1]:] == 0).all()


# ----------------------------------------------------------------------------- against the formulas
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", WIDTHS)
def test_forward_and_backward_over_widths(D, dtype):
    M = 19 if D <= 4096 else 5
    x, w, b, g = make(M, D, dtype, seed=D)
    xg, wg, bg, gg = cuda(x, w, b, g)
    y, mean, rstd = kernels.layer_norm(xg, wg, bg)
    assert y.dtype == dtype and mean.dtype == rstd.dtype == torch.float32
    check_forward(x, w, b, y, mean, rstd)
    gr = kernels.layer_norm_backward(gg, xg, mean, rstd, wg, bg)
    _, mean64, rstd64, _ = onorm.forward(x)
    check_backward(g, x.double() - mean64[:, None], rstd64, w, b, gr, mean64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", WIDTHS)
def test_held_over_widths(D, dtype):
    M = 7 if D <= 4096 else 3
    x, w, b, g = make(M, D, dtype, seed=D + 1)
    xg, wg, bg, gg = cuda(x, w, b, g)
    y, held, mean, rstd = kernels.layer_norm_held(xg, wg, bg)
    y0, mean0, rstd0 = kernels.layer_norm(xg, wg, bg)
    assert torch.equal(y, y0) and torch.equal(mean, mean0) and torch.equal(rstd, rstd0)
    check_held(x, held)
    gr = kernels.layer_norm_backward(gg, held, None, rstd, wg, bg)
    assert gr.x.dtype == dtype
    check_backward(g, held_values(held), rstd.cpu(), w, b, gr, mean, exact_input=True)


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 17, 255, 1021, 2049, 5003])
@pytest.mark.parametrize("D", [40, 520, 1003, 2304])
def test_row_counts(M, D):
    x, w, b, g = make(M, D, torch.bfloat16, seed=M)
    xg, wg, bg, gg = cuda(x, w, b, g)
    y, held, mean, rstd = kernels.layer_norm_held(xg, wg, bg)
    check_forward(x, w, b, y, mean, rstd)
    _, mean64, rstd64, _ = onorm.forward(x)
    check_backward(g, x.double() - mean64[:, None], rstd64, w, b, kernels.layer_norm_backward(gg, xg, mean, rstd, wg, bg), mean64)
    check_backward(g, held_values(held), rstd.cpu(), w, b, kernels.layer_norm_backward(gg, held, mean, rstd, wg, bg), mean64, exact_input=True)


def test_many_short_rows_and_few_long_ones():
    for M, D in ((70001, 8), (3, 40000), (200, 9000)):
        x, w, b, g = make(M, D, torch.float32, seed=M)
        xg, wg, bg, gg = cuda(x, w, b, g)
        y, mean, rstd = kernels.layer_norm(xg, wg, bg)
        check_forward(x, w, b, y, mean, rstd)
        _, mean64, rstd64, _ = onorm.forward(x)
        check_backward(g, x.double() - mean64[:, None], rstd64, w, b, kernels.layer_norm_backward(gg, xg, mean, rstd, wg, bg), mean64)


@pytest.mark.parametrize("x_dtype", DTYPES)
@pytest.mark.parametrize("w_dtype", DTYPES)
@pytest.mark.parametrize("out_dtype", DTYPES)
def test_types_mix(x_dtype, w_dtype, out_dtype):
    M, D = 33, 777
    x, w, b, g = make(M, D, x_dtype, w_dtype=w_dtype)
    g, b = g.to(out_dtype), b.to(x_dtype)
    xg, wg, bg, gg = cuda(x, w, b, g)
    y, held, mean, rstd = kernels.layer_norm_held(xg, wg, bg, out_dtype=out_dtype)
    assert y.dtype == out_dtype
    check_forward(x, w, b, y, mean, rstd)
    _, mean64, rstd64, _ = onorm.forward(x)
    gr = kernels.layer_norm_backward(gg, xg, mean, rstd, wg, bg)
    assert (gr.x.dtype, gr.weight.dtype, gr.bias.dtype) == (x_dtype, w_dtype, x_dtype)
    check_backward(g, x.double() - mean64[:, None], rstd64, w, b, gr, mean64)
    gr = kernels.layer_norm_backward(gg, held, None, rstd, wg, bg, out_dtype=w_dtype)
    assert gr.x.dtype == w_dtype
    check_backward(g, held_values(held), rstd.cpu(), w, b, gr, mean64, exact_input=True)


@pytest.mark.parametrize("D", [1003, 9001])
@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
def test_without_weight_or_bias(D, has_w, has_b):
    x, w, b, g = make(21, D, torch.float32)
    w, b = (w if has_w else None), (b if has_b else None)
    xg, wg, bg, gg = cuda(x, w, b, g)
    y, mean, rstd = kernels.layer_norm(xg, wg, bg)
    check_forward(x, w, b, y, mean, rstd)
    _, mean64, rstd64, _ = onorm.forward(x)
    d = x.double() - mean64[:, None]
    gr = kernels.layer_norm_backward(gg, xg, mean, rstd, wg, bg)
    assert (gr.weight is None) == (not has_w) and (gr.bias is None) == (not has_b)
    check_backward(g, d, rstd64, w, b, gr, mean64)
    if has_w or has_b:
        only = kernels.layer_norm_backward(gg, xg, mean, rstd, wg, bg, need_grad_x=False)
        assert only.x is None
        check_backward(g, d, rstd64, w, b, only, mean64)


@pytest.mark.parametrize("D", [40, 1000, 8500])
def test_gradients_of_mean_and_rstd(D):
    x, w, b, g = make(11, D, torch.float32)
    gm, gs = torch.randn(11), torch.randn(11)
    xg, wg, bg, gg, gmg, gsg = cuda(x, w, b, g, gm, gs)
    _, mean, rstd = kernels.layer_norm(xg, wg, bg)
    _, mean64, rstd64, _ = onorm.forward(x)
    gr = kernels.layer_norm_backward(gg, xg, mean, rstd, wg, bg, grad_mean=gmg, grad_rstd=gsg)
    check_backward(g, x.double() - mean64[:, None], rstd64, w, b, gr, mean64, gm, gs)


def test_strides_alignments_and_orders():
    M, D = 37, 1001
    big = torch.randn(2 * M, D + 60).to(torch.bfloat16)
    w, b = torch.randn(D + 3).bfloat16()[3:], torch.randn(2 * D).bfloat16()[::2]
    views = {"rows apart": big[::2, 3:3 + D], "an odd address": big.flatten()[1:1 + M * D].view(M, D),
             "columns contiguous": torch.randn(D, M).bfloat16().T, "every second element": torch.randn(M, 2 * D).bfloat16()[:, ::2],
             "one row for all": big[:1, :D].expand(M, D)}
    for what, x in views.items():
        g = torch.randn(D, M).bfloat16().T if "columns" in what else torch.randn(M, D + 7).bfloat16()[:, 7:]
        # the views of the device tensors have the same strides
        xg = {"rows apart": lambda: big.cuda()[::2, 3:3 + D], "an odd address": lambda: big.cuda().flatten()[1:1 + M * D].view(M, D),
              "columns contiguous": lambda: x.T.cuda().T, "every second element": lambda: torch.stack([x, x], 2).reshape(M, 2 * D).cuda()[:, ::2],
              "one row for all": lambda: big.cuda()[:1, :D].expand(M, D)}[what]()
        assert torch.equal(xg.cpu(), x)
        wg, bg = torch.cat([torch.zeros(3).bfloat16(), w]).cuda()[3:], torch.stack([b, b], 1).flatten().cuda()[::2]
        gg = g.T.cuda().T if "columns" in what else torch.cat([torch.zeros(M, 7).bfloat16(), g], 1).cuda()[:, 7:]
        y, held, mean, rstd = kernels.layer_norm_held(xg, wg, bg)
        check_forward(x, w, b, y, mean, rstd)
        check_held(x, held)
        _, mean64, rstd64, _ = onorm.forward(x)
        check_backward(g, x.double() - mean64[:, None], rstd64, w, b, kernels.layer_norm_backward(gg, xg, mean, rstd, wg, bg), mean64)
    # the gradient of a sum is one element expanded
    x, w, b, _ = make(M, D, torch.float32)
    xg, wg, bg = cuda(x, w, b)
    _, mean, rstd = kernels.layer_norm(xg, wg, bg)
    g = torch.ones(1, 1).expand(M, D)
    _, mean64, rstd64, _ = onorm.forward(x)
    gr = kernels.layer_norm_backward(g.cuda()[:1, :1].expand(M, D), xg, mean, rstd, wg, bg)
    check_backward(g, x.double() - mean64[:, None], rstd64, w, b, gr, mean64)


def test_rows_that_are_not_numbers_stay_by_themselves():
    for D in (1000, 5000):
        x, w, b, g = make(9, D, torch.float32)
        x[2, 5], x[4, D - 1], x[6, 0] = float("nan"), float("inf"), -float("inf")
        xg, wg, bg, gg = cuda(x, w, b, g)
        y, held, mean, rstd = kernels.layer_norm_held(xg, wg, bg)
        clean = [0, 1, 3, 5, 7, 8]
        assert torch.isnan(y[[2, 4, 6]]).all()
        check_forward(x[clean], w, b, y[clean], mean[clean], rstd[clean])
        for source in (xg, held):
            gr = kernels.layer_norm_backward(gg, source, mean, rstd, wg, bg)
            assert torch.isnan(gr.x[[2, 4, 6]]).all() and torch.isfinite(gr.x[clean]).all()
            assert torch.isnan(gr.weight).all() and torch.isfinite(gr.bias).all()


def test_constant_rows_extreme_values_and_eps():
    x = torch.stack([torch.full((300,), 3.5), torch.zeros(300), torch.linspace(-1, 1, 300) * 1e-20, torch.linspace(-1, 1, 300) + 1e4])
    xg = x.cuda()
    y, mean, rstd = kernels.layer_norm(xg, eps=1e-5)
    check_forward(x, None, None, y, mean, rstd)
    assert (y[0] == 0).all() and (y[1] == 0).all()
    y, mean, rstd = kernels.layer_norm(xg[3:], eps=0.0)
    check_forward(x[3:], None, None, y, mean, rstd, eps=0.0)
    one = torch.tensor([[2.0], [-7.0]])
    y, mean, rstd = kernels.layer_norm(one.cuda(), torch.tensor([2.0]).cuda(), torch.tensor([0.5]).cuda())
    assert (y == 0.5).all() and torch.equal(mean.cpu(), one[:, 0])
    gr = kernels.layer_norm_backward(torch.ones(2, 1).cuda(), one.cuda(), mean, rstd, torch.tensor([2.0]).cuda(), torch.tensor([0.5]).cuda())
    assert (gr.x == 0).all() and (gr.weight == 0).all() and (gr.bias == 2).all()


def test_no_rows():
    w = torch.ones(12, device="cuda", dtype=torch.float16)
    x = torch.empty(0, 12, device="cuda", dtype=torch.float16)
    y, held, mean, rstd = kernels.layer_norm_held(x, w, w)
    assert y.shape == (0, 12) and len(held) == 0 and mean.shape == rstd.shape == (0,)
    for source in (x, held):
        gr = kernels.layer_norm_backward(x, source, mean, rstd, w, w)
        assert gr.x.shape == (0, 12) and (gr.weight == 0).all() and (gr.bias == 0).all()
    assert kernels.denormalize(x, mean, rstd).shape == (0, 12)
    dh, dm, dr = kernels.denormalize_backward(x, x, rstd)
    assert dh.shape == (0, 12) and dm.shape == dr.shape == (0,)


def test_offsets_past_four_gigabytes():
    M, D = 1 << 20, 2304  # 4.8 GB
    x = torch.zeros(M, D, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(M, D, dtype=torch.bfloat16, device="cuda")
    tail, w, b, gt = make(8, D, torch.bfloat16)
    x[-8:], g[-8:] = tail.cuda(), gt.cuda()
    wg, bg = cuda(w, b)
    y, held, mean, rstd = kernels.layer_norm_held(x, wg, bg)
    check_forward(tail, w, b, y[-8:], mean[-8:], rstd[-8:])
    assert torch.equal(y[:-8], bg.expand(M - 8, D))
    gr = kernels.layer_norm_backward(g, held, None, rstd, wg, bg)
    check_backward(gt, held_values(held[M - 8:M]), rstd[-8:].cpu(), w, b, gr_rows(gr, slice(M - 8, M)), mean, exact_input=True)
    assert (gr.x[:-8] == 0).all()
    del held
    _, mean64, rstd64, _ = onorm.forward(tail)
    gr = kernels.layer_norm_backward(g, x, mean, rstd, wg, bg)
    check_backward(gt, tail.double() - mean64[:, None], rstd64, w, b, gr_rows(gr, slice(M - 8, M)), mean64)


def gr_rows(gr, rows):
    return type(gr)(x=gr.x[rows], weight=gr.weight, bias=gr.bias)


def test_repeated_calls_give_the_same_bits_and_neighbours_are_left_alone():
    x, w, b, g = make(2049, 1003, torch.bfloat16)
    xg, wg, bg, gg = cuda(x, w, b, g)
    y, held, mean, rstd = kernels.layer_norm_held(xg, wg, bg)
    a = kernels.layer_norm_backward(gg, held, None, rstd, wg, bg)
    for _ in range(3):
        c = kernels.layer_norm_backward(gg, held, None, rstd, wg, bg)
        for name in ("x", "weight", "bias"):
            assert torch.equal(getattr(a, name), getattr(c, name)), name
    # a row's result does not depend on the rows beside it
    y1, h1, m1, r1 = kernels.layer_norm_held(xg[700:701], wg, bg)
    assert torch.equal(y1[0], y[700]) and torch.equal(h1.q.view(torch.uint8)[0], held.q.view(torch.uint8)[700])
    g1 = kernels.layer_norm_backward(gg[700:701], held[700:701], None, rstd[700:701], wg, bg)
    assert torch.equal(g1.x[0], a.x[700])


# ----------------------------------------------------------------------------- undone
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,D", [(1, 1), (3, 7), (5, 513), (137, 1003), (33, 2304), (2, 30001)])
def test_denormalize(M, D, dtype):
    g = torch.Generator().manual_seed(D)
    h, gr = torch.randn(M, D, generator=g).to(dtype), torch.randn(M, D, generator=g).to(dtype)
    mean, rstd = torch.randn(M, generator=g), torch.exp(0.5 * torch.randn(M, generator=g))
    hg, gg, mg, rg = cuda(h, gr, mean, rstd)
    out = kernels.denormalize(hg, mg, rg)
    want = onorm.undone(h, mean, rstd)
    # h r + (h e + mean): three roundings, of terms no larger than |h| / rstd and |mean|
    mags = h.double().abs() / rstd.double()[:, None] + mean.double().abs()[:, None]
    within(out, want, 1.01 * half(dtype) * want.abs() + tiny(dtype) + 2 * U * mags, "out")
    dh, dmean, drstd = kernels.denormalize_backward(gg, hg, rg)
    wh, wm, wr = onorm.undone_backward(gr, h, rstd)
    within(dh, wh, 1.01 * half(dtype) * wh.abs() + tiny(dtype) + 2 * U * wh.abs(), "dh")
    n = D / 64 + 8
    within(dmean, wm, U * n * gr.double().abs().sum(1), "dmean")
    within(drstd, wr, U * (n + 4) * (gr.double() * h.double()).abs().sum(1) / rstd.double() ** 2, "drstd")
    only = kernels.denormalize_backward(gg, None, rg, need_grad_stats=False, out_dtype=torch.float32)
    assert only[1] is None and only[2] is None
    within(only[0], wh, 3 * U * wh.abs(), "dh alone")
    wide = torch.zeros(M, D + 5, dtype=dtype)
    wide[:, 5:] = h
    assert torch.equal(kernels.denormalize(wide.cuda()[:, 5:], mg, rg), out)


def test_layer_norm_undone_gives_the_rows_back():
    x, _, _, _ = make(64, 999, torch.float32)
    xg = x.cuda()
    y, mean, rstd = kernels.layer_norm(xg)
    back = kernels.denormalize(y, mean, rstd)
    scale = x.abs().double() + 1 / rstd.double().cpu()[:, None]
    within(back, x.double(), (stat_units(999) + 6) * U * scale, "x")


# ----------------------------------------------------------------------------- autograd
@pytest.mark.parametrize("hold", [None, torch.float8_e4m3fn])
def test_autograd_through_norm_and_back(hold):
    """layer_norm over leading dimensions, its statistics used twice, and the norm undone, against float64 autograd (with
    hold: against the formulas on what the rows hold)."""
    x, w, b, g = make(6 * 5, 200, torch.float32)
    leaves = [t.cuda().requires_grad_(True) for t in (x.view(6, 5, 200), w, b)]
    y, mean, rstd = saeflow_amd.layer_norm(*leaves, hold=hold, return_stats=True)
    assert y.shape == (6, 5, 200) and mean.shape == rstd.shape == (6, 5)
    out = saeflow_amd.denormalize(y * 0.5, mean, rstd)
    (out * g.view(6, 5, 200).cuda()).sum().backward()
    l64 = [t.double().requires_grad_(True) for t in (x, w, b)]
    m64 = l64[0].mean(1, keepdim=True)
    r64 = ((l64[0] - m64) ** 2).mean(1, keepdim=True).add(1e-5).rsqrt()
    y64 = (l64[0] - m64) * r64 * l64[1] + l64[2]
    out64 = y64 * 0.5 / r64 + m64
    torch.testing.assert_close(out.detach().double().cpu().view(30, 200), out64.detach(), atol=2e-5, rtol=2e-5)
    if hold is None:
        (out64 * g.double()).sum().backward()
        for leaf, want in zip(leaves, l64):
            got = leaf.grad.double().cpu().reshape(want.shape)
            torch.testing.assert_close(got, want.grad, atol=2e-5 * float(want.grad.abs().max()), rtol=2e-5)
    else:
        d = held_values(kernels.layer_norm_held(x.cuda())[1])
        r = r64.detach()[:, 0]
        gy = g.double() * 0.5 / r[:, None]
        _, gm, gs = onorm.undone_backward(g, y64.detach() * 0.5, r)
        want = onorm.backward(gy, d, r, w, gm, gs)
        for leaf, ref in zip(leaves, (want.x, want.weight, want.bias)):
            got = leaf.grad.double().cpu().reshape(ref.shape)
            torch.testing.assert_close(got, ref, atol=2e-5 * float(ref.abs().max()), rtol=2e-5)


def test_autograd_of_some_inputs_alone():
    x, w, b, g = make(12, 96, torch.bfloat16)
    xg, wg, bg, gg = cuda(x, w, b, g)
    _, mean, rstd = kernels.layer_norm(xg, wg, bg)
    full = kernels.layer_norm_backward(gg, xg, mean, rstd, wg, bg)
    for pick in ((0,), (1,), (2,), (0, 2)):
        leaves = [t.clone().requires_grad_(i in pick) for i, t in enumerate((xg, wg, bg))]
        saeflow_amd.layer_norm(*leaves).backward(gg)
        for i, name in enumerate(("x", "weight", "bias")):
            assert (leaves[i].grad is None) == (i not in pick)
            if i in pick:
                assert torch.equal(leaves[i].grad, getattr(full, name))
    xr = xg.clone().requires_grad_(True)
    saeflow_amd.layer_norm(xr, return_stats=True)[1].sum().backward()  # the mean alone
    torch.testing.assert_close(xr.grad.float(), torch.full((12, 96), 1 / 96, device="cuda"), atol=0, rtol=2.0 ** -8)
    with torch.no_grad():
        assert torch.equal(saeflow_amd.layer_norm(xr, wg, bg), saeflow_amd.layer_norm(xg, wg, bg))


# ----------------------------------------------------------------------------- streams and graphs
def test_on_another_stream():
    x, w, b, g = make(513, 768, torch.bfloat16)
    xg, wg, bg, gg = cuda(x, w, b, g)
    y, mean, rstd = kernels.layer_norm(xg, wg, bg)
    want = kernels.layer_norm_backward(gg, xg, mean, rstd, wg, bg)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y2, mean2, rstd2 = kernels.layer_norm(xg, wg, bg)
        got = kernels.layer_norm_backward(gg, xg, mean2, rstd2, wg, bg)
    side.synchronize()
    assert torch.equal(y, y2) and torch.equal(got.x, want.x) and torch.equal(got.weight, want.weight) and torch.equal(got.bias, want.bias)


def test_graph_replays_match_eager():
    M, D = 1030, 1003
    x, w, b, g = cuda(*make(M, D, torch.bfloat16))

    def step():
        y, held, mean, rstd = kernels.layer_norm_held(x, w, b)
        gr = kernels.layer_norm_backward(g, held, None, rstd, w, b)
        z = kernels.denormalize(y, mean, rstd)
        return y, gr.x, gr.weight, gr.bias, z, *kernels.denormalize_backward(g, y, rstd)

    step()
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    with torch.cuda.graph(other):  # a second one beside it, with its own workspaces
        outs2 = step()
    for seed in (1, 2, 3):
        nx, _, _, ng = make(M, D, torch.bfloat16, seed=seed)
        x.copy_(nx)
        g.copy_(ng)
        (torch.randn(500, 500, device="cuda") @ torch.randn(500, 500, device="cuda")).sum().item()
        want = step()
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        for i, (a, c, e) in enumerate(zip(want, outs, outs2)):
            assert torch.equal(a, c) and torch.equal(a, e), (seed, i)


@pytest.mark.parametrize("D", [40, 1000, 8500])
@pytest.mark.parametrize("size", [1e-18, 1e15])
def test_rows_of_any_size(size, D):
    """Deviations whose cubes leave fp32 (gradients of the rows go with 1 / size)."""
    x, w, b, g = make(9, D, torch.float32)
    x = x * size
    xg, wg, bg, gg = cuda(x, w, b, g)
    y, held, mean, rstd = kernels.layer_norm_held(xg, wg, bg, eps=0.0)
    check_forward(x, w, b, y, mean, rstd, eps=0.0)
    check_held(x, held)
    _, mean64, rstd64, _ = onorm.forward(x, eps=0.0)
    check_backward(g, x.double() - mean64[:, None], rstd64, w, b, kernels.layer_norm_backward(gg, xg, mean, rstd, wg, bg), mean64)
    check_backward(g, held_values(held), rstd.cpu(), w, b, kernels.layer_norm_backward(gg, held, None, rstd, wg, bg), mean64, exact_input=True)


@pytest.mark.parametrize("D", [96, 1003, 2304, 5000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_mean_and_rstd_from_held_rows(D, dtype):
    x, w, b, g = make(23, D, dtype)
    gm, gs = torch.randn(23), torch.randn(23)
    xg, wg, bg, gg, gmg, gsg = cuda(x, w, b, g, gm, gs)
    _, held, mean, rstd = kernels.layer_norm_held(xg, wg, bg)
    for a, c in ((gmg, gsg), (gmg, None), (None, gsg)):
        gr = kernels.layer_norm_backward(gg, held, None, rstd, wg, bg, grad_mean=a, grad_rstd=c)
        check_backward(g, held_values(held), rstd.cpu(), w, b, gr, mean, a, c, exact_input=True)
