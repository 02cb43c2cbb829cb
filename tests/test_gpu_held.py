"""GPU: training and applying dictionaries on normed activations, and their backward pass from activations held in 8 bits.

Tolerances of the gradients, with u = 2^-24 and e / 2 the half step of a result's type: dL/dpre of an entry is a dot
product of D terms (at most D / 64 + 24 additions to a lane's sum) plus a given gradient; a feature's sum over n entries
adds them one after the other (n + 8 with the parts of long columns). Each is bounded by u times that number times the
sum of magnitudes.
"""

import pytest
import torch

import saeflow_amd
from cache_model import TinyHooked
from oracle import norm as onorm
from saeflow_amd import SAE, Fp8Encoder, _lib, denormalize, forward_train, kernels, layer_norm
from saeflow_amd.cache import ActivationReader, cache_activations
from saeflow_amd.kernels import csr_to_dense, dequantize_rows, quantize_rows, sparse_backward
from test_gpu_norm import U, cuda, half, held_values, tiny, within

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def problem(M, D, N, dtype, seed=0, l0=6, hot=0):
    """Tokens, a dictionary, CSR features (some rows empty, `hot` features on in nearly every token) and gradients."""
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = (n(M, D) * torch.exp(0.5 * n(D)) + 0.2).to(dtype)
    W_enc, W_dec = (n(D, N) / D ** 0.5).to(dtype), (n(N, D) / D ** 0.5).to(dtype)
    b_enc, b_dec = (0.1 * n(N)).to(dtype), (0.1 * n(D)).to(dtype)
    f = n(M, N).abs() * (torch.rand(M, N, generator=g) < min(1.0, l0 / N))
    f[:, :hot] = n(M, hot).abs() + 0.1
    f[::5] = 0
    f = f.to(dtype)
    indptr = torch.zeros(M + 1, dtype=torch.int64)
    indptr[1:] = (f != 0).sum(1).cumsum(0)
    indices, values = f.nonzero()[:, 1].int(), f[f != 0]
    return x, W_enc, b_enc, W_dec, b_dec, (indptr, indices, values), f, (0.1 * n(M, D)).to(dtype), (0.05 * n(indices.numel())).to(dtype)


def check_held_backward(M, D, N, dtype, **kw):
    x, W_enc, b_enc, W_dec, b_dec, csr, f, G, H = problem(M, D, N, dtype, **kw)
    dev = cuda(x, W_enc, b_enc, W_dec, b_dec, *csr, G, H)
    xg, We, be, Wd, bd, ip, ix, va, Gg, Hg = dev
    held = quantize_rows(xg, shift=bd)
    got = sparse_backward(held, We, be, Wd, bd, (ip, ix, va), Gg, Hg)
    plain = sparse_backward(xg, We, be, Wd, bd, (ip, ix, va), Gg, Hg)
    for name in ("b_enc", "W_dec", "b_dec", "pre"):  # what does not depend on x
        assert torch.equal(getattr(got, name), getattr(plain, name)), name
    assert got.x.dtype == torch.float32 and torch.equal(got.x.to(dtype), plain.x)
    v = held_values(held)
    on = f != 0
    Hd = torch.zeros(M, N, dtype=torch.float64)
    Hd[on] = H.double()
    p = (G.double() @ W_dec.double().T + Hd) * on
    pa = (G.double().abs() @ W_dec.double().abs().T + Hd.abs()) * on
    want = v.T @ p
    entries = on.sum(0).double()
    tol = U * (entries + 8) * (v.abs().T @ p.abs()) + U * (D / 64 + 24) * (v.abs().T @ pa)
    within(got.W_enc, want, 1.01 * half(dtype) * want.abs() + tiny(dtype) + 1.01 * tol, "dW_enc")
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,D,N", [(1, 64, 256), (64, 128, 256), (37, 50, 129), (41, 1, 70), (29, 7, 64), (300, 129, 520),
                                   (203, 513, 192), (120, 1003, 333), (130, 2304, 256), (17, 4099, 65)])
def test_sparse_backward_from_held_rows(M, D, N, dtype):
    check_held_backward(M, D, N, dtype, seed=D)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [96, 1000, 2304])
def test_sparse_backward_from_held_rows_with_long_columns(D, dtype):
    """Features that are on in nearly every token: several parts of 256 entries each, and just over 64 entries."""
    check_held_backward(1500, D, 136, dtype, l0=9, hot=3)
    check_held_backward(90, D, 72, dtype, l0=4, hot=5)


def test_sparse_backward_from_held_rows_over_many_features():
    """More features than entries: four work items share a wave."""
    check_held_backward(200, 256, 9000, torch.bfloat16, l0=8)


def test_sparse_backward_from_held_rows_is_deterministic():
    a = check_held_backward(1500, 256, 384, torch.bfloat16, hot=3)
    b = check_held_backward(1500, 256, 384, torch.bfloat16, hot=3)
    assert torch.equal(a.W_enc, b.W_enc)


def test_held_rows_of_a_store_with_strides():
    x, W_enc, b_enc, W_dec, b_dec, csr, f, G, _ = problem(64, 300, 128, torch.bfloat16)
    xg, We, be, Wd, bd, ip, ix, va, Gg = cuda(x, W_enc, b_enc, W_dec, b_dec, *csr, G)
    held = quantize_rows(xg, shift=bd)
    store = kernels.Fp8Rows.empty(200, 300)
    quantize_rows(xg, shift=bd, out=store, row0=57)
    wide = kernels.Fp8Rows(torch.empty(64, 512, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :384],
                           torch.empty(64, 8, dtype=torch.uint8, device="cuda")[:, 4:], 300)
    quantize_rows(xg, shift=bd, out=wide)
    want = sparse_backward(held, We, be, Wd, bd, (ip, ix, va), Gg, need_grad_x=False).W_enc
    for rows in (store[57:121], wide):
        assert torch.equal(sparse_backward(rows, We, be, Wd, bd, (ip, ix, va), Gg, need_grad_x=False).W_enc, want)


def test_held_rows_are_refused_where_they_do_not_fit():
    x, W_enc, b_enc, W_dec, b_dec, csr, f, G, _ = problem(8, 64, 32, torch.bfloat16)
    xg, We, be, Wd, bd, ip, ix, va, Gg = cuda(x, W_enc, b_enc, W_dec, b_dec, *csr, G)
    with pytest.raises(ValueError):
        sparse_backward(quantize_rows(xg[:, :60]), We, be, Wd, bd, (ip, ix, va), Gg)
    with pytest.raises(ValueError):
        sparse_backward(quantize_rows(xg[:7]), We, be, Wd, bd, (ip, ix, va), Gg)


# ----------------------------------------------------------------------------- forward_train
def make_sae(D, N, activation, dtype, norm=None, k=8, seed=0):
    torch.manual_seed(seed)
    sae = SAE(D, N, activation, k=k if activation == "topk" else None, dtype=dtype, input_norm=norm).cuda()
    with torch.no_grad():
        sae.b_enc.copy_(0.1 * torch.randn(N) - (0.0 if activation == "topk" else 0.5))
        sae.b_dec.copy_(0.1 * torch.randn(D))
        if activation == "jumprelu":
            sae.threshold.copy_(0.3 * torch.rand(N))
    for name in ("W_enc", "b_enc", "W_dec", "b_dec"):
        getattr(sae, name).requires_grad_(True)
    return sae


def grads_of(sae):
    out = {n: getattr(sae, n).grad.clone() for n in ("W_enc", "b_enc", "W_dec", "b_dec")}
    for n in out:
        getattr(sae, n).grad = None
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ["relu", "jumprelu", "topk"])
def test_forward_train_held(activation, dtype):
    """The same features, reconstruction and gradients as without, but dW_enc, which is sparse_backward's from the rows."""
    sae = make_sae(100, 300, activation, dtype)
    x = torch.randn(70, 100, device="cuda").to(dtype).requires_grad_(True)
    G = torch.randn(70, 100, device="cuda").to(dtype)

    def run(hold):
        x_hat, csr = forward_train(sae, x, hold=hold)
        ((x_hat * G).sum() + 0.1 * csr[2].float().sum()).backward()
        gx, x.grad = x.grad, None
        return x_hat.detach(), csr, gx, grads_of(sae)

    x0, csr0, gx0, g0 = run(None)
    x1, csr1, gx1, g1 = run(torch.float8_e4m3fn)
    assert torch.equal(x0, x1) and all(torch.equal(a, b) for a, b in zip(csr0, csr1))
    assert torch.equal(gx0, gx1) and gx1.dtype == dtype
    for n in ("b_enc", "W_dec", "b_dec"):
        assert torch.equal(g0[n], g1[n]), n
    with torch.no_grad():
        held = quantize_rows(x, shift=sae.b_dec)
        want = sparse_backward(held, sae.W_enc, sae.b_enc, sae.W_dec, sae.b_dec, csr1, G,
                               torch.full_like(csr1[2], 0.1), need_grad_x=False)
    assert torch.equal(g1["W_enc"], want.W_enc)
    # elements are off by at most 2^-4 of themselves, or 2^-10 of their block's scale, itself at most 2^-7 of its largest
    # element: so is every sum of theirs, in magnitudes
    p = csr_to_dense(*csr1[:2], want.pre, 300).double().abs()
    xs = (x.detach().double() - sae.b_dec.detach().double()).abs()
    err = xs * 2.0 ** -4 + xs.amax(1, keepdim=True) * 2.0 ** -17
    bound = err.T.contiguous() @ p
    size = xs.T.contiguous() @ p
    diff = (g0["W_enc"].double() - g1["W_enc"].double()).abs()
    assert (diff <= bound + size * 8 * half(dtype) + tiny(dtype)).all() and diff.max() > 0


def test_forward_train_held_keeps_eight_bits_in_place_of_the_tokens():
    sae = make_sae(512, 256, "relu", torch.float32)
    x = torch.randn(4096, 512, device="cuda")
    for hold in (None, torch.float8_e4m3fn):
        x_hat, _ = forward_train(sae, x, hold=hold)
        kept = [t for t in x_hat.grad_fn.saved_tensors if t is not None and t.dim() == 2 and t.shape[0] == 4096]
        assert sum(t.nbytes for t in kept) == (4096 * 512 * 4 if hold is None else 4096 * (512 + 4))


# ----------------------------------------------------------------------------- an SAE with an input norm
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", ["relu", "jumprelu", "topk"])
def test_an_sae_with_an_input_norm_is_its_parts(activation, dtype):
    sae, bare = make_sae(96, 320, activation, dtype, "layer_norm"), make_sae(96, 320, activation, dtype)
    bare.load_state_dict(sae.state_dict())
    x = (torch.randn(50, 96, device="cuda") * 3 + 1).to(dtype)
    with torch.no_grad():
        z, mean, rstd = layer_norm(x, return_stats=True)
        csr, want = saeflow_amd.encode_sparse(sae, x), saeflow_amd.encode_sparse(bare, z)
        assert all(torch.equal(a, b) for a, b in zip(csr, want))
        assert torch.equal(sae.encode(x), bare.encode(z)) and torch.equal(sae.encode_pre(x), bare.encode_pre(z))
        h = saeflow_amd.decode_sparse(sae, csr)
        assert torch.equal(sae(x), denormalize(h, mean, rstd))
        assert torch.equal(saeflow_amd.forward(bare, x), saeflow_amd.decode_sparse(bare, saeflow_amd.encode_sparse(bare, x)))
        e8, b8 = Fp8Encoder.from_sae(sae), Fp8Encoder.from_sae(bare)
        assert all(torch.equal(a, b) for a, b in zip(e8.encode_sparse(x), b8.encode_sparse(z)))
        rows = quantize_rows(z, shift=sae.b_dec)
        assert torch.equal(e8.encode(rows), b8.encode(rows))
    x_hat, csr_t = forward_train(sae, x)
    assert torch.equal(x_hat, sae(x)) and all(torch.equal(a, b) for a, b in zip(csr_t, csr))


@pytest.mark.parametrize("hold", [None, torch.float8_e4m3fn])
def test_training_through_the_input_norm(hold):
    """norm -> encode -> decode -> the norm undone, all gradients against float64: without hold autograd of the whole, with
    hold the formulas on what the rows hold."""
    M, D, N = 60, 96, 320
    sae = make_sae(D, N, "jumprelu", torch.float32, "layer_norm")
    x = (torch.randn(M, D, device="cuda") * 2 + 0.7).requires_grad_(True)
    G = torch.randn(M, D, device="cuda")
    x_hat, (ip, ix, va) = forward_train(sae, x, hold=hold)
    ((x_hat * G).sum() + 0.3 * va.sum()).backward()
    active = csr_to_dense(ip, ix, torch.ones_like(va), N).double().cpu()
    X, We, be, Wd, bd = (t.detach().double().cpu().requires_grad_(True) for t in (x, sae.W_enc, sae.b_enc, sae.W_dec, sae.b_dec))
    mean = X.mean(1, keepdim=True)
    rstd = ((X - mean) ** 2).mean(1, keepdim=True).add(1e-5).rsqrt()
    z = (X - mean) * rstd
    f = ((z - bd) @ We + be) * active
    h = f @ Wd + bd
    out = h / rstd + mean
    torch.testing.assert_close(x_hat.detach().double().cpu(), out.detach(), atol=1e-4, rtol=1e-4)
    if hold is None:
        ((out * G.double().cpu()).sum() + 0.3 * f.sum()).backward()
        want = {"x": X.grad, "W_enc": We.grad, "b_enc": be.grad, "W_dec": Wd.grad, "b_dec": bd.grad}
    else:
        with torch.no_grad():
            zg, h8, _, _ = kernels.layer_norm_held(x.detach())
            d, zv = held_values(h8), held_values(quantize_rows(zg, shift=sae.b_dec.detach()))
            r = rstd[:, 0]
            gh, gm, gs = onorm.undone_backward(G, h, r)
            p = (gh @ Wd.T + 0.3) * active
            gz = p @ We.T
            want = {"x": onorm.backward(gz, d, r, None, gm, gs).x, "W_enc": zv.T @ p, "b_enc": p.sum(0), "W_dec": f.T @ gh,
                    "b_dec": gh.sum(0) - gz.sum(0)}
    got = {n: getattr(sae, n).grad for n in ("W_enc", "b_enc", "W_dec", "b_dec")} | {"x": x.grad}
    for name, w in want.items():
        torch.testing.assert_close(got[name].double().cpu(), w, atol=1e-4 * float(w.abs().max()), rtol=1e-4, msg=name)


def test_a_training_step_of_all_of_it_and_a_cache_of_the_features(tmp_path):
    """As it would be used: a layer norm with weights ahead of a dictionary, both trained with 8 bits held, by AdamW; then
    the features of a normed dictionary cached on the fly."""
    sae = make_sae(128, 512, "topk", torch.bfloat16)
    w, b = torch.ones(128, device="cuda", requires_grad=True), torch.zeros(128, device="cuda", requires_grad=True)
    params = [w, b, sae.W_enc, sae.b_enc, sae.W_dec, sae.b_dec]
    opt = torch.optim.AdamW(params, lr=1e-3)
    before = [p.detach().clone() for p in params]
    for step in range(3):
        x = torch.randn(4, 64, 128, device="cuda").to(torch.bfloat16)
        z = layer_norm(x, w, b, hold=torch.float8_e4m3fn).view(-1, 128)
        x_hat, _ = forward_train(sae, z, hold=torch.float8_e4m3fn)
        loss = (x_hat - z).float().pow(2).sum(-1).mean()
        opt.zero_grad()
        loss.backward()
        assert all(torch.isfinite(p.grad).all() and p.grad.dtype == p.dtype for p in params)
        opt.step()
    assert all(not torch.equal(p, q) for p, q in zip(params, before))

    model = TinyHooked(device="cuda")
    normed = make_sae(32, 96, "relu", torch.float32, "layer_norm")
    tokens = torch.randint(0, 100, (6, 10))
    hook = "blocks.1.hook_resid_post"
    out = cache_activations(model, tokens, [hook], tmp_path / "c", batch_size=2, batches_per_shard=2, encoders={hook: normed})
    with torch.inference_mode():
        rows = model.run_with_cache(tokens.cuda(), names_filter=[hook])[1][hook].reshape(60, 32)
        want = csr_to_dense(*saeflow_amd.encode_sparse(normed, rows), 96).cpu()
    got = torch.cat([csr_to_dense(*(t.cuda() for t in csr), 96).cpu() for csr in ActivationReader(out).iter_batches(hook, 25)])
    torch.testing.assert_close(got, want, atol=1e-5, rtol=1e-5)


def test_graph_replays_of_a_held_backward_match_eager():
    x, W_enc, b_enc, W_dec, b_dec, csr, f, G, H = problem(150, 1000, 256, torch.bfloat16, hot=2)
    xg, We, be, Wd, bd, ip, ix, va, Gg, Hg = cuda(x, W_enc, b_enc, W_dec, b_dec, *csr, G, H)

    def step():
        gr = sparse_backward(quantize_rows(xg, shift=bd), We, be, Wd, bd, (ip, ix, va), Gg, Hg, need_grad_x=False)
        return gr.W_enc, gr.b_enc, gr.W_dec, gr.b_dec

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (1, 2, 3):
        torch.manual_seed(seed)
        xg.copy_(torch.randn(150, 1000))
        Gg.copy_(0.1 * torch.randn(150, 1000))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(want, outs)), seed


def test_rows_that_are_not_numbers_reach_only_their_features():
    x, W_enc, b_enc, W_dec, b_dec, csr, f, G, _ = problem(40, 200, 64, torch.bfloat16)
    x[7, 3] = float("nan")
    xg, We, be, Wd, bd, ip, ix, va, Gg = cuda(x, W_enc, b_enc, W_dec, b_dec, *csr, G)
    gr = sparse_backward(quantize_rows(xg, shift=bd), We, be, Wd, bd, (ip, ix, va), Gg, need_grad_x=False)
    on = f[7] != 0
    assert on.any() and torch.isnan(gr.W_enc.cpu()[3][on]).all()
    rest = gr.W_enc.cpu().clone()
    rest[3, on] = 0
    assert torch.isfinite(rest).all()
    assert torch.equal(dequantize_rows(quantize_rows(xg, shift=bd))[8].isnan().any().cpu(), torch.tensor(False))


def test_sparse_backward_from_held_rows_four_items_a_wave():
    """Over 40000 work items of less than four entries each, as on wide dictionaries."""
    M, D, N = 2500, 72, 45100
    g = torch.Generator().manual_seed(5)
    cols = torch.stack([torch.randperm(N, generator=g)[:24].sort().values for _ in range(M)])
    indptr, indices = torch.arange(0, 24 * M + 1, 24), cols.flatten().int()
    values = torch.rand(24 * M, generator=g) + 0.1
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, W_enc, W_dec, G = n(M, D), n(D, N) / D ** 0.5, n(N, D) / D ** 0.5, 0.1 * n(M, D)
    b_enc, b_dec = torch.zeros(N), torch.zeros(D)
    xg, We, be, Wd, bd, ip, ix, va, Gg = cuda(x, W_enc, b_enc, W_dec, b_dec, indptr, indices, values, G)
    held = quantize_rows(xg)
    got = sparse_backward(held, We, be, Wd, bd, (ip, ix, va), Gg)
    rows, j = torch.arange(M).repeat_interleave(24), indices.long()
    p = (G.double()[rows] * W_dec.double()[j]).sum(1)
    pa = (G.double()[rows].abs() * W_dec.double()[j].abs()).sum(1)
    v = held_values(held)[rows]
    want = torch.zeros(N, D, dtype=torch.float64).index_add_(0, j, p[:, None] * v)
    size = torch.zeros(N, D, dtype=torch.float64).index_add_(0, j, pa[:, None] * v.abs())
    within(got.W_enc, want.T, U * (D / 64 + 24 + 16) * size.T, "dW_enc")
    wd = torch.zeros(N, D, dtype=torch.float64).index_add_(0, j, values.double()[:, None] * G.double()[rows])
    wa = torch.zeros(N, D, dtype=torch.float64).index_add_(0, j, values.double()[:, None] * G.double()[rows].abs())
    within(got.W_dec, wd, U * 16 * wa, "dW_dec")


@pytest.mark.parametrize("dtype,top", [(torch.float16, 65504.0), (torch.float32, 1e36), (torch.float32, 1e-37), (torch.bfloat16, 1e-38)])
def test_held_rows_at_the_ends_of_their_range(dtype, top):
    """Tokens near a type's largest number (whose code may stand for more than fp16 holds) and near the smallest."""
    M, D, N = 12, 256, 64
    x, W_enc, b_enc, W_dec, b_dec, csr, f, G, _ = problem(M, D, N, dtype, l0=10)
    x = (torch.rand(M, D) * 2 - 1) * top
    x[:, 0] = top
    x[3, 130:] = 0
    x = x.to(dtype)
    b_dec = torch.zeros_like(b_dec)
    scale = 1e-4 if top > 1 else 1e4  # of the gradients, so that results are ordinary numbers of their type
    G = (G * scale).to(dtype)
    xg, We, be, Wd, bd, ip, ix, va, Gg = cuda(x, W_enc, b_enc, W_dec, b_dec, *csr, G)
    held = quantize_rows(xg, shift=bd)
    got = sparse_backward(held, We, be, Wd, bd, (ip, ix, va), Gg, need_grad_x=False)
    v, p = held_values(held), (G.double() @ W_dec.double().T) * (f != 0)
    pa = (G.double().abs() @ W_dec.double().abs().T) * (f != 0)
    want = v.T @ p
    n = (f != 0).sum(0).double()
    tol = U * (n + 8) * (v.abs().T @ p.abs()) + U * (D / 64 + 24) * (v.abs().T @ pa) + M * 2.0 ** -149
    within(got.W_enc, want, 1.01 * half(dtype) * want.abs() + tiny(dtype) + 1.01 * tol, "dW_enc")
    assert torch.isfinite(got.W_enc).all() and (want != 0).any()


@pytest.mark.parametrize("M", [1_100_000, 1_870_000])  # 2.5 and 4.3 GB of codes
def test_held_rows_past_two_and_four_gigabytes(M):
    D, N = 2304, 64
    dt = torch.bfloat16
    at = torch.tensor([0, 1, 934_999, M - 2, M - 1])
    g = torch.Generator().manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    xs, Gs = n(5, D).to(dt), (0.1 * n(5, D)).to(dt)
    W_enc, W_dec = (n(D, N) / 48).to(dt), (n(N, D) / 48).to(dt)
    cols = torch.stack([torch.randperm(N, generator=g)[:40].sort().values for _ in range(5)])
    counts = torch.zeros(M, dtype=torch.int64)
    counts[at] = 40
    indptr = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
    values = (torch.rand(200, generator=g) + 0.1).to(dt)
    x, G = torch.zeros(M, D, dtype=dt, device="cuda"), torch.zeros(M, D, dtype=dt, device="cuda")
    x[at.cuda()], G[at.cuda()] = xs.cuda(), Gs.cuda()
    held = quantize_rows(x)
    del x
    We, Wd, be, bd = W_enc.cuda(), W_dec.cuda(), torch.zeros(N, dtype=dt, device="cuda"), torch.zeros(D, dtype=dt, device="cuda")
    got = sparse_backward(held, We, be, Wd, bd, (indptr.cuda(), cols.flatten().int().cuda(), values.cuda()), G, need_grad_x=False)
    on = torch.zeros(5, N, dtype=torch.float64).scatter_(1, cols, 1.0)
    v = torch.cat([held_values(held[i:i + 1]) for i in at.tolist()])
    p, pa = (Gs.double() @ W_dec.double().T) * on, (Gs.double().abs() @ W_dec.double().abs().T) * on
    want = v.T @ p
    tol = U * 16 * (v.abs().T @ p.abs()) + U * (D / 64 + 24) * (v.abs().T @ pa)
    within(got.W_enc, want, 1.01 * half(dt) * want.abs() + tiny(dt) + 1.01 * tol, "dW_enc")


def test_an_sae_called_outside_of_training_gives_no_gradient():
    """As without an input norm: what sae(x) returns is not part of a graph, not even through the rows' means."""
    for norm in (None, "layer_norm"):
        sae = make_sae(64, 128, "relu", torch.float32, norm)
        x = torch.randn(8, 64, device="cuda", requires_grad=True)
        assert sae(x).grad_fn is None and sae.encode(x).grad_fn is None and sae.encode_pre(x).grad_fn is None
        assert Fp8Encoder.from_sae(sae).encode(x).grad_fn is None


def test_a_frozen_norm_ahead_of_a_trained_one():
    """Gradients of x alone through a layer norm whose parameters are fixed."""
    x = torch.randn(40, 96, device="cuda", requires_grad=True)
    w, b = torch.randn(96, device="cuda"), torch.randn(96, device="cuda")
    G = torch.randn(40, 96, device="cuda")
    layer_norm(x, w, b).backward(G)
    with torch.no_grad():
        _, mean, rstd = kernels.layer_norm(x, w, b)
        gr = kernels.layer_norm_backward(G, x, mean, rstd, w, b, need_grad_weight=False)
    assert gr.weight is None and torch.equal(x.grad, gr.x)
    assert torch.equal(gr.bias, kernels.layer_norm_backward(G, x.detach(), mean, rstd, w, b).bias)


def test_no_tokens_and_tokens_without_features():
    sae = make_sae(48, 96, "relu", torch.float32, "layer_norm")
    for M, shift in ((0, 0.0), (5, -1e6)):
        with torch.no_grad():
            sae.b_enc.fill_(shift)
        x = torch.randn(M, 48, device="cuda", requires_grad=True)
        x_hat, csr = forward_train(sae, x, hold=torch.float8_e4m3fn)
        assert x_hat.shape == (M, 48) and csr[1].numel() == 0
        x_hat.sum().backward()
        g = grads_of(sae)
        assert all((g[n] == 0).all() for n in ("W_enc", "b_enc", "W_dec")) and x.grad.shape == (M, 48)
        assert sae(x.detach()).shape == (M, 48)


def test_two_streams_at_once():
    """Backward passes side by side on two streams, each with its own workspaces."""
    def inputs(seed):
        x, W_enc, b_enc, W_dec, b_dec, csr, f, G, H = problem(800, 768, 512, torch.bfloat16, seed=seed, hot=2)
        return cuda(x, W_enc, b_enc, W_dec, b_dec, *csr, G, H, torch.randn(768).bfloat16(), torch.randn(768).bfloat16())

    def work(x, We, be, Wd, bd, ip, ix, va, G, H, w, b):
        y, held, mean, rstd = kernels.layer_norm_held(x, w, b)
        a = kernels.layer_norm_backward(G, held, None, rstd, w, b)
        c = sparse_backward(quantize_rows(y, shift=bd), We, be, Wd, bd, (ip, ix, va), G, H)
        return y, a.x, a.weight, a.bias, c.W_enc, c.W_dec, c.b_enc, c.b_dec, c.x

    sets = [inputs(1), inputs(2)]
    want = [work(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i] = work(*sets[i])
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(a, c) for a, c in zip(want[i], got[i]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,D,N", [(1, 64, 256), (300, 1003, 777), (0, 40, 50), (17, 40, 0), (900, 513, 20000)])
@pytest.mark.parametrize("transposed", [False, True])
def test_biases_are_the_sums_of_their_parts(M, D, N, dtype, transposed):
    """sf_backward_biases against sf_column_sums and sf_matvec, bit for bit, and rounded."""
    lib, dev = _lib.load(), torch.device("cuda", torch.cuda.current_device())
    g = torch.randn(M, D + 3, device="cuda").to(dtype)[:, :D]
    W = torch.randn(N, D, device="cuda").to(dtype).T if transposed else torch.randn(D, N, device="cuda").to(dtype)
    v = torch.randn(N, device="cuda")
    code, s = _lib.DTYPE[dtype], _lib.stream(dev)
    ws = torch.empty((min(256, max(M, 1)) + min(256, max(N, 1))) * D, device="cuda")
    want = torch.empty(D, device="cuda")
    _lib.check(lib.sf_column_sums(g.data_ptr(), M, D, D + 3, code, 1.0, 0, want.data_ptr(), ws.data_ptr(), ws.numel(), s))
    _lib.check(lib.sf_matvec(W.data_ptr(), D, N, W.stride(0), W.stride(1), code, v.data_ptr(), -1.0, 1, want.data_ptr(),
                             ws.data_ptr(), ws.numel(), s))
    for out in DTYPES:
        d_bdec, d_benc = torch.empty(D, dtype=out, device="cuda"), torch.empty(N, dtype=out, device="cuda")
        _lib.check(lib.sf_backward_biases(g.data_ptr(), M, D, D + 3, code, W.data_ptr(), N, W.stride(0), W.stride(1), code,
                                          v.data_ptr(), d_benc.data_ptr(), _lib.DTYPE[out], d_bdec.data_ptr(), _lib.DTYPE[out],
                                          ws.data_ptr(), ws.numel(), s))
        assert torch.equal(d_bdec, want.to(out)) and torch.equal(d_benc, v.to(out))


def test_transposes_of_few_tokens_are_those_of_many():
    """The plan of the counting sort changes with the number of tokens; its result does not."""
    from saeflow_amd.kernels import csr_transpose

    g = torch.Generator().manual_seed(9)
    for M in (1, 16, 85, 86, 340, 341, 342, 700):
        counts = torch.randint(0, 90, (M,), generator=g)
        indptr = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
        indices = torch.randint(0, 24576, (int(indptr[-1]),), generator=g).int()
        colptr, rows, pos = csr_transpose(indptr.cuda(), indices.cuda(), 24576)
        order = torch.sort(indices, stable=True).indices
        assert torch.equal(pos.cpu().long(), order)
        assert torch.equal(rows.cpu().long(), torch.arange(M).repeat_interleave(counts)[order])
        assert torch.equal(colptr.cpu(), torch.cat([torch.zeros(1, dtype=torch.int64), torch.bincount(indices.long(), minlength=24576).cumsum(0)]))


def test_scratch_is_given_back_before_the_gradient_of_the_tokens():
    """W_enc's transpose and dx do not lie beside the scratch of the sums over the features."""
    M, D, N = 2048, 512, 8192
    x, W_enc, b_enc, W_dec, b_dec, csr, _, G, _ = problem(M, D, N, torch.float32, l0=32)
    args = cuda(x, W_enc, b_enc, W_dec, b_dec)
    csr, G = cuda(*csr), G.cuda()

    def peak(need_grad_x):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        got = sparse_backward(*args, csr, G, need_grad_x=need_grad_x)
        return torch.cuda.max_memory_allocated() - before, torch.cuda.memory_allocated() - before, got

    sums, kept, got = peak(False)
    del got
    transposed, dx = 4 * N * D, 4 * M * D
    assert sums - kept > 4 << 20  # there is scratch to speak of
    assert peak(True)[0] <= max(sums, kept + transposed + dx) + (1 << 20)
