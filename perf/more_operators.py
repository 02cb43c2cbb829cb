"""Timing cases of layer norm around a dictionary and of backward passes from activations held in 8 bits.

A case is a plain dict: `call` names what a pass does, the rest its sizes and types. The calls:

  norm   saeflow_amd.layer_norm: tokens normed with a weight and a bias, no gradient wanted.
  train  kernels.layer_norm then kernels.layer_norm_backward: the forward pass and, given the gradient of its result,
         the gradients of tokens, weight and bias.
  held   kernels.layer_norm_held then kernels.layer_norm_backward: the same, with 8 bits of x - mean kept for the
         backward pass in place of x.
  sae    kernels.quantize_rows then kernels.sparse_backward: a dictionary's training step keeps x - b_dec in 8 bits;
         the gradients of all its parameters from those, the CSR features and the gradients of reconstruction and
         feature values.
  undo   kernels.denormalize then kernels.denormalize_backward: a reconstruction of normed tokens carried back to the
         tokens' own space, and the gradients of reconstruction, means and inverse deviations.

Ranges: 1 to 16384 tokens; d from 64 to 4096, odd ones among them; dictionaries of 1024 to 65536 features with a mean
of 8 to 128 features a token, rows without any among them; fp32, bf16 and fp16.

Definitions, for a row x of D elements:
  mean = sum x / D, var = sum (x - mean)^2 / D, rstd = 1 / sqrt(var + eps), xh = (x - mean) rstd, y = xh w + b.
  Given g: q = g w, dx = rstd (q - mean(q) - xh mean(q xh)), dw = sum over rows of g xh, db = sum over rows of g.
  Undone: out = h / rstd + mean; given g: dh = g / rstd, dmean = sum g, drstd = -sum g h / rstd^2.
  Held in 8 bits: a block of 128 elements v of a row (the last may be short) has the scale 2^e with the smallest
  e >= -127 that gives max |v| <= 448 * 2^e; an element is v / 2^e rounded to e4m3, ties to even, times 2^e. v is x
  minus the mean (the 64-bit sum's, rounded to 32 bits), or x - b_dec, in 32 bits.
  Dictionary, entry (m, j) of the features with value f > 0: p = g[m] . W_dec[j] + gf; dW_dec[j] = sum f g[m],
  dW_enc[:, j] = sum p held[m], db_enc[j] = sum p, db_dec = sum of g over rows - W_enc db_enc.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 128
EPS = 1e-5
MOST_ENTRIES = 16384 * 64 * 2304    # of a drawn case's features times d: the largest listed one's
DEVICE = "cuda"


def _case(name, call, dtype, tokens, d, d_sae=0, l0=0):
    return {"name": name, "call": call, "dtype": dtype, "tokens": tokens, "d": d, "d_sae": d_sae, "l0": l0}


def listed():
    return [
        # one token at a time: a transcoder's input inside a generation loop
        _case("norm-token", "norm", "bf16", 1, 2304),
        # a forward pass's activations, on their way into a cache or an encoder
        _case("norm-batch", "norm", "bf16", 16384, 2304),
        # a small model's batch in fp32
        _case("train-fp32", "train", "fp32", 2048, 768),
        # sizes that fit no tile and no vector
        _case("train-odd", "train", "fp16", 1021, 1003),
        # the headline batch
        _case("train-batch", "train", "bf16", 16384, 2304),
        # the headline batch with the input held in 8 bits
        _case("held-batch", "held", "bf16", 16384, 2304),
        # one short sequence of an odd width, fp32
        _case("held-odd", "held", "fp32", 61, 1000),
        # the headline dictionary's training batch
        _case("sae-batch", "sae", "bf16", 16384, 2304, 65536, 64),
        # a small model's dictionary, fp32
        _case("sae-fp32", "sae", "fp32", 2048, 768, 24576, 64),
        # sizes that fit no tile
        _case("sae-odd", "sae", "fp16", 1000, 1000, 10007, 40),
        # reconstructions of the headline batch
        _case("undo-batch", "undo", "bf16", 16384, 2304),
        # one prompt of an odd width
        _case("undo-odd", "undo", "fp16", 137, 1003),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    call = rng.choice(["norm", "train", "train", "held", "held", "sae", "sae", "undo"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    d = rng.choice([768, 1024, 2304, 4096, 8 * _log(rng, 8, 512), _log(rng, 64, 4096)])
    tokens = _log(rng, 1, 16384)
    if call == "sae":
        d = min(d, 2304)
        l0 = _log(rng, 8, 128)
        d_sae = max(1024, 4 * l0, _log(rng, 1024, 65536))
        if rng.random() < 0.7:
            d_sae = -(-d_sae // 64) * 64
        tokens = max(1, min(tokens, MOST_ENTRIES // (l0 * d)))
        return _case("", call, dtype, tokens, d, min(d_sae, 65536), l0)
    # the largest listed passes move 16384 x 2304 elements of 2 bytes
    return _case("", call, dtype, max(1, min(tokens, 16384 * 2304 * 2 // (d * DTYPES[dtype].itemsize))), d)


# ----------------------------------------------------------------------------- the format, plainly
def _held(v):
    """fp32 [R, D] -> the values that 8-bit rows hold for it, fp32."""
    R, D = v.shape
    nb = -(-D // BLOCK)
    blocks = torch.nn.functional.pad(v, (0, nb * BLOCK - D)).view(R, nb, BLOCK)
    m, e = torch.frexp(blocks.abs().amax(-1))                 # amax = m 2^e, m in [1/2, 1); 448 = 7/8 * 2^9
    byte = torch.where(m > 0, e - 9 + (m > 0.875).int() + 127, 0).clamp(min=0)
    inverse = ((254 - byte) << 23).view(torch.float32)        # 2^-(byte - 127)
    power = torch.where(byte > 0, byte << 23, 1 << 22).view(torch.float32)
    codes = (blocks * inverse[..., None]).to(torch.float8_e4m3fn)
    return (codes.float() * power[..., None]).view(R, nb * BLOCK)[:, :D]


# ----------------------------------------------------------------------------- inputs
def _spread(d, g):
    """The dimensions' scales: log-normal, mean square 1."""
    return torch.exp(0.5 * torch.randn(d, generator=g, device=DEVICE) - 0.25)


def _tokens(M, D, g):
    """A residual stream: dimensions of different sizes around offsets of their own, tokens of different norms."""
    s, at = _spread(D, g), 0.3 * torch.randn(D, generator=g, device=DEVICE)
    r = torch.exp(0.3 * torch.randn(M, 1, generator=g, device=DEVICE))
    return torch.randn(M, D, generator=g, device=DEVICE).mul_(s).add_(at).mul_(r)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    call, dtype, M, D, N = case["call"], DTYPES[case["dtype"]], case["tokens"], case["d"], case["d_sae"]
    state = {"case": case}

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=DEVICE).mul_(scale)

    if call in ("norm", "train", "held"):
        state["x"] = _tokens(M, D, g).to(dtype)
        state["w"] = (1.0 + normal(D, scale=0.2)).to(dtype)
        state["b"] = normal(D, scale=0.1).to(dtype)
        if call != "norm":
            state["g"] = normal(M, D, scale=0.1).to(dtype)
        return state
    if call == "undo":
        state["h"] = normal(M, D).to(dtype)
        state["mean"] = normal(M, scale=0.05)
        state["rstd"] = torch.exp(-0.3 * normal(M))
        state["g"] = normal(M, D, scale=0.1).to(dtype)
        return state
    b_dec = normal(D, scale=0.1)
    state["x"] = (_tokens(M, D, g) + b_dec).to(dtype)
    state["b_dec"] = b_dec.to(dtype)
    state["W_enc"] = normal(D, N, scale=D ** -0.5).to(dtype)
    state["W_dec"] = normal(N, D, scale=D ** -0.5).to(dtype)
    state["b_enc"] = torch.zeros(N, device=DEVICE, dtype=dtype)
    state["g"] = normal(M, D, scale=0.1).to(dtype)
    # features of log-normal frequencies; a token has up to twice the mean number of them, one in sixteen has none
    k = torch.randint(0, 2 * case["l0"], (M,), generator=g, device=DEVICE)
    k[torch.rand(M, generator=g, device=DEVICE) < 1 / 16] = 0
    p = torch.exp(1.5 * normal(N))
    picks = torch.multinomial(p, M * 2 * case["l0"], replacement=True, generator=g).view(M, -1)
    live = torch.arange(2 * case["l0"], device=DEVICE) < k[:, None]
    picks = torch.where(live, picks, N).sort(dim=1).values
    live = picks < N
    live[:, 1:] &= picks[:, 1:] != picks[:, :-1]
    indptr = torch.zeros(M + 1, dtype=torch.int64, device=DEVICE)
    indptr[1:] = live.sum(1).cumsum(0)
    indices = picks[live].int()
    values = (normal(indices.numel()).abs_() + 0.05).to(dtype)
    state["csr"] = (indptr, indices, values)
    state["gf"] = (0.01 + normal(indices.numel(), scale=0.001)).to(dtype)
    return state


# ----------------------------------------------------------------------------- one pass
def _run_own(state):
    import saeflow_amd
    from saeflow_amd import kernels

    call = state["case"]["call"]
    if call == "norm":
        return saeflow_amd.layer_norm(state["x"], state["w"], state["b"], EPS)
    if call == "train":
        y, mean, rstd = kernels.layer_norm(state["x"], state["w"], state["b"], EPS)
        gr = kernels.layer_norm_backward(state["g"], state["x"], mean, rstd, state["w"], state["b"])
        return y, gr.x, gr.weight, gr.bias
    if call == "held":
        y, held, mean, rstd = kernels.layer_norm_held(state["x"], state["w"], state["b"], EPS)
        gr = kernels.layer_norm_backward(state["g"], held, mean, rstd, state["w"], state["b"])
        return y, gr.x, gr.weight, gr.bias
    if call == "undo":
        out = kernels.denormalize(state["h"], state["mean"], state["rstd"])
        return out, *kernels.denormalize_backward(state["g"], state["h"], state["rstd"])
    held = kernels.quantize_rows(state["x"], shift=state["b_dec"])
    gr = kernels.sparse_backward(held, state["W_enc"], state["b_enc"], state["W_dec"], state["b_dec"], state["csr"],
                                 state["g"], state["gf"], need_grad_x=False)
    return gr.W_enc, gr.b_enc, gr.W_dec, gr.b_dec


def _norm(state, held, backward):
    dtype = DTYPES[state["case"]["dtype"]]
    x, w, b = state["x"].float(), state["w"].float(), state["b"].float()
    # summed in 64 bits: codes of x - mean are those of the definition only if the mean is
    mean = state["x"].double().mean(1, keepdim=True).float() if held else x.mean(1, keepdim=True)
    d = x - mean
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
    y = (d * rstd * w + b).to(dtype)
    if not backward:
        return y
    g = state["g"].float()
    xh = (_held(d) if held else d) * rstd
    q = g * w
    dx = rstd * (q - q.mean(1, keepdim=True) - xh * (q * xh).mean(1, keepdim=True))
    return y, dx.to(dtype), (g * xh).sum(0).to(dtype), g.sum(0).to(dtype)


def _undo(state):
    dtype = DTYPES[state["case"]["dtype"]]
    h, g, mean, rstd = state["h"].float(), state["g"].float(), state["mean"][:, None], state["rstd"][:, None]
    return ((h / rstd + mean).to(dtype), (g / rstd).to(dtype), g.sum(1), -(g * h).sum(1) / state["rstd"] ** 2)


def _dictionary(state):
    case, dtype = state["case"], DTYPES[state["case"]["dtype"]]
    (M, D), N = state["x"].shape, case["d_sae"]
    indptr, indices, values = state["csr"]
    rows = torch.repeat_interleave(torch.arange(M, device=DEVICE), indptr[1:] - indptr[:-1])
    held = _held(state["x"].float() - state["b_dec"].float())
    g, W_dec = state["g"].float(), state["W_dec"].float()
    dW_dec = torch.zeros(N, D, device=DEVICE)
    dW_encT = torch.zeros(N, D, device=DEVICE)
    db_enc = torch.zeros(N, device=DEVICE)
    step = 1 << 17
    for e in range(0, indices.numel(), step):
        r, j, f, gf = rows[e:e + step], indices[e:e + step].long(), values[e:e + step].float(), state["gf"][e:e + step]
        gr = g[r]
        p = torch.where(f > 0, (gr * W_dec[j]).sum(1) + gf.float(), 0.0)
        dW_dec.index_add_(0, j, gr * f[:, None])
        dW_encT.index_add_(0, j, held[r] * p[:, None])
        db_enc.index_add_(0, j, p)
    db_dec = g.sum(0) - state["W_enc"].float() @ db_enc
    return dW_encT.T.to(dtype), db_enc.to(dtype), dW_dec.to(dtype), db_dec.to(dtype)


def run(state):
    if own:
        return _run_own(state)
    call = state["case"]["call"]
    if call == "undo":
        return _undo(state)
    if call == "sae":
        return _dictionary(state)
    return _norm(state, call == "held", call != "norm")


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    M, D, N, e = case["tokens"], case["d"], case["d_sae"], DTYPES[case["dtype"]].itemsize
    held = M * (D + -(-D // BLOCK))   # bytes of the tokens in 8 bits
    call = case["call"]
    if call == "norm":
        return {"bytes": 2 * M * D * e + 2 * D * e, "flops": 8 * M * D}
    if call in ("train", "held"):
        # x, g in; y, dx, the parameters' gradients out; codes written and read
        return {"bytes": 4 * M * D * e + 4 * D * e + (2 * held if call == "held" else 0), "flops": 22 * M * D}
    if call == "undo":
        return {"bytes": 4 * M * D * e + 16 * M, "flops": 7 * M * D}
    nnz = M * case["l0"] * 15 // 16
    # x, g, both dictionaries and the features in; codes written and read; four gradients out
    return {"bytes": 2 * M * D * e + 2 * held + 4 * N * D * e + 8 * M + nnz * (4 + 2 * e) + 2 * (N + D) * e,
            "flops": 6 * nnz * D + 2 * N * D}


# ----------------------------------------------------------------------------- 64-bit results
def _grid64(v):
    """The values that 8-bit rows hold for the 64-bit rows v, from the definition: e4m3 has steps of an eighth of
    the power of two below an element, of 2^-9 from 2^-6 down."""
    R, D = v.shape
    nb = -(-D // BLOCK)
    out = torch.zeros(R, nb * BLOCK, dtype=torch.float64, device=v.device)
    out[:, :D] = v
    out = out.view(R, nb, BLOCK)
    a = out.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(a / 448.0))
    e = torch.where(448.0 * torch.exp2(e - 1) >= a, e - 1, e)   # (log2 rounds: put right by the definition)
    e = torch.where(448.0 * torch.exp2(e) < a, e + 1, e).clamp(min=-127.0)
    unit = torch.exp2(e)
    u = out / unit
    low = u.abs().clamp(min=2.0 ** -6)
    top = torch.floor(torch.log2(low))
    top = torch.where(torch.exp2(top) > low, top - 1, top)
    top = torch.where(torch.exp2(top + 1) <= low, top + 1, top)
    step = torch.exp2(top - 3)
    return (torch.round(u / step) * step * unit).view(R, nb * BLOCK)[:, :D]


def _exact_norm(state, call):
    x, w, b = state["x"].double(), state["w"].double(), state["b"].double()
    D = x.shape[1]
    mean = x.sum(1, keepdim=True) / D
    centred = x - mean
    std = ((centred ** 2).sum(1, keepdim=True) / D + EPS).sqrt()
    y = centred / std * w + b
    if call == "norm":
        return y
    if call == "held":
        centred = _grid64((x - mean.float().double()).float().double())
    g = state["g"].double()
    u = centred / std
    # d y / d x of a row is diag(w) (I - 1 1^T / D - u u^T / D) / std
    q = g * w / std
    dx = q - (q.sum(1, keepdim=True) + u * (u * q).sum(1, keepdim=True)) / D
    return y, dx, torch.einsum("md,md->d", g, u), g.sum(0)


def _exact_dictionary(state):
    """Through dense features, a part of the dictionary at a time."""
    (M, D), N = state["x"].shape, state["case"]["d_sae"]
    indptr, indices, values = state["csr"]
    rows = torch.bucketize(torch.arange(indices.numel(), device=DEVICE), indptr[1:], right=True)
    held = _grid64((state["x"].double() - state["b_dec"].double()).float().double())
    g, cols = state["g"].double(), indices.long()
    dW_enc = torch.empty(D, N, dtype=torch.float64, device=DEVICE)
    dW_dec = torch.empty(N, D, dtype=torch.float64, device=DEVICE)
    db_enc = torch.empty(N, dtype=torch.float64, device=DEVICE)
    part = 8192
    for n in range(0, N, part):
        stop = min(N, n + part)
        here = (cols >= n) & (cols < stop)
        at = (rows[here], cols[here] - n)
        f = torch.zeros(M, stop - n, dtype=torch.float64, device=DEVICE)
        f[at] = values[here].double()
        gf = torch.zeros_like(f)
        gf[at] = state["gf"][here].double()
        p = (g @ state["W_dec"][n:stop].double().T.contiguous() + gf) * (f > 0)
        dW_dec[n:stop] = f.T.contiguous() @ g
        dW_enc[:, n:stop] = held.T.contiguous() @ p
        db_enc[n:stop] = p.sum(0)
    db_dec = g.sum(0) - (state["W_enc"].double() * db_enc).sum(1)
    return dW_enc, db_enc, dW_dec, db_dec


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    call = case["call"]
    if call == "sae":
        return _exact_dictionary(state)
    if call != "undo":
        return _exact_norm(state, call)
    h, g, mean, rstd = (state[k].double() for k in ("h", "g", "mean", "rstd"))
    std = 1.0 / rstd
    return (h * std[:, None] + mean[:, None], g * std[:, None], g.sum(1), (g * h).sum(1) * -(std * std))
