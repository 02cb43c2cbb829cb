"""Timing cases of the 8-bit operators: activations and dictionaries held in e4m3 with one
power-of-two scale for each block of 128 elements of a row.

A case is a plain dict: `call` names what a pass does, the rest its sizes and types. The calls:

  encode   Fp8Encoder.encode: tokens in hand are shifted by b_dec, quantised and multiplied with the
           8-bit dictionary; bias and ReLU; the dense features.
  rows     fused_encode_fp8: the same product from rows that an 8-bit activation cache already holds.
  write    ActivationBuffer.write then read of the rows just written: a cache round trip. What 8 bits
           hold is given back as the values it stands for.
  weights  quantize_rows of a dictionary's W_enc^T (its rows lie along the other axis in memory), read
           back with dequantize_rows.
  read     ActivationBuffer.read of shuffled rows: a training batch from a long cache.

Ranges: 1 to 16384 tokens; d_in 64 to 4096, odd ones among them; dictionaries of 4096 to 2^20
features; caches of up to 2^21 rows (4.8 GB, so byte offsets pass 32 bits); fp32, bf16 and fp16.

Tokens are x = b_dec + s * N(0, 1) with log-normal s for each dimension (activations of language models
differ widely between dimensions), W_enc ~ N(0, 1/d_in), so that pre-activations are about N(0, 1),
and biases that leave a mean of 64 positive features a token.

The format, for a block of 128 elements v of a row (the last block may be short): a = max |v|; the scale is
2^e with the smallest e that has a <= 448 * 2^e, at least -127, held as the byte e + 127; a code is v / 2^e
rounded to e4m3, ties to even.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 128
L0 = 64
MOST_FLOPS = 5e12   # of a drawn case: the largest listed product
DEVICE = "cuda"


def _case(name, call, dtype, tokens, d_in, d_sae=0, cache=0, activation="relu"):
    return {"name": name, "call": call, "dtype": dtype, "tokens": tokens, "d_in": d_in, "d_sae": d_sae, "cache": cache,
            "activation": activation}


def listed():
    return [
        # one token at a time: interactive inspection, or steering inside a generation loop
        _case("token", "encode", "bf16", 1, 2304, 16384),
        # one prompt of ordinary length over the headline dictionary
        _case("prompt", "encode", "bf16", 137, 2304, 65536),
        # a small model's activations, fp32 in and out
        _case("small-fp32", "encode", "fp32", 2048, 768, 24576),
        # sizes that fit no tile, no block and no vector
        _case("odd", "encode", "fp16", 1000, 1000, 10007),
        # the headline batch, out of the cache
        _case("batch", "rows", "bf16", 16384, 2304, 65536),
        # a few sequences of the cache over the largest dictionary, bare pre-activations
        _case("wide", "rows", "bf16", 512, 2304, 1048576, activation="none"),
        # a forward pass's activations go into the cache
        _case("write", "write", "bf16", 16384, 2304, cache=32768),
        # one short sequence of an odd width, in fp32, at the end of a small ring
        _case("write-odd", "write", "fp32", 61, 1000, cache=64),
        # a dictionary is made ready
        _case("weights", "weights", "bf16", 65536, 2304),
        # a shuffled training batch out of a long cache
        _case("read", "read", "bf16", 8192, 2304, cache=1 << 21),
        # the same of a small model, odd number of rows, fp32
        _case("read-fp32", "read", "fp32", 1021, 768, cache=100003),
        # a handful of rows for inspection
        _case("read-few", "read", "fp16", 5, 1000, cache=4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    call = rng.choice(["encode", "encode", "rows", "rows", "write", "weights", "read"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    d_in = rng.choice([768, 1024, 2304, 4096, 8 * _log(rng, 8, 320), _log(rng, 64, 2560)])
    tokens = _log(rng, 1, 16384)
    if call in ("encode", "rows"):
        d_sae = _log(rng, 4096, 131072 if rng.random() < 0.9 else 1048576)
        d_sae = {0: d_sae, 1: -(-d_sae // 8) * 8}.get(rng.randrange(4), -(-d_sae // 256) * 256)
        # the plain form's products and the features stay within those of the headline batch
        tokens = max(1, min(tokens, int(MOST_FLOPS / (2 * d_in * d_sae)), (1 << 30) // d_sae))
        return _case("", call, dtype, tokens, d_in, d_sae, 0, rng.choice(["relu", "none"]) if call == "rows" else "relu")
    if call == "write":
        return _case("", call, dtype, tokens, d_in, cache=tokens + rng.randrange(0, tokens + 1))
    if call == "weights":
        return _case("", call, dtype, _log(rng, 4096, 65536), d_in)
    return _case("", call, dtype, tokens, d_in, cache=max(tokens, _log(rng, 4096, 1 << 20)))


# ----------------------------------------------------------------------------- the format, plainly
def _power(byte):
    """2^(byte - 127) in fp32 (byte 0 is subnormal there)."""
    bits = byte.int()
    return torch.where(bits > 0, bits << 23, 1 << 22).view(torch.float32)


def _quantized(v):
    """fp32 [R, D] -> e4m3 codes [R, D] and scale bytes [R, ceil(D / 128)]."""
    R, D = v.shape
    nb = -(-D // BLOCK)
    blocks = torch.nn.functional.pad(v, (0, nb * BLOCK - D)).view(R, nb, BLOCK)
    amax = blocks.abs().amax(-1)
    m, e = torch.frexp(amax)                                  # amax = m 2^e, m in [1/2, 1); 448 = 7/8 * 2^9
    byte = torch.where(amax > 0, e - 9 + (m > 0.875).int() + 127, 0).clamp(min=0)
    inverse = ((254 - byte) << 23).view(torch.float32)        # 2^-(byte - 127)
    codes = (blocks * inverse[..., None]).to(torch.float8_e4m3fn)
    return codes.view(R, nb * BLOCK)[:, :D], byte.to(torch.uint8)


def _values(codes, scale):
    """What codes [R, D] and scale bytes stand for, in fp32."""
    R, D = codes.shape
    nb = scale.shape[1]
    v = torch.nn.functional.pad(codes.float(), (0, nb * BLOCK - D)).view(R, nb, BLOCK) * _power(scale)[..., None]
    return v.view(R, nb * BLOCK)[:, :D]


# ----------------------------------------------------------------------------- inputs
def _spread(d_in, g):
    """The dimensions' scales: log-normal, mean square 1."""
    return torch.exp(0.5 * torch.randn(d_in, generator=g, device=DEVICE) - 0.25)


def _tokens(n, d_in, s, b_dec, g, dtype):
    return (b_dec.float() + s * torch.randn(n, d_in, generator=g, device=DEVICE)).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    call, dtype, T, D, N = case["call"], DTYPES[case["dtype"]], case["tokens"], case["d_in"], case["d_sae"]
    state = {"case": case}
    s = _spread(D, g)
    b_dec = (0.1 * torch.randn(D, generator=g, device=DEVICE)).to(dtype)
    if call in ("encode", "rows"):
        W_enc = (torch.randn(D, N, generator=g, device=DEVICE) / math.sqrt(D)).to(dtype)
        b_enc = torch.full((N,), -float(torch.special.ndtri(torch.tensor(1.0 - min(0.5, L0 / N)))), device=DEVICE)
        state["b_enc"], state["b_dec"] = b_enc.to(dtype), b_dec
        x = _tokens(T, D, s, b_dec, g, dtype)
        if own:
            import saeflow_amd
            from saeflow_amd.kernels import quantize_rows

        if call == "encode":
            state["x"] = x
            if own:
                state["encoder"] = saeflow_amd.Fp8Encoder(W_enc, state["b_enc"], b_dec, activation="relu")
                return state
        elif own:
            state["rows"] = quantize_rows(x, shift=b_dec)
            state["W"] = quantize_rows(W_enc.T)
            return state
        else:
            state["rows"] = _quantized(x.float() - b_dec.float())
        codes, scale = torch.empty(N, D, dtype=torch.float8_e4m3fn, device=DEVICE), []
        for n in range(0, N, 65536):
            part, byte = _quantized(W_enc[:, n:n + 65536].T.float())
            codes[n:n + 65536] = part
            scale.append(byte)
        state["W"] = (codes, torch.cat(scale))
        return state
    if call == "weights":
        state["W_enc"] = (torch.randn(D, T, generator=g, device=DEVICE) / math.sqrt(D)).to(dtype)
        return state
    R = case["cache"]
    if own:
        import saeflow_amd

        state["buffer"] = saeflow_amd.ActivationBuffer(R, D, center=b_dec, device=DEVICE)
    state["b_dec"] = b_dec
    if call == "write":
        state["x"] = _tokens(T, D, s, b_dec, g, dtype)
        return state
    codes = None if own else torch.empty(R, D, dtype=torch.float8_e4m3fn, device=DEVICE)
    scale = []
    for r in range(0, R, 65536):
        x = _tokens(min(65536, R - r), D, s, b_dec, g, dtype)
        if own:
            state["buffer"].write(x)
        else:
            part, byte = _quantized(x.float() - b_dec.float())
            codes[r:r + 65536] = part
            scale.append(byte)
    if not own:
        state["cache"] = (codes, torch.cat(scale))
    state["ids"] = torch.randperm(R, generator=g, device=DEVICE)[:T]
    return state


# ----------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    call, dtype = case["call"], DTYPES[case["dtype"]]
    if own:
        if call == "encode":
            return state["encoder"].encode(state["x"])
        if call == "rows":
            from saeflow_amd.kernels import fused_encode_fp8

            return fused_encode_fp8(state["rows"], state["W"], state["b_enc"], activation=case["activation"],
                                    out_dtype=dtype)
        if call == "write":
            at = state["buffer"].write(state["x"])
            return state["buffer"].read(at, out_dtype=dtype)
        if call == "weights":
            from saeflow_amd.kernels import dequantize_rows, quantize_rows

            return dequantize_rows(quantize_rows(state["W_enc"].T), out_dtype=dtype)
        return state["buffer"].read(state["ids"], out_dtype=dtype)
    if call in ("encode", "rows"):
        codes = state["rows"] if call == "rows" else _quantized(state["x"].float() - state["b_dec"].float())
        f = _values(*codes) @ _values(*state["W"]).T + state["b_enc"].float()
        return (f.clamp(min=0.0) if case["activation"] == "relu" else f).to(dtype)
    if call == "weights":
        return _values(*_quantized(state["W_enc"].T.float())).to(dtype)
    b_dec = state["b_dec"].float()
    if call == "write":
        return (_values(*_quantized(state["x"].float() - b_dec)) + b_dec).to(dtype)
    codes, scale = state["cache"]
    return (_values(codes[state["ids"]], scale[state["ids"]]) + b_dec).to(dtype)


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    T, D, N, e = case["tokens"], case["d_in"], case["d_sae"], DTYPES[case["dtype"]].itemsize
    held = D + -(-D // BLOCK)  # bytes of a row in 8 bits
    call = case["call"]
    if call == "encode":
        return {"bytes": T * D * e + D * e + N * (held + e) + T * N * e, "flops": 2 * T * D * N + 4 * T * D}
    if call == "rows":
        return {"bytes": T * held + N * (held + e) + T * N * e, "flops": 2 * T * D * N}
    if call == "write":
        return {"bytes": T * D * e + T * held + T * D * e + D * e, "flops": 6 * T * D}
    if call == "weights":
        return {"bytes": T * D * e + T * held + T * D * e, "flops": 4 * T * D}
    return {"bytes": T * 8 + T * held + T * D * e + D * e, "flops": 2 * T * D}


# ----------------------------------------------------------------------------- 64-bit results
_E4M3 = torch.tensor([(-1.0) ** (c >> 7) * (math.nan if c & 127 == 127 else
                                             (c & 7) * 2.0 ** -9 if (c >> 3) & 15 == 0 else
                                             (8 + (c & 7)) * 2.0 ** (((c >> 3) & 15) - 10)) for c in range(256)],
                     dtype=torch.float64)


def _held64(v):
    """The values that the format holds for the rows v (64 bits): the grid of each element worked out
    from the definition, with e4m3's three fraction bits above 2^-6 and steps of 2^-9 below."""
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
    top = torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6)))
    top = torch.where(torch.exp2(top) > u.abs().clamp(min=2.0 ** -6), top - 1, top)
    step = torch.exp2(top - 3)
    return (torch.round(u / step) * step * unit).view(R, nb * BLOCK)[:, :D]


def _rounded_once(v):
    """Differences are formed in fp32 by the format's definition."""
    return v.float().double()


@torch.no_grad()
def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    call = case["call"]
    if call in ("encode", "rows"):
        b_enc = state["b_enc"].double()
        table = _E4M3.to(DEVICE)

        def held(codes, byte):
            v = table[codes.contiguous().view(torch.uint8).int()]
            two = torch.exp2(byte.double() - 127.0)
            return v * two.repeat_interleave(BLOCK, dim=1)[:, :v.shape[1]]

        if call == "encode":
            rows = _held64(_rounded_once(state["x"].double() - state["b_dec"].double()))
        else:
            rows = held(*state["rows"])
        out = torch.empty(case["tokens"], case["d_sae"], dtype=torch.float64, device=DEVICE)
        codes, byte = state["W"]
        step = max(1, (1 << 27) // case["d_in"])
        for n in range(0, case["d_sae"], step):
            f = rows @ held(codes[n:n + step], byte[n:n + step]).T.contiguous() + b_enc[n:n + step]
            out[:, n:n + step] = f.clamp(min=0.0) if case["activation"] == "relu" else f
        return out
    if call == "weights":
        W = state["W_enc"].T
        return torch.cat([_held64(W[r:r + 16384].double()) for r in range(0, case["tokens"], 16384)])
    b_dec = state["b_dec"].double()
    if call == "write":
        return _held64(_rounded_once(state["x"].double() - b_dec)) + b_dec
    codes, byte = (t[state["ids"]] for t in state["cache"])
    v = _E4M3.to(DEVICE)[codes.view(torch.uint8).int()]
    return v * torch.exp2(byte.double() - 127.0).repeat_interleave(BLOCK, dim=1)[:, :case["d_in"]] + b_dec
