"""GPU: dictionaries with an input norm where the activations' type is not the dictionary's, and where their 8-bit rows
were not normed."""

import copy

import pytest
import torch

import saeflow_amd
from saeflow_amd import SAE, ActivationBuffer, Fp8Encoder, kernels
from saeflow_amd.cache import ActivationReader, cache_activations
from saeflow_amd.kernels import quantize_rows

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HOOK = "hook"


class Table(torch.nn.Module):
    """A model whose activations are rows of a table."""

    def __init__(self, rows):
        super().__init__()
        self.rows = torch.nn.Parameter(rows)

    def run_with_cache(self, tokens, names_filter=None, stop_at_layer=None, return_type=None):
        return None, {HOOK: self.rows[tokens]}


def normed_sae(D, N, activation, dtype):
    torch.manual_seed(1)
    sae = SAE(D, N, activation, k=8 if activation == "topk" else None, dtype=dtype, input_norm="layer_norm").cuda()
    sae.b_enc.copy_(0.1 * torch.randn(N) - 0.5)
    sae.b_dec.copy_(0.1 * torch.randn(D))
    return sae


@pytest.mark.parametrize("sae_dtype", DTYPES)
@pytest.mark.parametrize("rows_dtype", DTYPES)
@pytest.mark.parametrize("activation", ["relu", "topk"])
def test_cached_features_are_those_of_the_same_rows(activation, rows_dtype, sae_dtype, tmp_path):
    """Rows far from zero, which a rounding to the dictionary's type ahead of the norm would take apart, and bf16 rows past
    the largest number of fp16."""
    torch.manual_seed(0)
    rows = (torch.randn(50, 96) * 2 + 300).to(rows_dtype)
    if rows_dtype == torch.bfloat16:
        rows[::3] = (torch.randn(17, 96) * 3e4 + 7e4).bfloat16()
    model, sae = Table(rows.cuda()), normed_sae(96, 256, activation, sae_dtype)
    tokens = torch.randint(0, 50, (6, 10))
    out = cache_activations(model, tokens, [HOOK], tmp_path / "c", batch_size=2, batches_per_shard=2, encoders={HOOK: sae})
    parts = [saeflow_amd.encode_sparse(sae, model.rows.detach()[t.cuda()].flatten(0, 1)) for t in tokens.split(2)]
    assert all(torch.isfinite(p[2]).all() and p[2].numel() for p in parts)
    for got, want in zip(ActivationReader(out).iter_batches(HOOK, 20), parts):
        assert torch.equal(got[0], want[0].cpu()) and torch.equal(got[1], want[1].cpu())
        assert torch.equal(got[2], want[2].float().cpu())


def test_cached_features_of_a_model_in_64_bits(tmp_path):
    """Its rows are rounded to 32 bits, the widest type that the norm takes."""
    torch.manual_seed(0)
    rows = torch.randn(50, 96, dtype=torch.float64) * 2 + 300
    model, sae = Table(rows.cuda()), normed_sae(96, 256, "relu", torch.bfloat16)
    tokens = torch.randint(0, 50, (2, 10))
    out = cache_activations(model, tokens, [HOOK], tmp_path / "c", encoders={HOOK: sae})
    want = saeflow_amd.encode_sparse(sae, model.rows.detach()[tokens.cuda()].flatten(0, 1).float())
    (got,) = ActivationReader(out).iter_batches(HOOK, 20)
    assert torch.equal(got[1], want[1].cpu()) and torch.equal(got[2], want[2].float().cpu())


# ----------------------------------------------------------------------------- 8-bit rows and an encoder that norms
def test_rows_that_were_not_normed_are_refused_by_an_encoder_that_norms(tmp_path):
    sae = normed_sae(96, 256, "relu", torch.bfloat16)
    bare = SAE(96, 256, "relu", dtype=torch.bfloat16).cuda()
    bare.load_state_dict(sae.state_dict())
    enc, plain = Fp8Encoder.from_sae(sae), Fp8Encoder.from_sae(bare)
    torch.manual_seed(0)
    x = (torch.randn(40, 96, device="cuda") * 2 + 3).bfloat16()
    z = saeflow_amd.layer_norm(x)
    raw, normed = ActivationBuffer(64, 96, center=sae.b_dec), ActivationBuffer(64, 96, center=sae.b_dec, normed=True)
    raw.write(x)
    normed.write(z)
    for call in (enc.encode, enc.encode_sparse):
        for rows in (raw.rows(0, 40), raw.rows(3, 20)[2:5], copy.copy(raw.rows(0, 40)), kernels.layer_norm_held(x)[1]):
            with pytest.raises(ValueError, match="normed"):
                call(rows)
    want = plain.encode(quantize_rows(z, shift=sae.b_dec))
    assert torch.equal(enc.encode(normed.rows(0, 40)), want)
    assert torch.equal(enc.encode(quantize_rows(z, shift=sae.b_dec)), want)  # rows that nobody said anything about
    assert torch.equal(plain.encode(raw.rows(0, 40)), plain.encode(quantize_rows(x, shift=sae.b_dec)))
    assert torch.equal(plain.encode(normed.rows(0, 40)), want)
    assert enc.encode(raw.read()).shape == (40, 256)

    tokens = torch.arange(40).view(4, 10)
    out = cache_activations(Table(x), tokens, [HOOK], tmp_path / "c", dtype=torch.float8_e4m3fn)
    behind = cache_activations(Table(z), tokens, [HOOK], tmp_path / "z", dtype=torch.float8_e4m3fn)
    zeros = Fp8Encoder.from_sae(sae, center=torch.zeros(96, device="cuda"))
    for rows in ActivationReader(out).iter_batches(HOOK, 20):
        with pytest.raises(ValueError, match="normed"):
            zeros.encode(rows.to("cuda"))
    (rows,) = ActivationReader(behind).iter_batches(HOOK, 40, normed=True)
    assert torch.equal(zeros.encode(rows.to("cuda")), zeros.encode(quantize_rows(z)))
