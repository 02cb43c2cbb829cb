"""GPU: dictionaries with an input norm where the activations' type is not the dictionary's, and where their 8-bit rows
were not normed."""

import pytest
import torch

import saeflow_amd
from saeflow_amd import SAE
from saeflow_amd.cache import ActivationReader, cache_activations

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
