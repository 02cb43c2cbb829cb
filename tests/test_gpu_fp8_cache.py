"""8-bit rows through the activation cache on disk: dense hooks quantised as they are written and read back,
encoded on the fly by an 8-bit encoder, and encoded again from the stored rows."""

import pytest
import torch

import saeflow_amd
from cache_model import BudgetedModel, ForwardBudgetExceeded, TinyHooked, hook_rows
from saeflow_amd.cache import ActivationReader, cache_activations
from saeflow_amd.kernels import Fp8Rows, dequantize_rows, quantize_rows

pytestmark = pytest.mark.gpu

HOOKS = ["blocks.0.hook_resid_post", "blocks.1.attn.hook_z"]


@pytest.fixture
def tokens():
    return torch.randint(0, 100, (22, 16), generator=torch.Generator().manual_seed(1))


def test_dense_hooks_in_8_bits_read_back(tokens, tmp_path):
    model = TinyHooked(d_model=160, device="cuda").eval()
    with pytest.raises(ForwardBudgetExceeded):
        cache_activations(BudgetedModel(model, 3), tokens, HOOKS, tmp_path, batch_size=4, batches_per_shard=2,
                          dtype=torch.float8_e4m3fn)
    cache_activations(model, tokens, HOOKS, tmp_path, batch_size=4, batches_per_shard=2, dtype=torch.float8_e4m3fn)
    reader = ActivationReader(tmp_path)
    assert len(reader.manifest["shards"]) == 3 and reader.n_rows() == 22 * 16
    for hook in HOOKS:
        assert reader.manifest["hooks"][hook] == {"format": "fp8", "d": 160}
        want = quantize_rows(hook_rows(model, tokens, hook))
        got = list(reader.iter_batches(hook, 100))
        assert all(isinstance(b, Fp8Rows) and b.device.type == "cpu" for b in got) and [len(b) for b in got] == [100] * 3 + [52]
        assert torch.equal(torch.cat([b.q.view(torch.uint8) for b in got]), want.q.view(torch.uint8).cpu())
        assert torch.equal(torch.cat([b.scale for b in got]), want.scale.cpu())
        back = torch.cat([dequantize_rows(b.to("cuda"), out_dtype=torch.float32) for b in got])
        assert torch.equal(back, dequantize_rows(want, out_dtype=torch.float32))


def test_8_bit_encoder_on_the_fly_and_from_stored_rows(tokens, tmp_path):
    model = TinyHooked(d_model=160, device="cuda").eval()
    sae = saeflow_amd.SAE(160, 600, "relu", device="cuda")
    sae.b_dec.copy_(torch.randn(160) * 0.1)
    sae.b_enc.fill_(-0.3)
    hook, acts = HOOKS[0], hook_rows(model, tokens, HOOKS[0])
    enc = saeflow_amd.Fp8Encoder.from_sae(sae)
    cache_activations(model, tokens, HOOKS, tmp_path / "a", batch_size=4, batches_per_shard=2,
                      dtype=torch.float8_e4m3fn, encoders={hook: enc})
    reader = ActivationReader(tmp_path / "a")
    assert reader.manifest["hooks"][hook] == {"format": "csr", "d": 600}
    got = next(reader.iter_batches(hook, 10 ** 6))
    want = enc.encode_sparse(acts)
    assert got[2].dtype == torch.bfloat16
    assert torch.equal(got[0], want[0].cpu()) and torch.equal(got[1], want[1].cpu())
    assert torch.equal(got[2], want[2].bfloat16().cpu())
    # rows stored in 8 bits as they are (no center), encoded after reading
    cache_activations(model, tokens, [hook], tmp_path / "b", batch_size=8, dtype=torch.float8_e4m3fn)
    raw = saeflow_amd.Fp8Encoder.from_sae(sae, center=torch.zeros(160, device="cuda"))
    rows = next(ActivationReader(tmp_path / "b").iter_batches(hook, 10 ** 6)).to("cuda")
    f = raw.encode(rows, out_dtype=torch.float32)
    x = dequantize_rows(rows, out_dtype=torch.float32).double() - sae.b_dec.double()
    W = dequantize_rows(raw.W, out_dtype=torch.float32).double()
    want = (x @ W.T.contiguous() + sae.b_enc.double()).clamp(min=0)
    size = x.abs() @ W.abs().T.contiguous() + sae.b_dec.abs().double() @ W.abs().T + 1
    assert ((f.double() - want).abs() <= 3 * 162 * 2.0 ** -23 * size).all()
